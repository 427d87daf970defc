// Causal attention of a step's tokens over a paged key-value cache, the C entry: o = softmax(scale q K^T) V over the keys of
// the token's sequence up to its position, the last `window` of them if that is not 0. A token without keys gets zeros.
//
// Up to TOKEN_ROWS rows of a key head (its query heads times the new tokens of a sequence) go to cache_token.hip, which reads
// every key once and shares a sequence's keys out; more rows, and packed prompts, to cache_prompt.hip.
#include "cache_parts.h"

using namespace krn;

// The plan of a call without starts; without memory for its parts the keys of a sequence stay in one workgroup
static TokenPlan plan_of(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t d, int64_t page, int64_t sequences,
                         int64_t width, int64_t bytes) {
  const int64_t step = tokens / sequences;
  TokenPlan p = token_plan(step, heads / kv_heads, kv_heads, d, page, sequences, width);
  if (p.bytes > bytes) p = token_plan(step, heads / kv_heads, kv_heads, d, page, sequences, 0);
  return p;
}

extern "C" int64_t krn_cache_attention_workspace(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t d, int64_t page,
                                                 int packed, int64_t sequences, int64_t width) {
  if (tokens <= 0 || sequences <= 0 || kv_heads <= 0 || heads < kv_heads || width <= 0 || page <= 0) return 0;
  const int64_t group = heads / kv_heads, step = packed ? 0 : tokens / sequences;
  if (packed || step * group > TOKEN_ROWS)
    return prompt_plan(tokens, step, group, kv_heads, d, page, sequences, width, INT64_MAX).bytes;
  return plan_of(tokens, heads, kv_heads, d, page, sequences, width, INT64_MAX).bytes;
}

extern "C" int krn_cache_attention(int kind, const void* q, const void* keys, const void* values, void* o, int64_t tokens,
                                   int64_t heads, int64_t kv_heads, int64_t d, int64_t pages, int64_t page,
                                   const int* starts, int64_t step, const int* lengths, const int* table,
                                   int64_t sequences, int64_t width, float scale, int64_t window, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  CacheView cache{};
  SequencesView s{};
  const CacheArguments a{"cache_attention", kind, keys, values, starts, lengths, table, tokens, heads, kv_heads, d, pages, page,
                         step, sequences, width};
  if (!krn_cache_arguments(a, cache, s)) return -1;
  if ((uintptr_t)q % 16 || (uintptr_t)o % 16) {
    krn_set_error("cache_attention: tensors must be 16-byte aligned");
    return -1;
  }
  const float by = scale * 1.4426950408889634f;  // weights are powers of two
  if (!(scale > 0.0f) || by - by != 0.0f) {
    krn_set_error("cache_attention: the scale is a positive finite number");
    return -1;
  }
  if (window < 0) {
    krn_set_error("cache_attention: a window of %lld keys", (long long)window);
    return -1;
  }
  if (tokens * heads > 0x7fffffff - PROMPT_ROWS) {
    krn_set_error("cache_attention: %lld tokens of %lld heads", (long long)tokens, (long long)heads);
    return -1;
  }
  const int64_t bytes = tokens * heads * d * 2, held = pages * page * kv_heads * d * 2;
  if ((o != q && share_memory(o, bytes, q, bytes)) || share_memory(o, bytes, keys, held) ||
      share_memory(o, bytes, values, held) || share_memory(o, bytes, starts, starts ? (sequences + 1) * 4 : 0) ||
      share_memory(o, bytes, lengths, sequences * 4) || share_memory(o, bytes, table, sequences * width * 4)) {
    krn_set_error("cache_attention: the result shares memory with another tensor (over the queries alone it may lie)");
    return -1;
  }
  if (tokens == 0 || sequences == 0) return 0;
  if ((uintptr_t)workspace % 16) {
    krn_set_error("cache_attention: the workspace must be 16-byte aligned");
    return -1;
  }
  const int group = (int)(heads / kv_heads), span = window > 0x7fffffff ? 0 : (int)window;
  if (!starts && step * group <= TOKEN_ROWS) {
    const TokenPlan p = plan_of(tokens, heads, kv_heads, d, page, sequences, width, workspace ? workspace_bytes : 0);
    if (p.workgroups * kv_heads >= (int64_t)1 << 24) {
      krn_set_error("cache_attention: %lld sequences of %lld key heads", (long long)sequences, (long long)kv_heads);
      return -1;
    }
    TokenCall c{};
    c.q = (const uint16_t*)q, c.o = (uint16_t*)o, c.cache = cache, c.s = s, c.heads = (int)heads, c.group = group;
    c.window = span, c.scale = by;
    launch_cache_tokens(kind == BF16, (int)d, c, p, workspace, (hipStream_t)stream);
  } else {
    const PromptPlan p = prompt_plan(tokens, starts ? 0 : step, group, kv_heads, d, page, sequences, width,
                                     workspace ? workspace_bytes : 0);
    if (p.workgroups * kv_heads >= (int64_t)1 << 23) {
      krn_set_error("cache_attention: %lld tokens of %lld sequences and %lld heads", (long long)tokens, (long long)sequences,
                    (long long)heads);
      return -1;
    }
    PromptCall c{};
    c.q = (const uint16_t*)q, c.o = (uint16_t*)o, c.cache = cache, c.s = s, c.heads = (int)heads, c.kv_heads = (int)kv_heads;
    c.group = group, c.window = span, c.scale = by;
    launch_cache_prompt(kind == BF16, (int)d, c, p, workspace, (hipStream_t)stream);
  }
  const hipError_t err = hipGetLastError();
  if (err == hipSuccess) return 0;
  krn_set_error("cache_attention launch: %s", hipGetErrorString(err));
  return (int)err;
}
