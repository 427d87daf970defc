// Causal attention of a step's tokens over a paged key-value cache: o = softmax(scale q K^T) V over the keys of the token's
// sequence up to its position, the last `window` of them if that is not 0. A token without keys gets zeros.
//
// One wave a token and head: 64 keys at a time, a lane a key for the scores, a lane a column (or two) for the output.
#include "cache_parts.h"

namespace krn {

struct CacheAttention {
  const uint16_t* q;
  uint16_t* o;
  CacheView cache;
  SequencesView s;
  int heads, window;
  float scale;  // of the scores, times log2(e)
};

template <bool BF>
__device__ __forceinline__ float wide(uint16_t x) {
  return BF ? bf2f(x) : h2f(x);
}

template <bool BF, int D>
__global__ __launch_bounds__(64) void cache_attention_simple(CacheAttention c) {
  const int token = blockIdx.x / c.heads, head = blockIdx.x % c.heads, lane = threadIdx.x;
  int i = 0;
  if (c.s.starts) {
    for (int j = 1; j <= c.s.n; ++j) i += c.s.starts[j] <= token;
    if (i >= c.s.n) return;
  } else {
    i = token / c.s.step;
  }
  const TokenRange range = token_range(c.s, i);
  if (token < range.first || token >= range.first + range.count) return;
  const int length = sequence_length(c.s, i), at = length - (range.first + range.count - token);
  const int end = min(at + 1, held_keys(c.s, length, c.cache.page_shift)), begin = c.window ? max(0, at + 1 - c.window) : 0;
  const int kv = head / (c.heads / c.cache.kv_heads), page = 1 << c.cache.page_shift;
  const uint16_t* q = c.q + ((int64_t)token * c.heads + head) * D;
  float m = -INFINITY, total = 0.0f, acc[D / 64] = {};
  for (int k0 = begin; k0 < end; k0 += 64) {
    const int key = k0 + lane;
    int64_t row = -1;
    float s = -INFINITY;
    if (key < end) {
      const int number = c.s.table[(int64_t)i * c.s.width + (key >> c.cache.page_shift)];
      if (number >= 0 && number < c.cache.pages)
        row = (((int64_t)number * c.cache.kv_heads + kv) << c.cache.page_shift) + (key & (page - 1));
      s = 0.0f;
      if (row >= 0)
        for (int d = 0; d < D; ++d) s += wide<BF>(q[d]) * wide<BF>(((const uint16_t*)c.cache.keys)[row * D + d]);
      s *= c.scale;
    }
    float top = s;
    for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
    const float m_new = fmaxf(m, top), base = m_new == -INFINITY ? 0.0f : m_new;
    const float corr = __builtin_amdgcn_exp2f(m - base), p = key < end ? __builtin_amdgcn_exp2f(s - base) : 0.0f;
    total = total * corr + p;
    m = m_new;
    for (int x = 0; x < D / 64; ++x) acc[x] *= corr;
    for (int j = 0; j < 64 && k0 + j < end; ++j) {
      const int64_t r = __shfl(row, j);
      const float w = __shfl(p, j);
      if (r >= 0)
        for (int x = 0; x < D / 64; ++x) acc[x] += w * wide<BF>(((const uint16_t*)c.cache.values)[r * D + x * 64 + lane]);
    }
  }
  for (int x = 32; x; x >>= 1) total += __shfl_xor(total, x);
  for (int x = 0; x < D / 64; ++x) {
    const float y = end > begin ? acc[x] / total : 0.0f;
    c.o[((int64_t)token * c.heads + head) * D + x * 64 + lane] = BF ? f2bf(y) : f2h(y);
  }
}

}  // namespace krn

using namespace krn;

static int launched() {
  const hipError_t err = hipGetLastError();
  if (err == hipSuccess) return 0;
  krn_set_error("cache_attention launch: %s", hipGetErrorString(err));
  return (int)err;
}

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
  if (packed || tokens <= 0 || sequences <= 0 || heads <= 0 || kv_heads <= 0 || width <= 0) return 0;
  if (tokens / sequences * (heads / kv_heads) > TOKEN_ROWS) return 0;
  return plan_of(tokens, heads, kv_heads, d, page, sequences, width, INT64_MAX).bytes;
}

extern "C" int krn_cache_attention(int kind, const void* q, const void* keys, const void* values, void* o, int64_t tokens,
                                   int64_t heads, int64_t kv_heads, int64_t d, int64_t pages, int64_t page,
                                   const int* starts, int64_t step, const int* lengths, const int* table,
                                   int64_t sequences, int64_t width, float scale, int64_t window, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  CacheAttention c{};
  const CacheArguments a{"cache_attention", kind, keys, values, starts, lengths, table, tokens, heads, kv_heads, d, pages, page,
                         step, sequences, width};
  if (!krn_cache_arguments(a, c.cache, c.s)) return -1;
  if ((uintptr_t)q % 16 || (uintptr_t)o % 16) {
    krn_set_error("cache_attention: tensors must be 16-byte aligned");
    return -1;
  }
  if (!(scale > 0.0f) || scale - scale != 0.0f) {
    krn_set_error("cache_attention: the scale is a positive finite number");
    return -1;
  }
  if (window < 0) {
    krn_set_error("cache_attention: a window of %lld keys", (long long)window);
    return -1;
  }
  if (tokens * heads > 0x7fffffff / 64) {
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
  c.q = (const uint16_t*)q, c.o = (uint16_t*)o, c.heads = (int)heads;
  c.window = window > 0x7fffffff ? 0 : (int)window;
  c.scale = scale * 1.4426950408889634f;
  if (!starts && step * (heads / kv_heads) <= TOKEN_ROWS) {
    if ((uintptr_t)workspace % 16) {
      krn_set_error("cache_attention: the workspace must be 16-byte aligned");
      return -1;
    }
    const TokenPlan p = plan_of(tokens, heads, kv_heads, d, page, sequences, width, workspace ? workspace_bytes : 0);
    if (p.workgroups * p.columns >= (int64_t)1 << 24) {
      krn_set_error("cache_attention: %lld sequences of %lld key heads", (long long)sequences, (long long)kv_heads);
      return -1;
    }
    TokenCall t{};
    t.q = c.q, t.o = c.o, t.cache = c.cache, t.s = c.s, t.heads = c.heads, t.group = (int)(heads / kv_heads);
    t.window = c.window, t.scale = c.scale;
    launch_cache_tokens(kind == BF16, (int)d, t, p, workspace, (hipStream_t)stream);
    return launched();
  }
  const dim3 grid((unsigned)(tokens * heads));
#define KRN_SIMPLE(BF, D) hipLaunchKernelGGL((cache_attention_simple<BF, D>), grid, dim3(64), 0, (hipStream_t)stream, c)
  if (kind == BF16 && d == 128) KRN_SIMPLE(true, 128);
  else if (kind == BF16) KRN_SIMPLE(true, 64);
  else if (d == 128) KRN_SIMPLE(false, 128);
  else KRN_SIMPLE(false, 64);
#undef KRN_SIMPLE
  return launched();
}
