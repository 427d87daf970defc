// Queries, keys and values of a step's tokens from their fused projection: queries and keys rotated by their positions, keys
// and values stored into a paged cache, in one pass over the projection.
//
// Pair j of a head, (a, b), becomes m (a cos t - b sin t, b cos t + a sin t) with t = position * frequency[j]. The angle is
// kept in turns as a 64-bit fraction: frequency / 2 pi mod 1 times 2^64, multiplied by the position modulo 2^64, is exact at
// any position, where a float32 angle is off by 0.06 rad at a million. Its upper 32 bits go to sincospif as half turns. The
// sines of a token serve all its heads, so a workgroup has one token, or some heads of it, and computes them once, into LDS.
// It has 256 lanes whatever the heads: rows of few heads leave most idle (16384 tokens of 4 heads of 64 on 1 22.7 us, the
// bytes 5; 64 lanes there 12.0, but wide rows 1 to 3 % slower). A packed token's sequence is counted out of all starts by each
// workgroup (8192 sequences of one token 65 us, without starts 32).
//
// Bound by memory: every byte of the projection is read once and written once, 16 bytes a lane.
#include "cache_parts.h"

namespace krn {

// Workgroups, as far as the heads of few tokens fill them (32 query and 8 key heads of 128, one workgroup a token and this:
// 16 tokens 7.4 and 3.5 us, 128 tokens 7.6 and 3.8)
constexpr int ROTARY_SPREAD = 1024;
// Bytes of a projection that is read and written non-temporally, half of the last-level cache: neither a larger one nor its
// results stay there (192 MiB 76.9 and 67.9 us, and with the product before and the attention behind it 766 and 758). Of a
// smaller one much does (48 MiB 21.4 and 17.8 us by itself, 104.4 and 106.1 in that company)
constexpr int64_t ROTARY_ONCE = (int64_t)128 << 20;

// How a head's pairs lie: full halves or interleaved pairs in whole 16-byte chunks, or anything else, by elements
enum RotaryForm : int { HALVES = 0, INTERLEAVED = 1, HALVES_ODD = 2, INTERLEAVED_ODD = 3 };

struct RotaryCall {
  const uint16_t* qkv;
  uint16_t *q, *keys, *values;
  CacheView cache;
  SequencesView s;
  const uint64_t* turns;
  int heads, rotary;
  float magnitude;
  int parts;  // workgroups that share the heads of a token
};

template <bool BF>
__device__ __forceinline__ float widen(uint16_t x) {
  return BF ? bf2f(x) : h2f(x);
}
template <bool BF>
__device__ __forceinline__ uint32_t narrow2(float lo, float hi) {
  return BF ? f2bf2(lo, hi) : (uint32_t)f2h(lo) | ((uint32_t)f2h(hi) << 16);
}
template <bool BF>
__device__ __forceinline__ void unpack8(u32x4 w, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = widen<BF>((uint16_t)(w[i] & 0xffff));
    x[2 * i + 1] = widen<BF>((uint16_t)(w[i] >> 16));
  }
}
template <bool BF>
__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
  return {narrow2<BF>(x[0], x[1]), narrow2<BF>(x[2], x[3]), narrow2<BF>(x[4], x[5]), narrow2<BF>(x[6], x[7])};
}

template <bool BF, int D, int FORM, bool ONCE>
__global__ __launch_bounds__(256) void rotary_append(RotaryCall c) {
  __shared__ float2 turn[D / 2];  // cos and sin
  __shared__ int ended[4];
  __shared__ int position;
  __shared__ int64_t slot;  // the cache row of the token's first key head; negative: none; NOBODY: nor a query
  constexpr int64_t NOBODY = -2;
  const int t = threadIdx.x, token = blockIdx.x / c.parts, part = blockIdx.x % c.parts;
  const int kv = c.cache.kv_heads, page = 1 << c.cache.page_shift;

  // the token's sequence: as many as end at or before it come first
  int owner = 0;
  if (c.s.starts) {
    int count = 0;
    for (int i = t + 1; i <= c.s.n; i += 256) count += c.s.starts[i] <= token;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) count += __shfl_xor(count, d);
    if (t % 64 == 0) ended[t / 64] = count;
    __syncthreads();
    owner = ended[0] + ended[1] + ended[2] + ended[3];
  } else {
    owner = token / c.s.step;
  }
  if (t == 0) {
    int at = 0;
    int64_t row = NOBODY;
    if (owner < c.s.n) {
      const TokenRange range = token_range(c.s, owner);
      at = sequence_length(c.s, owner) - (range.first + range.count - token);
      if (token >= range.first && token < range.first + range.count) {
        row = -1;
        if (at >= 0 && (at >> c.cache.page_shift) < c.s.width) {
          const int number = c.s.table[(int64_t)owner * c.s.width + (at >> c.cache.page_shift)];
          if ((uint32_t)number < (uint32_t)c.cache.pages)
            row = ((int64_t)number * kv << c.cache.page_shift) + (at & (page - 1));
        }
      }
    }
    position = at, slot = row;
  }
  __syncthreads();
  if (slot == NOBODY) return;
  const int half = c.rotary / 2;
  if (t < half) {
    const uint64_t angle = (uint64_t)(int64_t)position * c.turns[t];
    float sin, cos;
    sincospif((float)(int32_t)(angle >> 32) * 0x1p-31f, &sin, &cos);
    turn[t] = {cos * c.magnitude, sin * c.magnitude};
  }
  __syncthreads();

  // a rotated head is `units` pieces of work, a value head D / 8
  const int rotated = c.heads + kv, width = (rotated + kv) * D;
  const int units = FORM == HALVES ? c.rotary / 16 + (D - c.rotary) / 8 : D / 8;
  const int pieces = rotated * units + kv * (D / 8);
  const int begin = (int)((int64_t)pieces * part / c.parts), end = (int)((int64_t)pieces * (part + 1) / c.parts);
  const auto read = [&](const uint16_t* at) {
    const u32x4* x = reinterpret_cast<const u32x4*>(at);
    if constexpr (ONCE) return __builtin_nontemporal_load(x);
    else return *x;
  };
  const auto write = [&](uint16_t* at, u32x4 w) {
    u32x4* x = reinterpret_cast<u32x4*>(at);
    if constexpr (ONCE) __builtin_nontemporal_store(w, x);
    else *x = w;
  };
  for (int u = begin + t; u < end; u += 256) {
    const int over = u - rotated * units;
    const bool value = over >= 0;
    const int head = value ? rotated + over / (D / 8) : u / units, unit = value ? over % (D / 8) : u % units;
    const uint16_t* from = c.qkv + (int64_t)token * width + head * D;
    uint16_t* to;
    if (head < c.heads) {
      to = c.q + ((int64_t)token * c.heads + head) * D;
    } else {
      if (slot < 0) continue;
      const int h = value ? head - rotated : head - c.heads;
      to = (value ? c.values : c.keys) + (slot + ((int64_t)h << c.cache.page_shift)) * D;
    }
    if (value) {
      write(to + unit * 8, read(from + unit * 8));
    } else if (FORM == HALVES) {
      const int pairs = c.rotary / 16;
      if (unit >= pairs) {
        const int at = c.rotary + (unit - pairs) * 8;
        write(to + at, read(from + at));
        continue;
      }
      float a[8], b[8];
      unpack8<BF>(read(from + unit * 8), a);
      unpack8<BF>(read(from + half + unit * 8), b);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float2 w = turn[unit * 8 + e];
        const float x = a[e] * w.x - b[e] * w.y, y = b[e] * w.x + a[e] * w.y;
        a[e] = x, b[e] = y;
      }
      write(to + unit * 8, pack8<BF>(a));
      write(to + half + unit * 8, pack8<BF>(b));
    } else if (FORM == INTERLEAVED) {
      u32x4 w = read(from + unit * 8);
      if (unit * 8 < c.rotary) {
        float x[8];
        unpack8<BF>(w, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 z = turn[unit * 4 + e];
          const float a = x[2 * e], b = x[2 * e + 1];
          x[2 * e] = a * z.x - b * z.y, x[2 * e + 1] = b * z.x + a * z.y;
        }
        w = pack8<BF>(x);
      }
      write(to + unit * 8, w);
    } else {
      float x[8];
      unpack8<BF>(read(from + unit * 8), x);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int at = unit * 8 + e;
        if (at >= c.rotary) continue;
        const bool second = FORM == INTERLEAVED_ODD ? at & 1 : at >= half;
        const int other = FORM == INTERLEAVED_ODD ? at ^ 1 : second ? at - half : at + half;
        const float2 z = turn[FORM == INTERLEAVED_ODD ? at / 2 : second ? other : at];
        const float y = widen<BF>(from[other]);
        x[e] = x[e] * z.x + (second ? y * z.y : -(y * z.y));
      }
      write(to + unit * 8, pack8<BF>(x));
    }
  }
}

}  // namespace krn

using namespace krn;

bool krn_cache_arguments(const CacheArguments& a, CacheView& cache, SequencesView& sequences) {
  if (a.kind != BF16 && a.kind != F16) {
    krn_set_error("%s: element kind %d; bf16 or f16 tensors only", a.name, a.kind);
    return false;
  }
  if (a.d != 64 && a.d != 128) {
    krn_set_error("%s: head dimension %lld; 64 or 128 only", a.name, (long long)a.d);
    return false;
  }
  if (a.tokens < 0 || a.pages < 0 || a.sequences < 0 || a.width < 0) {
    krn_set_error("%s: negative extent", a.name);
    return false;
  }
  if (a.kv_heads < 1 || a.heads < 1 || a.heads % a.kv_heads) {
    krn_set_error("%s: %lld query heads cannot share %lld key heads evenly", a.name, (long long)a.heads, (long long)a.kv_heads);
    return false;
  }
  if (a.heads > 4096) {
    krn_set_error("%s: %lld heads; at most 4096", a.name, (long long)a.heads);
    return false;
  }
  if (a.page < 16 || a.page > 65536 || (a.page & (a.page - 1))) {
    krn_set_error("%s: pages of %lld keys; a power of two from 16 to 65536", a.name, (long long)a.page);
    return false;
  }
  if (a.pages > 0x7fffffff || a.pages * a.page > (int64_t)1 << 40 || a.width > 0x7fffffff || a.sequences > 0x7fffff ||
      a.tokens > 0x7fffff) {
    krn_set_error("%s: at most 2^31 - 1 pages of 2^40 keys in all, 2^23 - 1 sequences and as many tokens", a.name);
    return false;
  }
  if (a.width > 0x7fffff00 / a.page) {  // key numbers, rounded up to a tile, are 32-bit
    krn_set_error("%s: tables of %lld pages of %lld keys; fewer than 2^31 - 255 keys a sequence", a.name, (long long)a.width,
                  (long long)a.page);
    return false;
  }
  if (!a.starts && (a.step < 1 || a.step > 0x7fffff || a.tokens != a.step * a.sequences)) {
    krn_set_error("%s: %lld tokens are not %lld for each of %lld sequences", a.name, (long long)a.tokens, (long long)a.step,
                  (long long)a.sequences);
    return false;
  }
  if ((uintptr_t)a.keys % 16 || (uintptr_t)a.values % 16) {
    krn_set_error("%s: the cache must be 16-byte aligned", a.name);
    return false;
  }
  if ((uintptr_t)a.starts % 4 || (uintptr_t)a.lengths % 4 || (uintptr_t)a.table % 4) {
    krn_set_error("%s: starts, lengths and page numbers must be 4-byte aligned", a.name);
    return false;
  }
  int shift = 4;
  while ((1 << shift) < a.page) ++shift;
  cache = {a.keys, a.values, (int)a.pages, (int)a.kv_heads, shift};
  sequences = {(const int*)a.starts, (const int*)a.lengths, (const int*)a.table, (int)a.sequences,
               (int)a.width, a.starts ? 0 : (int)a.step, (int)a.tokens};
  return true;
}

template <bool BF, int D, int FORM, bool ONCE>
static void launch_form(const RotaryCall& c, hipStream_t stream) {
  hipLaunchKernelGGL((rotary_append<BF, D, FORM, ONCE>), dim3((unsigned)((int64_t)c.s.tokens * c.parts)), dim3(256), 0, stream, c);
}
template <bool BF, int D>
static void launch(const RotaryCall& c, RotaryForm form, bool once, hipStream_t stream) {
  if (form == HALVES) once ? launch_form<BF, D, HALVES, true>(c, stream) : launch_form<BF, D, HALVES, false>(c, stream);
  else if (form == INTERLEAVED) once ? launch_form<BF, D, INTERLEAVED, true>(c, stream) : launch_form<BF, D, INTERLEAVED, false>(c, stream);
  else if (form == HALVES_ODD) launch_form<BF, D, HALVES_ODD, false>(c, stream);
  else launch_form<BF, D, INTERLEAVED_ODD, false>(c, stream);
}

extern "C" int krn_rotary_append(int kind, const void* qkv, void* q, void* keys, void* values, int64_t tokens,
                                 int64_t heads, int64_t kv_heads, int64_t d, int64_t pages, int64_t page, const int* starts,
                                 int64_t step, const int* lengths, const int* table, int64_t sequences, int64_t width,
                                 const uint64_t* turns, int64_t rotary, int interleaved, float magnitude, void* stream) {
  RotaryCall c{};
  const CacheArguments a{"rotary_append", kind, keys, values, starts, lengths, table, tokens, heads, kv_heads, d, pages, page,
                         step, sequences, width};
  if (!krn_cache_arguments(a, c.cache, c.s)) return -1;
  if (rotary < 0 || rotary > d || rotary % 2) {
    krn_set_error("rotary_append: %lld rotated columns; an even number up to the head dimension %lld", (long long)rotary,
                  (long long)d);
    return -1;
  }
  if ((uintptr_t)qkv % 16 || (uintptr_t)q % 16 || (uintptr_t)turns % 8) {
    krn_set_error("rotary_append: tensors must be 16-byte aligned (frequencies 8-byte)");
    return -1;
  }
  if (!(magnitude - magnitude == 0.0f)) {
    krn_set_error("rotary_append: the magnitude is a finite number");
    return -1;
  }
  const int64_t in = tokens * (heads + 2 * kv_heads) * d * 2, out = tokens * heads * d * 2, held = pages * page * kv_heads * d * 2;
  const void *outs[] = {q, keys, values}, *ins[] = {qkv, starts, lengths, table, turns, q, keys, values};
  const int64_t out_bytes[] = {out, held, held},
                in_bytes[] = {in, starts ? (sequences + 1) * 4 : 0, sequences * 4, sequences * width * 4, rotary * 4, out, held, held};
  for (int o = 0; o < 3; ++o)
    for (int i = 0; i < 8; ++i)
      if (i != o + 5 && share_memory(outs[o], out_bytes[o], ins[i], in_bytes[i])) {
        krn_set_error("rotary_append: a result shares memory with another tensor");
        return -1;
      }
  if (tokens == 0 || sequences == 0) return 0;
  c.qkv = (const uint16_t*)qkv, c.q = (uint16_t*)q, c.keys = (uint16_t*)keys, c.values = (uint16_t*)values;
  c.turns = turns, c.heads = (int)heads, c.rotary = (int)rotary, c.magnitude = magnitude;
  const int64_t pieces = (heads + 2 * kv_heads) * (d / 8), spread = (ROTARY_SPREAD + tokens - 1) / tokens, most = (pieces + 255) / 256;
  c.parts = (int)(spread < most ? spread : most);
  const bool whole = interleaved ? rotary % 8 == 0 : rotary % 16 == 0;
  const RotaryForm form = interleaved ? whole ? INTERLEAVED : INTERLEAVED_ODD : whole ? HALVES : HALVES_ODD;
  const bool once = in >= ROTARY_ONCE;
  if (kind == BF16) d == 128 ? launch<true, 128>(c, form, once, (hipStream_t)stream) : launch<true, 64>(c, form, once, (hipStream_t)stream);
  else d == 128 ? launch<false, 128>(c, form, once, (hipStream_t)stream) : launch<false, 64>(c, form, once, (hipStream_t)stream);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) {
    krn_set_error("rotary_append launch: %s", hipGetErrorString(err));
    return (int)err;
  }
  return 0;
}
