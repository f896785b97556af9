// RBF attention of new tokens over the paged 8-bit cache (cache.cuh): softmax(2 g q.k - g |k|^2) V, or exp(-g |q - k|^2) V
// without the denominator, for tokens 0 .. held + i of a sequence as seen by its i-th new token.
//
// A step of generation reads the whole cache once and does two products per byte: the roofline is HBM, and what has to be cheap
// is making 16-bit operands of the bytes. So the products are mma.m16n8k16 with the *cache* as the 16-row operand (tokens of a
// block, then dims) and the queries - the new tokens of the query heads that share a key/value head - as the 8 columns: a byte
// is widened once for 8 columns (32 where there are that many), and a lane's bytes lie in the cache in the order in which the
// instruction wants them. A code becomes an exact fp16 number in one permute (the byte under 0x64 is 1024 + byte) and one
// subtraction, for two values. Scales stay outside: a block's scores are multiplied by its key scale in fp32, its products with
// the values by its value scale as they are added to the output. |k|^2 is the integer sum of the codes' squares.
//   S^T (16 tokens x 8 columns) = K Q^T,  P^T by exponentials in fp32,  O^T (16 dims x 8 columns) += V^T P^T
// Queries are multiplied by the power of two that brings their largest element to [1, 2) and rounded to fp16: exact for every
// element within 2^-14 of the largest in 16-bit types, off by 2^-25 of it below. P is rounded to fp16 (2^-11 of it).
// The block that is not complete yet is held in 16 bits and multiplied in its own type.
//
// Work is split evenly whatever the lengths: all (sequence, head, column tile) segments in a row, cut into units of one load,
// are dealt to the warps of one wave in contiguous ranges. A warp works by itself - no barrier - with a running maximum (moved
// only when a score exceeds it by 2^8, which keeps P below 2^8) and writes its segment's output, or its part (unnormalised
// output, maximum, sum) where the segment is shared with other warps; a second kernel joins the parts in the order of the tokens.
#include <cstdint>
#include <cuda_runtime.h>

#include "cache.cuh"
#include "launch.h"

namespace rbf {
namespace {

constexpr int kAttnWarps = 8;
constexpr float kSlack = 8.f;                      // growth of a score, in powers of two, that does not move the maximum

template <int P>
struct Tile {
  static constexpr int kUnitBlocks = 256 / P;      // blocks of one load: 8 KB of codes
  static constexpr int kUnit = kUnitBlocks * kBlockTokens;
  static constexpr int kKeyChunks = P / 32;        // 16-byte words of a lane per block and operand
  static constexpr int kDims = P / 16;             // 16-row tiles of the output
};

__device__ __forceinline__ float attn_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <bool kBf16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kBf16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

// 8 x 8 16-bit matrix, row lane / 4 and columns 2 (lane % 4), + 1 in each lane, transposed
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Bytes 0, 1 (2, 3) of a word of codes as two fp16 numbers
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) {
  const uint32_t x = __byte_perm(w, 0x64646464u, 0x4140);
  const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&y);
}
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) {
  const uint32_t x = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&y);
}
__device__ __forceinline__ int dot4(uint32_t w) {
  const int s = static_cast<int>(w ^ 0x80808080u);
  return __dp4a(s, s, 0);
}

// How the units are dealt: segment = (sequence, column tile, head), in that order; warp w of `workers` has units
// [begin(w), begin(w + 1)).
struct Deal {
  int64_t each, rest;                              // `rest` warps have one more
  __device__ Deal(int64_t units, int64_t workers) : each(units / workers), rest(units % workers) {}
  __device__ int64_t begin(int64_t w) const { return w * each + (w < rest ? w : rest); }
  __device__ int64_t worker(int64_t unit) const {
    const int64_t longer = rest * (each + 1);
    return unit < longer ? unit / (each + 1) : rest + (unit - longer) / each;
  }
};

// Units of one segment of sequence b
template <int P>
__device__ __forceinline__ int segment_units(const CacheAttnArgs& a, int b) {
  const CacheSpan s = cache_span(a.lengths, a.fresh, b, a.T, a.max_pages);
  return s.fresh == 0 ? 0 : (s.held + s.fresh + Tile<P>::kUnit - 1) / Tile<P>::kUnit;
}

// Sum over sequences [0, n) of segment_units, by a whole warp
template <int P>
__device__ __forceinline__ int64_t units_before(const CacheAttnArgs& a, int n) {
  int64_t sum = 0;
  for (int b = threadIdx.x & 31; b < n; b += 32) sum += segment_units<P>(a, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}

// Element offset of output column c of a segment (new token c / G of query head h * G + c % G)
__device__ __forceinline__ int64_t out_offset(const CacheAttnArgs& a, int b, int h, int c) {
  return ((static_cast<int64_t>(b) * a.H * a.G + h * a.G + c % a.G) * a.T + c / a.G) * a.D;
}

// One part: per column P outputs, then the maxima and the sums of all columns
template <int P, int NT>
__device__ __forceinline__ float* part_of(const CacheAttnArgs& a, int64_t index) {
  return a.parts + index * (8 * NT) * (P + 2);
}

template <bool kBf16, int P, int NT>
__global__ void __launch_bounds__(kAttnWarps * 32) cache_attn_kernel(const CacheAttnArgs a) {
  using T = Tile<P>;
  constexpr int UB = T::kUnitBlocks, KC = T::kKeyChunks, J = T::kDims;
  constexpr int kSlot = cache_slot_bytes(P), kBytes = cache_page_bytes(P);
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t workers = static_cast<int64_t>(gridDim.x) * kAttnWarps;
  const int64_t self = static_cast<int64_t>(threadIdx.x >> 5) * gridDim.x + blockIdx.x;    // neighbours on other SMs
  const int segments = a.column_tiles * a.H;       // of a sequence
  const Deal deal(units_before<P>(a, a.B) * segments, workers);
  int64_t pos = deal.begin(self);
  const int64_t stop = deal.begin(self + 1);

  // the sequence of the first unit
  int b = 0;
  int64_t seq_begin = 0;
  if (pos < stop) {
    for (; b < a.B; b += 32) {
      const int64_t mine = b + lane < a.B ? static_cast<int64_t>(segment_units<P>(a, b + lane)) * segments : 0;
      int64_t upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
      }
      const unsigned past = __ballot_sync(0xffffffffu, seq_begin + upto > pos);
      if (past != 0) {
        const int l = __ffs(past) - 1;
        seq_begin += __shfl_sync(0xffffffffu, upto - mine, l);
        b += l;
        break;
      }
      seq_begin += __shfl_sync(0xffffffffu, upto, 31);
    }
  }

  while (pos < stop && b < a.B) {
    const CacheSpan span = cache_span(a.lengths, a.fresh, b, a.T, a.max_pages);
    const int total = span.held + span.fresh;
    const int units = span.fresh == 0 ? 0 : (total + T::kUnit - 1) / T::kUnit;
    if (pos >= seq_begin + static_cast<int64_t>(units) * segments) {       // on to the next sequence (some have no units)
      seq_begin += static_cast<int64_t>(units) * segments;
      ++b;
      continue;
    }
    const int seg = static_cast<int>((pos - seq_begin) / units);
    const int u0 = static_cast<int>((pos - seq_begin) % units);
    const int64_t left = stop - pos;
    const int u1 = left < units - u0 ? u0 + static_cast<int>(left) : units;
    const int h = seg % a.H, c0 = seg / a.H * (8 * NT);

    // ---- queries: operand columns, their scales, and how far each column sees
    uint32_t qh[NT][P / 16][2];                      // fp16, scaled
    float qmul[NT][2], qsq[NT][2];                   // of columns 2t, 2t + 1
    int limit[NT][2];                                // last token that the column sees
    // operand words of column n * 8 + g as they are in memory: k step i has dims 64 (i / 4) + 16 t + 4 (i % 4) ... + 3
    auto load_q = [&](int n, uint32_t (&w)[P / 16][2]) {
      const int c = c0 + n * 8 + g;
      const bool real = c < a.T * a.G;
      const uint16_t* q = static_cast<const uint16_t*>(a.q) + b * a.qs[0] + (real ? (h * a.G + c % a.G) * a.qs[1] + c / a.G * a.qs[2] : 0);
#pragma unroll
      for (int d = 0; d < P / 64; ++d) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int col = d * 64 + t * 16 + e * 8;
          uint4 raw = make_uint4(0, 0, 0, 0);
          if (real && col < a.D) raw = *reinterpret_cast<const uint4*>(q + col);
          w[d * 4 + e * 2][0] = raw.x;
          w[d * 4 + e * 2][1] = raw.y;
          w[d * 4 + e * 2 + 1][0] = raw.z;
          w[d * 4 + e * 2 + 1][1] = raw.w;
        }
      }
    };
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      uint32_t raw[P / 16][2];
      load_q(n, raw);
      uint32_t top = 0;
      float sq = 0.f;
#pragma unroll
      for (int i = 0; i < P / 16; ++i) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 f = unpack2<kBf16>(raw[i][e]);
          top = max(top, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
          sq = fmaf(f.x, f.x, fmaf(f.y, f.y, sq));
        }
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        sq += __shfl_xor_sync(0xffffffffu, sq, o);
      }
      uint32_t exponent = top >> 23;                 // of the largest element; zero and infinity keep their meaning
      exponent = exponent == 0 ? 127u : min(exponent, 253u);
      const float down = __uint_as_float((254u - exponent) << 23), up = __uint_as_float(exponent << 23);
#pragma unroll
      for (int i = 0; i < P / 16; ++i) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 f = unpack2<kBf16>(raw[i][e]);
          qh[n][i][e] = pack2<false>(f.x * down, f.y * down);
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int from = (2 * t + e) * 4;
        qmul[n][e] = 2.f * a.scale * __shfl_sync(0xffffffffu, up, from);
        qsq[n][e] = a.scale * __shfl_sync(0xffffffffu, sq, from);
        const int c2 = c0 + n * 8 + 2 * t + e;
        limit[n][e] = c2 < a.T * a.G ? span.held + c2 / a.G : total - 1;
      }
    }
    const int first_limit = span.held + c0 / a.G;    // every column of the tile sees at least this far

    float o[J][NT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][n][e] = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[n][e] = -INFINITY;
        l[n][e] = 0.f;
      }

    for (int u = u0; u < u1; ++u) {
      const int begin = u * T::kUnit;                // first token
      if (begin > span.held + (c0 + 8 * NT - 1) / a.G) break;              // no column of the tile sees this far
      const uint8_t* page = cache_page(a.pages, a.table, b, a.max_pages, a.num_pages, a.H, h, kBytes, begin);
      if (page == nullptr) continue;
      const uint8_t* slots = page + kPageHeader + begin % kPageTokens / kBlockTokens * kSlot;
      const float2* scales = reinterpret_cast<const float2*>(page) + begin % kPageTokens / kBlockTokens;
      const int whole = min(UB, total / kBlockTokens - begin / kBlockTokens);            // complete blocks of the unit
      const bool hidden = begin + T::kUnit - 1 > first_limit;
      float s[UB][NT][4];
      float2 sc[UB];
      // ---- scores
#pragma unroll
      for (int k = 0; k < UB; ++k) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[k][n][e] = -INFINITY;
        sc[k] = make_float2(0.f, 0.f);
        if (k >= whole) continue;
        sc[k] = scales[k];
        const uint4* key = reinterpret_cast<const uint4*>(slots + k * kSlot) + lane;
        uint4 w[KC];
#pragma unroll
        for (int i = 0; i < KC; ++i) w[i] = key[i * 32];
        int sq0 = 0, sq1 = 0;
        float acc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
#pragma unroll
        for (int d = 0; d < P / 64; ++d) {
          const uint32_t r0[4] = {w[2 * d].x, w[2 * d].y, w[2 * d].z, w[2 * d].w};
          const uint32_t r1[4] = {w[2 * d + 1].x, w[2 * d + 1].y, w[2 * d + 1].z, w[2 * d + 1].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sq0 += dot4(r0[i]);
            sq1 += dot4(r1[i]);
            const uint32_t A[4] = {codes_lo(r0[i]), codes_lo(r1[i]), codes_hi(r0[i]), codes_hi(r1[i])};
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816<false>(acc[n], A, qh[n][d * 4 + i][0], qh[n][d * 4 + i][1]);
          }
        }
#pragma unroll
        for (int x = 1; x < 4; x <<= 1) {
          sq0 += __shfl_xor_sync(0xffffffffu, sq0, x);
          sq1 += __shfl_xor_sync(0xffffffffu, sq1, x);
        }
        const float bias = a.scale * sc[k].x * sc[k].x;
        const float b0 = bias * static_cast<float>(sq0), b1 = bias * static_cast<float>(sq1);
        const int tok = begin + k * kBlockTokens + 4 * (g >> 1) + (g & 1);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float mul = qmul[n][e] * sc[k].x;
            s[k][n][e] = fmaf(acc[n][e], mul, -b0);
            s[k][n][2 + e] = fmaf(acc[n][2 + e], mul, -b1);
            if (hidden) {
              if (tok > limit[n][e]) s[k][n][e] = -INFINITY;
              if (tok + 2 > limit[n][e]) s[k][n][2 + e] = -INFINITY;
            }
          }
        }
      }
      // the incomplete block, in 16 bits: it is the last one of its unit
      const int at = whole;                          // its place in the unit, if it is there
      const bool partial = whole < UB && begin + whole * kBlockTokens < total;
      const uint16_t* tail = reinterpret_cast<const uint16_t*>(page + kPageHeader + kPageBlocks * kSlot);
      if (partial) {
        const int tok = 4 * (g >> 1) + (g & 1), base = begin + at * kBlockTokens;
        float acc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
        float sq[2] = {0.f, 0.f};
        uint32_t qt[NT][P / 16][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) load_q(n, qt[n]);
#pragma unroll
        for (int d = 0; d < P / 64; ++d) {
          uint32_t r[2][8];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const bool there = base + tok + 2 * half < total;
            const uint4* row = reinterpret_cast<const uint4*>(tail + (tok + 2 * half) * P + d * 64 + t * 16);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint4 x = there ? row[e] : make_uint4(0, 0, 0, 0);
              r[half][4 * e] = x.x; r[half][4 * e + 1] = x.y; r[half][4 * e + 2] = x.z; r[half][4 * e + 3] = x.w;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float2 f = unpack2<kBf16>(r[half][i]);
              sq[half] = fmaf(f.x, f.x, fmaf(f.y, f.y, sq[half]));
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t A[4] = {r[0][2 * i], r[1][2 * i], r[0][2 * i + 1], r[1][2 * i + 1]};
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816<kBf16>(acc[n], A, qt[n][d * 4 + i][0], qt[n][d * 4 + i][1]);
          }
        }
#pragma unroll
        for (int x = 1; x < 4; x <<= 1) {
          sq[0] += __shfl_xor_sync(0xffffffffu, sq[0], x);
          sq[1] += __shfl_xor_sync(0xffffffffu, sq[1], x);
        }
#pragma unroll
        for (int k = 0; k < UB; ++k)
          if (k == at)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const bool seen = base + tok + 2 * (e / 2) <= limit[n][e % 2] && base + tok + 2 * (e / 2) < total;
                s[k][n][e] = seen ? fmaf(acc[n][e], 2.f * a.scale, -a.scale * sq[e / 2]) : -INFINITY;
              }
      }
      // ---- the running maximum moves only if a score exceeds it by more than the slack
      float top[NT][2];
      bool over = false;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[n][e] = s[0][n][e];
#pragma unroll
          for (int k = 0; k < UB; ++k) top[n][e] = fmaxf(top[n][e], fmaxf(s[k][n][e], s[k][n][2 + e]));
          over |= top[n][e] > m[n][e] + kSlack;
        }
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = fmaxf(top[n][e], m[n][e]);
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
            const float f = m[n][e] == x ? 1.f : attn_ex2(m[n][e] - x);
            m[n][e] = x;
            l[n][e] *= f;
#pragma unroll
            for (int j = 0; j < J; ++j) {
              o[j][n][e] *= f;
              o[j][n][2 + e] *= f;
            }
          }
      }
      // ---- exponentials, the sum, and the products with the values
      uint32_t p[UB][NT][2], pt[NT][2];              // operand columns; pt: of the incomplete block, in its own type
#pragma unroll
      for (int k = 0; k < UB; ++k)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float e4[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float ref = m[n][e % 2] == -INFINITY ? 0.f : m[n][e % 2];       // no token seen yet
            e4[e] = attn_ex2(s[k][n][e] - ref);
          }
          l[n][0] += e4[0] + e4[2];
          l[n][1] += e4[1] + e4[3];
          p[k][n][0] = transpose8(pack2<false>(e4[0], e4[1]));
          p[k][n][1] = transpose8(pack2<false>(e4[2], e4[3]));
          if (k == at && partial) {
            pt[n][0] = transpose8(pack2<kBf16>(e4[0], e4[1]));
            pt[n][1] = transpose8(pack2<kBf16>(e4[2], e4[3]));
          }
        }
#pragma unroll
      for (int k = 0; k < UB; ++k) {
        if (k >= whole) continue;
        const uint4* value = reinterpret_cast<const uint4*>(slots + k * kSlot + 16 * P) + lane;
        uint4 w[KC];
#pragma unroll
        for (int i = 0; i < KC; ++i) w[i] = value[i * 32];
        const bool finite = fabsf(sc[k].y) < INFINITY;
        const int base = begin + k * kBlockTokens;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const uint32_t r0 = j % 2 ? w[j / 2].z : w[j / 2].x, r1 = j % 2 ? w[j / 2].w : w[j / 2].y;
          const uint32_t A[4] = {codes_lo(r0), codes_lo(r1), codes_hi(r0), codes_hi(r1)};
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            mma16816<false>(acc, A, p[k][n][0], p[k][n][1]);
#pragma unroll
            for (int e = 0; e < 4; ++e)               // a block that is not finite reaches the columns that see it
              if (finite || base <= limit[n][e % 2]) o[j][n][e] = fmaf(acc[e], sc[k].y, o[j][n][e]);
          }
        }
      }
      if (partial) {
        const int base = begin + at * kBlockTokens;
        const uint16_t* values = tail + kSlot / 2;
        uint2 x[KC][4];                              // dims 32 i + 4 g ... + 3 of tokens 4 t + r
        bool odd = false;                            // a value that is not finite behind what some column sees
#pragma unroll
        for (int i = 0; i < KC; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            x[i][r] = make_uint2(0, 0);
            if (base + 4 * t + r < total) x[i][r] = *reinterpret_cast<const uint2*>(values + (4 * t + r) * P + 32 * i + 4 * g);
            const uint32_t inf = kBf16 ? 0x7f80u : 0x7c00u;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t y = half ? x[i][r].y : x[i][r].x;
              odd |= (y & inf) == inf || (y >> 16 & inf) == inf;
            }
          }
        // A product 0 * inf of a column that does not see the token must not reach it: such blocks go token by token.
        const bool slow = __any_sync(0xffffffffu, odd) && total - 1 > first_limit;
#pragma unroll 1
        for (int only = slow ? 0 : kBlockTokens; only <= kBlockTokens; ++only) {
          if (slow && only == kBlockTokens) break;
#pragma unroll
          for (int j = 0; j < J; ++j) {
            uint32_t A[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {            // row g: dim 4 g + 2 (j % 2), row g + 8: the next; k 2t.. : tokens 0, 1 then 2, 3
              uint32_t lo = j % 2 ? x[j / 2][e / 2 * 2].y : x[j / 2][e / 2 * 2].x;
              uint32_t hi = j % 2 ? x[j / 2][e / 2 * 2 + 1].y : x[j / 2][e / 2 * 2 + 1].x;
              if (slow) {
                if (only != 4 * t + e / 2 * 2) lo = 0;
                if (only != 4 * t + e / 2 * 2 + 1) hi = 0;
              }
              A[e] = __byte_perm(lo, hi, e % 2 ? 0x7632 : 0x5410);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float acc[4] = {0.f, 0.f, 0.f, 0.f};
              mma16816<kBf16>(acc, A, pt[n][0], pt[n][1]);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (!slow || base + only <= limit[n][e % 2]) o[j][n][e] += acc[e];
            }
          }
        }
      }
    }

    // ---- the segment's output, or this warp's part of it
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], w);
    if (u0 == 0 && u1 == units) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int c = c0 + n * 8 + 2 * t + e;
          if (c >= a.T * a.G) continue;
          float f = m[n][e] == -INFINITY ? 0.f : a.softmax ? 1.f / l[n][e] : attn_ex2(m[n][e] - qsq[n][e]);
          const bool none = c / a.G >= span.fresh || m[n][e] == -INFINITY && l[n][e] == 0.f;
          uint16_t* out = static_cast<uint16_t*>(a.out) + out_offset(a, b, h, c);
#pragma unroll
          for (int i = 0; i < KC; ++i) {
            const int d = 32 * i + 4 * g;
            if (d >= a.D) continue;
            uint2 y = make_uint2(pack2<kBf16>(o[2 * i][n][e] * f, o[2 * i][n][2 + e] * f),
                                 pack2<kBf16>(o[2 * i + 1][n][e] * f, o[2 * i + 1][n][2 + e] * f));
            if (none) y = make_uint2(0, 0);
            *reinterpret_cast<uint2*>(out + d) = y;
          }
        }
    } else {
      float* part = part_of<P, NT>(a, 2 * self + (u0 == 0));
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int c = n * 8 + 2 * t + e;
          if (c0 + c >= a.T * a.G) continue;
#pragma unroll
          for (int i = 0; i < KC; ++i)
            *reinterpret_cast<float4*>(part + c * P + 32 * i + 4 * g) =
                make_float4(o[2 * i][n][e], o[2 * i][n][2 + e], o[2 * i + 1][n][e], o[2 * i + 1][n][2 + e]);
          if (g == 0) {
            part[8 * NT * P + c] = m[n][e];
            part[8 * NT * (P + 1) + c] = l[n][e];
          }
        }
    }
    pos += u1 - u0;
  }
  grid_dependents_launch();
}

constexpr int kJoinThreads = 128;

// One block per segment joins the parts of segments that several warps worked on, and clears those that no warp did.
template <bool kBf16, int P, int NT>
__global__ void __launch_bounds__(kJoinThreads) cache_join_kernel(const CacheAttnArgs a, const int64_t workers) {
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int segments = a.column_tiles * a.H;
  const int b = blockIdx.x / segments, seg = blockIdx.x % segments;
  const int h = seg % a.H, c0 = seg / a.H * (8 * NT);
  const CacheSpan span = cache_span(a.lengths, a.fresh, b, a.T, a.max_pages);
  const int units = segment_units<P>(a, b);
  const int columns = min(8 * NT, a.T * a.G - c0);
  uint16_t* out = static_cast<uint16_t*>(a.out);
  constexpr int kPer = P / 32;
  int64_t first = 0, last = 0;
  if (units > 0) {
    const Deal deal(units_before<P>(a, a.B) * segments, workers);
    const int64_t begin = units_before<P>(a, b) * segments + static_cast<int64_t>(seg) * units;
    first = min(deal.worker(begin), workers - 1);
    last = min(deal.worker(begin + units - 1), workers - 1);
    if (first == last) return;
  }
  for (int c = warp; c < columns; c += kJoinThreads / 32) {
    float y[kPer] = {};
    if (units > 0 && (c0 + c) / a.G < span.fresh) {
      float top = -INFINITY;
      for (int64_t w = first + lane; w <= last; w += 32)
        top = fmaxf(top, part_of<P, NT>(a, 2 * w + (w == first))[8 * NT * P + c]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float ref = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
#pragma unroll 4
      for (int64_t w = first; w <= last; ++w) {
        const float* part = part_of<P, NT>(a, 2 * w + (w == first));
        const float f = attn_ex2(part[8 * NT * P + c] - ref);
        sum = fmaf(part[8 * NT * (P + 1) + c], f, sum);
#pragma unroll
        for (int i = 0; i < kPer; ++i) y[i] = fmaf(part[c * P + lane * kPer + i], f, y[i]);
      }
      float f = 1.f / sum;
      if (!a.softmax) {
        const int col = c0 + c;
        const uint16_t* q = static_cast<const uint16_t*>(a.q) + b * a.qs[0] + (h * a.G + col % a.G) * a.qs[1] + col / a.G * a.qs[2];
        float sq = 0.f;
        for (int d = lane * 2; d < a.D; d += 64) {
          const float2 x = unpack2<kBf16>(*reinterpret_cast<const uint32_t*>(q + d));
          sq = fmaf(x.x, x.x, fmaf(x.y, x.y, sq));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
        f = attn_ex2(ref - a.scale * sq);
      }
      const bool none = top == -INFINITY && sum == 0.f;
#pragma unroll
      for (int i = 0; i < kPer; ++i) y[i] = none ? 0.f : y[i] * f;
    }
    uint16_t* to = out + out_offset(a, b, h, c0 + c) + lane * kPer;
    if (lane * kPer < a.D) {
#pragma unroll
      for (int i = 0; i < kPer; i += 2) *reinterpret_cast<uint32_t*>(to + i) = pack2<kBf16>(y[i], y[i + 1]);
    }
  }
}

template <bool kBf16, int P, int NT>
cudaError_t attn_t(const CacheAttnArgs& a, int sms, cudaStream_t stream) {
  cache_attn_kernel<kBf16, P, NT><<<sms, kAttnWarps * 32, 0, stream>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int64_t blocks = static_cast<int64_t>(a.B) * a.column_tiles * a.H;
  return launch_dependent(cache_join_kernel<kBf16, P, NT>, dim3(static_cast<unsigned>(blocks)), kJoinThreads, 0, stream, a,
                          static_cast<int64_t>(sms) * kAttnWarps);
}

template <bool kBf16, int P>
cudaError_t attn_p(const CacheAttnArgs& a, int sms, cudaStream_t stream) {
  return cache_attn_tiles(a.T, a.G, P) == 1 ? attn_t<kBf16, P, 1>(a, sms, stream) : attn_t<kBf16, P, 256 / P>(a, sms, stream);
}

}  // namespace

// Operand tiles of 8 columns that a warp works on at a time: as many as its registers hold where there is more than one.
int cache_attn_tiles(int T, int G, int P) { return static_cast<int64_t>(T) * G <= 8 ? 1 : 256 / P; }

size_t cache_attn_workspace_bytes(int T, int G, int D, int sms) {
  const int P = cache_columns(D);
  return static_cast<size_t>(sms) * kAttnWarps * 2 * 8 * cache_attn_tiles(T, G, P) * (P + 2) * sizeof(float);
}

cudaError_t launch_cache_attn(CacheAttnArgs a, bool bf16, int sms, cudaStream_t stream) {
  if (a.B == 0 || a.T == 0) return cudaSuccess;
  const int64_t columns = 8 * cache_attn_tiles(a.T, a.G, cache_columns(a.D)), tiles = (static_cast<int64_t>(a.T) * a.G + columns - 1) / columns;
  if (tiles * a.H * a.B > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  a.column_tiles = static_cast<int>(tiles);
  if (cache_columns(a.D) == 64) return bf16 ? attn_p<true, 64>(a, sms, stream) : attn_p<false, 64>(a, sms, stream);
  return bf16 ? attn_p<true, 128>(a, sms, stream) : attn_p<false, 128>(a, sms, stream);
}

}  // namespace rbf
