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
constexpr int kStages = 3;                         // units of a warp that are loaded ahead, the current one among them
constexpr float kSlack = 8.f;                      // growth of a score, in powers of two, that does not move the maximum

template <int P>
struct Tile {
  static constexpr int kUnitBlocks = 256 / P;      // blocks of one load: 8 KB of codes
  static constexpr int kUnit = kUnitBlocks * kBlockTokens;
  static constexpr int kChunks = P / 32;           // 16-byte words of a lane per block and operand
  static constexpr int kDims = P / 16;             // 16-row tiles of the output
  static constexpr int kScales = 8192;             // a stage: codes or an incomplete block, the scales, whether there is a page
  static constexpr int kFlag = kScales + 48;
  static constexpr int kStage = kScales + 64;
};

__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_close() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// The warp's copies up to the `kLeft` last groups have arrived; after it, every lane sees every lane's.
template <int kLeft>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
  __syncwarp();
}

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

// A segment's units: groups of complete blocks, then the incomplete block
template <int P>
struct Units {
  int held, fresh, groups, count;
  __device__ Units(const CacheAttnArgs& a, int b) {
    const CacheSpan s = cache_span(a.lengths, a.fresh, b, a.T, a.max_pages);
    held = s.held;
    fresh = s.fresh;
    const int total = held + fresh;
    groups = fresh == 0 ? 0 : (total / kBlockTokens + Tile<P>::kUnitBlocks - 1) / Tile<P>::kUnitBlocks;
    count = groups + (fresh != 0 && total % kBlockTokens != 0);
  }
};

// Sums over sequences [0, n) and over all of the units of a segment, by a whole warp
template <int P>
__device__ __forceinline__ void sum_units(const CacheAttnArgs& a, int n, int64_t& before, int64_t& all) {
  before = all = 0;
  for (int b = threadIdx.x & 31; b < a.B; b += 32) {
    const int u = Units<P>(a, b).count;
    all += u;
    if (b < n) before += u;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    all += __shfl_xor_sync(0xffffffffu, all, o);
  }
}

// Element offset of output column c of a segment (new token c / G of query head h * G + c % G)
__device__ __forceinline__ int64_t out_offset(const CacheAttnArgs& a, int b, int h, int c) {
  return ((static_cast<int64_t>(b) * a.H * a.G + h * a.G + c % a.G) * a.T + c / a.G) * a.D;
}
__device__ __forceinline__ const uint16_t* q_row(const CacheAttnArgs& a, int b, int h, int c) {
  return static_cast<const uint16_t*>(a.q) + b * a.qs[0] + (h * a.G + c % a.G) * a.qs[1] + c / a.G * a.qs[2];
}

// One part: per column P outputs, then the maxima and the sums of all columns
template <int P, int NT>
__device__ __forceinline__ float* part_of(const CacheAttnArgs& a, int64_t index) {
  return a.parts + index * (8 * NT) * (P + 2);
}

// A warp's state for one segment
template <int P, int NT>
struct Running {
  float o[Tile<P>::kDims][NT][4];                  // tile j: dims 32 (j / 2) + 4 g + 2 (j % 2), + 1 of columns 2t, 2t + 1
  float m[NT][2], l[NT][2];                        // of columns 8n + 2t, + 1; l: this lane's share
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < Tile<P>::kDims; ++j)
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
  }
  // The maximum moves only if a score exceeds it by more than the slack; s becomes the weights, l their sum.
  template <int kBlocks>
  __device__ __forceinline__ void weigh(float (&s)[kBlocks][NT][4]) {
    float top[NT][2];
    bool over = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        top[n][e] = fmaxf(s[0][n][e], s[0][n][2 + e]);
#pragma unroll
        for (int k = 1; k < kBlocks; ++k) top[n][e] = fmaxf(top[n][e], fmaxf(s[k][n][e], s[k][n][2 + e]));
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
          for (int j = 0; j < Tile<P>::kDims; ++j) {
            o[j][n][e] *= f;
            o[j][n][2 + e] *= f;
          }
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float ref[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) ref[e] = m[n][e] == -INFINITY ? 0.f : m[n][e];      // no token seen yet
#pragma unroll
      for (int k = 0; k < kBlocks; ++k) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[k][n][e] = attn_ex2(s[k][n][e] - ref[e % 2]);
        l[n][0] += s[k][n][0] + s[k][n][2];
        l[n][1] += s[k][n][1] + s[k][n][3];
      }
    }
  }
};

template <bool kBf16, int P, int NT>
__global__ void __launch_bounds__(kAttnWarps * 32) cache_attn_kernel(const CacheAttnArgs a) {
  using T = Tile<P>;
  constexpr int UB = T::kUnitBlocks, KC = T::kChunks, J = T::kDims;
  constexpr int kSlot = cache_slot_bytes(P), kBytes = cache_page_bytes(P);
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + (threadIdx.x >> 5) * (kStages * T::kStage);       // a warp has its own
  const int64_t workers = static_cast<int64_t>(gridDim.x) * kAttnWarps;
  const int64_t self = static_cast<int64_t>(threadIdx.x >> 5) * gridDim.x + blockIdx.x;    // neighbours on other SMs
  const int segments = a.column_tiles * a.H;       // of a sequence
  int64_t unused, all;
  sum_units<P>(a, 0, unused, all);
  const Deal deal(all * segments, workers);
  int64_t pos = deal.begin(self);
  const int64_t stop = deal.begin(self + 1);
  if (pos >= stop) return;

  // the sequence of the first unit
  int b = 0;
  int64_t seq_begin = 0;
  for (; b < a.B; b += 32) {
    const int64_t mine = b + lane < a.B ? static_cast<int64_t>(Units<P>(a, b + lane).count) * segments : 0;
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

  // ---- loads: lane i looks up the i-th of the next 32 units, so that page numbers are waited for once in 32 units
  struct Lookup {
    const uint8_t* base;                           // of the head's page, null where there is nothing to load
    int what;                                      // complete blocks: first in the page | count << 8; incomplete: tokens | 1 << 16
  };
  int look_b = b;                                  // this lane's sequence
  int64_t look_begin = seq_begin;
  auto look_up = [&](int64_t x) {
    Lookup r{nullptr, 0};
    while (x < stop && look_b < a.B) {
      const Units<P> units(a, look_b);
      const int64_t span = static_cast<int64_t>(units.count) * segments;
      if (x >= look_begin + span) {
        look_begin += span;
        ++look_b;
        continue;
      }
      const int64_t in = x - look_begin;
      const int u = static_cast<int>(in % units.count), h = static_cast<int>(in / units.count % a.H);
      const int total = units.held + units.fresh, blocks = total / kBlockTokens;
      const int first = u < units.groups ? u * UB : blocks;
      r.base = cache_page(a.pages, a.table, look_b, a.max_pages, a.num_pages, a.H, h, kBytes, first * kBlockTokens);
      r.what = u < units.groups ? first % kPageBlocks | min(UB, blocks - first) << 8 : total % kBlockTokens | 1 << 16;
      break;
    }
    return r;
  };
  Lookup now = look_up(pos + lane), next = look_up(pos + 32 + lane);
  int64_t fetched = 0;                             // units asked for
  const int64_t mine = stop - pos;
  auto fetch = [&]() {
    if (fetched < mine) {
      const int from = static_cast<int>(fetched & 31);
      if (from == 0 && fetched != 0) {
        now = next;
        next = look_up(pos + fetched + 32 + lane);
      }
      const uint64_t base64 = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(now.base), from);
      const int what = __shfl_sync(0xffffffffu, now.what, from);
      const uint8_t* base = reinterpret_cast<const uint8_t*>(base64);
      uint8_t* stage = ring + static_cast<int>(fetched % kStages) * T::kStage;
      const uint32_t to = smem_u32(stage);
      if (lane == 0) *reinterpret_cast<int*>(stage + T::kFlag) = base != nullptr;
      if (base != nullptr) {
        if (what >> 16) {
          const uint8_t* src = base + kPageHeader + kPageBlocks * kSlot + lane * 16;
#pragma unroll
          for (int i = 0; i < 2 * kSlot / 512; ++i)          // keys, then values
            if ((i % (kSlot / 512) * 512 + lane * 16) / (2 * P) < (what & 0xff)) copy16(to + i * 512 + lane * 16, src + i * 512);
        } else {
          const uint8_t* src = base + kPageHeader + (what & 0xff) * kSlot + lane * 16;
          const int bytes = (what >> 8) * kSlot;
          if (bytes == UB * kSlot) {
#pragma unroll
            for (int i = 0; i < UB * kSlot / 512; ++i) copy16(to + i * 512 + lane * 16, src + i * 512);
          } else {
#pragma unroll
            for (int i = 0; i < UB * kSlot / 512; ++i)
              if (i * 512 < bytes) copy16(to + i * 512 + lane * 16, src + i * 512);
          }
          if (lane < UB / 2) copy16(to + T::kScales + lane * 16, base + (what & 0xff) * 8 + lane * 16);
        }
      }
      ++fetched;
    }
    copies_close();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch();

  int64_t taken = 0;                               // units worked on
  int64_t at = pos;
  while (at < stop && b < a.B) {
    const Units<P> units(a, b);
    if (at >= seq_begin + static_cast<int64_t>(units.count) * segments) {  // on to the next sequence (some have no units)
      seq_begin += static_cast<int64_t>(units.count) * segments;
      ++b;
      continue;
    }
    const int total = units.held + units.fresh;
    const int seg = static_cast<int>((at - seq_begin) / units.count);
    const int u0 = static_cast<int>((at - seq_begin) % units.count);
    const int64_t left = stop - at;
    const int u1 = left < units.count - u0 ? u0 + static_cast<int>(left) : units.count;
    const int h = seg % a.H, c0 = seg / a.H * (8 * NT);

    // ---- queries: operand columns, their scales, and how far each column sees
    uint32_t qh[NT][P / 16][2];                      // fp16, scaled
    float qmul[NT][2], qsq[NT][2];                   // of columns 2t, 2t + 1
    int limit[NT][2];                                // last token that the column sees
    // operand words of column n * 8 + g as they are in memory: k step i has dims 64 (i / 4) + 16 t + 4 (i % 4) ... + 3
    auto load_q = [&](int n, uint32_t (&w)[P / 16][2]) {
      const int c = c0 + n * 8 + g;
      const bool real = c < a.T * a.G;
      const uint16_t* q = q_row(a, b, h, real ? c : 0);
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
        limit[n][e] = c2 < a.T * a.G ? units.held + c2 / a.G : total - 1;
      }
    }
    const int first_limit = units.held + c0 / a.G;   // every column of the tile sees at least this far,
    const int last_limit = units.held + (c0 + 8 * NT - 1) / a.G;           // and none further than this

    Running<P, NT> run;
    run.clear();
    for (int u = u0; u < u1; ++u) {
      const uint8_t* stage = ring + static_cast<int>(taken % kStages) * T::kStage;
      copies_wait<kStages - 2>();
      fetch();
      ++taken;
      if (*reinterpret_cast<const int*>(stage + T::kFlag) == 0) continue;  // a page outside the pool: its tokens are absent
      if (u < units.groups) {
        // ================================================================ complete blocks
        const int begin = u * T::kUnit;              // first token
        if (begin > last_limit) continue;
        const int whole = min(UB, total / kBlockTokens - begin / kBlockTokens);
        const bool hidden = begin + T::kUnit - 1 > first_limit;
        const float2* scales = reinterpret_cast<const float2*>(stage + T::kScales);
        float s[UB][NT][4];
#pragma unroll
        for (int k = 0; k < UB; ++k) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[k][n][e] = -INFINITY;
          if (k >= whole) continue;
          const float scale = scales[k].x;
          const uint4* key = reinterpret_cast<const uint4*>(stage + k * kSlot) + lane;
          int sq0 = 0, sq1 = 0;
          float acc[NT][4];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
#pragma unroll
          for (int d = 0; d < P / 64; ++d) {
            const uint4 w0 = key[2 * d * 32], w1 = key[(2 * d + 1) * 32];
            const uint32_t r0[4] = {w0.x, w0.y, w0.z, w0.w}, r1[4] = {w1.x, w1.y, w1.z, w1.w};
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
          const float bias = a.scale * scale * scale;
          const float b0 = bias * static_cast<float>(sq0), b1 = bias * static_cast<float>(sq1);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float mul = qmul[n][e] * scale;
              s[k][n][e] = fmaf(acc[n][e], mul, -b0);
              s[k][n][2 + e] = fmaf(acc[n][2 + e], mul, -b1);
            }
          }
          if (hidden) {
            const int tok = begin + k * kBlockTokens + 4 * (g >> 1) + (g & 1);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (tok + 2 * (e / 2) > limit[n][e % 2]) s[k][n][e] = -INFINITY;
          }
        }
        run.weigh(s);
#pragma unroll
        for (int k = 0; k < UB; ++k) {
          if (k >= whole) continue;
          uint32_t p[NT][2];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            p[n][0] = transpose8(pack2<false>(s[k][n][0], s[k][n][1]));
            p[n][1] = transpose8(pack2<false>(s[k][n][2], s[k][n][3]));
          }
          const uint4* value = reinterpret_cast<const uint4*>(stage + k * kSlot + 16 * P) + lane;
          const float scale = scales[k].y;
          const bool finite = fabsf(scale) < INFINITY;
          const int base = begin + k * kBlockTokens;
#pragma unroll
          for (int i = 0; i < KC; ++i) {
            const uint4 w = value[i * 32];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t r0 = half ? w.z : w.x, r1 = half ? w.w : w.y;
              const uint32_t A[4] = {codes_lo(r0), codes_lo(r1), codes_hi(r0), codes_hi(r1)};
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                float acc[4] = {0.f, 0.f, 0.f, 0.f};
                mma16816<false>(acc, A, p[n][0], p[n][1]);
                float(&o)[4] = run.o[2 * i + half][n];
#pragma unroll
                for (int e = 0; e < 4; ++e)           // a block that is not finite reaches the columns that see it
                  if (finite || base <= limit[n][e % 2]) o[e] = fmaf(acc[e], scale, o[e]);
              }
            }
          }
        }
      } else {
        // ================================================================ the incomplete block, in 16 bits
        const int base = total / kBlockTokens * kBlockTokens, tok = 4 * (g >> 1) + (g & 1);
        if (base > last_limit) continue;
        const uint16_t* keys = reinterpret_cast<const uint16_t*>(stage);
        const uint16_t* values = keys + kSlot / 2;
        float s[1][NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[0][n][e] = 0.f;
        float sq[2] = {0.f, 0.f};
        uint32_t qt[NT][P / 16][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) load_q(n, qt[n]);
#pragma unroll
        for (int d = 0; d < P / 64; ++d) {
          uint32_t r[2][8];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const bool row_there = base + tok + 2 * half < total;
            const uint4* row = reinterpret_cast<const uint4*>(keys + (tok + 2 * half) * P + d * 64 + t * 16);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint4 x = row_there ? row[e] : make_uint4(0, 0, 0, 0);
              r[half][4 * e] = x.x;
              r[half][4 * e + 1] = x.y;
              r[half][4 * e + 2] = x.z;
              r[half][4 * e + 3] = x.w;
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
            for (int n = 0; n < NT; ++n) mma16816<kBf16>(s[0][n], A, qt[n][d * 4 + i][0], qt[n][d * 4 + i][1]);
          }
        }
#pragma unroll
        for (int x = 1; x < 4; x <<= 1) {
          sq[0] += __shfl_xor_sync(0xffffffffu, sq[0], x);
          sq[1] += __shfl_xor_sync(0xffffffffu, sq[1], x);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int token = base + tok + 2 * (e / 2);
            s[0][n][e] = token <= limit[n][e % 2] && token < total ? fmaf(s[0][n][e], 2.f * a.scale, -a.scale * sq[e / 2]) : -INFINITY;
          }
        run.weigh(s);
        uint32_t p[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          p[n][0] = transpose8(pack2<kBf16>(s[0][n][0], s[0][n][1]));
          p[n][1] = transpose8(pack2<kBf16>(s[0][n][2], s[0][n][3]));
        }
        uint2 x[KC][4];                              // dims 32 i + 4 g ... + 3 of tokens 4 t + r
        bool odd = false;                            // a value that is not finite
#pragma unroll
        for (int i = 0; i < KC; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            x[i][r] = make_uint2(0, 0);
            if (base + 4 * t + r < total) x[i][r] = *reinterpret_cast<const uint2*>(values + (4 * t + r) * P + 32 * i + 4 * g);
            constexpr uint32_t kInf = kBf16 ? 0x7f80u : 0x7c00u;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t y = half ? x[i][r].y : x[i][r].x;
              odd |= (y & kInf) == kInf || (y >> 16 & kInf) == kInf;
            }
          }
        // A product 0 * inf of a column that does not see the token must not reach it: such blocks go token by token.
        const bool slow = __any_sync(0xffffffffu, odd) && total - 1 > first_limit;
#pragma unroll 1
        for (int only = slow ? 0 : kBlockTokens - 1; only < kBlockTokens; ++only) {
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
              mma16816<kBf16>(acc, A, p[n][0], p[n][1]);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (!slow || base + only <= limit[n][e % 2]) run.o[j][n][e] += acc[e];
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
        for (int w = 4; w < 32; w <<= 1) run.l[n][e] += __shfl_xor_sync(0xffffffffu, run.l[n][e], w);
    const bool complete = u0 == 0 && u1 == units.count;
    float* part = part_of<P, NT>(a, 2 * self + (u0 == 0));
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int in = n * 8 + 2 * t + e, c = c0 + in;
        if (c >= a.T * a.G) continue;
        const float m = run.m[n][e], l = run.l[n][e];
        if (complete) {
          const float f = m == -INFINITY ? 0.f : a.softmax ? 1.f / l : attn_ex2(m - qsq[n][e]);
          const bool none = c / a.G >= units.fresh || (m == -INFINITY && l == 0.f);
          uint16_t* out = static_cast<uint16_t*>(a.out) + out_offset(a, b, h, c);
#pragma unroll
          for (int i = 0; i < KC; ++i) {
            const int d = 32 * i + 4 * g;
            if (d >= a.D) continue;
            uint2 y = make_uint2(pack2<kBf16>(run.o[2 * i][n][e] * f, run.o[2 * i][n][2 + e] * f),
                                 pack2<kBf16>(run.o[2 * i + 1][n][e] * f, run.o[2 * i + 1][n][2 + e] * f));
            if (none) y = make_uint2(0, 0);
            *reinterpret_cast<uint2*>(out + d) = y;
          }
        } else {
#pragma unroll
          for (int i = 0; i < KC; ++i)
            *reinterpret_cast<float4*>(part + in * P + 32 * i + 4 * g) =
                make_float4(run.o[2 * i][n][e], run.o[2 * i][n][2 + e], run.o[2 * i + 1][n][e], run.o[2 * i + 1][n][2 + e]);
          if (g == 0) {
            part[8 * NT * P + in] = m;
            part[8 * NT * (P + 1) + in] = l;
          }
        }
      }
    at += u1 - u0;
  }
  grid_dependents_launch();
}

constexpr int kJoinWarps = 8;

// Joins the parts of the segments that several warps worked on, and clears those that no warp did: `split` warps of a block
// share the parts of a column, 8 where there are few columns (and many parts of each), else one.
template <bool kBf16, int P, int NT>
__global__ void __launch_bounds__(kJoinWarps * 32) cache_join_kernel(const CacheAttnArgs a, const int64_t workers, const int split) {
  __shared__ float s_y[kJoinWarps][P], s_m[kJoinWarps], s_l[kJoinWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int segments = a.column_tiles * a.H, width = min(8 * NT, a.T * a.G);
  const int64_t column = static_cast<int64_t>(blockIdx.x) * (kJoinWarps / split) + warp / split;
  const int64_t segment = column / width;
  const int in = static_cast<int>(column % width), share = warp % split;
  const int b = static_cast<int>(segment / segments), seg = static_cast<int>(segment % segments);
  const int h = seg % a.H, c = seg / a.H * (8 * NT) + in;
  grid_dependency_wait();
  constexpr int kPer = P / 32;
  float y[kPer] = {}, top = -INFINITY, sum = 0.f;
  bool write = b < a.B && c < a.T * a.G, some = false;
  if (write) {
    const Units<P> units(a, b);
    if (units.count > 0) {
      int64_t before, all;
      sum_units<P>(a, b, before, all);
      const Deal deal(all * segments, workers);
      const int64_t begin = before * segments + static_cast<int64_t>(seg) * units.count;
      const int64_t first = min(deal.worker(begin), workers - 1), last = min(deal.worker(begin + units.count - 1), workers - 1);
      write = first != last;
      some = write && c / a.G < units.fresh;
      if (some) {
        for (int64_t w0 = first + share * 32; w0 <= last; w0 += 32 * split) {
          const int n = static_cast<int>(min(last - w0 + 1, int64_t{32}));
          float m = -INFINITY, l = 0.f;
          if (lane < n) {
            const float* part = part_of<P, NT>(a, 2 * (w0 + lane) + (w0 + lane == first));
            m = part[8 * NT * P + in];
            l = part[8 * NT * (P + 1) + in];
          }
          float x = m;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
          x = fmaxf(x, top);
          const float ref = x == -INFINITY ? 0.f : x, f = attn_ex2(m - ref), old = attn_ex2(top - ref);
          top = x;
          l *= f;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
          sum = fmaf(sum, old, l);
#pragma unroll
          for (int i = 0; i < kPer; ++i) y[i] *= old;
#pragma unroll 8
          for (int j = 0; j < n; ++j) {
            const float* part = part_of<P, NT>(a, 2 * (w0 + j) + (w0 + j == first)) + in * P + lane * kPer;
            const float fj = __shfl_sync(0xffffffffu, f, j);
#pragma unroll
            for (int i = 0; i < kPer; ++i) y[i] = fmaf(part[i], fj, y[i]);
          }
        }
      }
    }
  }
  if (split > 1) {                                 // the whole block has one column
#pragma unroll
    for (int i = 0; i < kPer; ++i) s_y[warp][lane * kPer + i] = y[i];
    if (lane == 0) {
      s_m[warp] = top;
      s_l[warp] = sum;
    }
    __syncthreads();
    if (warp != 0) return;
    for (int w = 1; w < kJoinWarps; ++w) {
      const float x = fmaxf(top, s_m[w]), ref = x == -INFINITY ? 0.f : x;
      const float f0 = attn_ex2(top - ref), f1 = attn_ex2(s_m[w] - ref);
      top = x;
      sum = sum * f0 + s_l[w] * f1;
#pragma unroll
      for (int i = 0; i < kPer; ++i) y[i] = y[i] * f0 + s_y[w][lane * kPer + i] * f1;
    }
  }
  if (!write) return;
  if (some) {
    float f = 1.f / sum;
    if (!a.softmax) {
      const uint16_t* q = q_row(a, b, h, c);
      float sq = 0.f;
      for (int d = lane * 2; d < a.D; d += 64) {
        const float2 x = unpack2<kBf16>(*reinterpret_cast<const uint32_t*>(q + d));
        sq = fmaf(x.x, x.x, fmaf(x.y, x.y, sq));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
      f = attn_ex2((top == -INFINITY ? 0.f : top) - a.scale * sq);
    }
    if (top == -INFINITY && sum == 0.f) f = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) y[i] *= f;
  }
  if (lane * kPer >= a.D) return;
  uint16_t* to = static_cast<uint16_t*>(a.out) + out_offset(a, b, h, c) + lane * kPer;
#pragma unroll
  for (int i = 0; i < kPer; i += 2) *reinterpret_cast<uint32_t*>(to + i) = pack2<kBf16>(y[i], y[i + 1]);
}

template <bool kBf16, int P, int NT>
cudaError_t attn_t(const CacheAttnArgs& a, int sms, cudaStream_t stream) {
  constexpr int kSmem = kAttnWarps * kStages * Tile<P>::kStage;
  static PerDeviceFlags flags;
  cudaError_t e = ensure_dynamic_smem(cache_attn_kernel<kBf16, P, NT>, kSmem, flags);
  if (e != cudaSuccess) return e;
  cache_attn_kernel<kBf16, P, NT><<<sms, kAttnWarps * 32, kSmem, stream>>>(a);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  const int64_t width = static_cast<int64_t>(a.T) * a.G < 8 * NT ? a.T * a.G : 8 * NT;
  const int64_t columns = static_cast<int64_t>(a.B) * a.column_tiles * a.H * width;
  const int split = columns <= sms * 4 ? kJoinWarps : 1;
  const int64_t blocks = (columns + kJoinWarps / split - 1) / (kJoinWarps / split);
  return launch_dependent(cache_join_kernel<kBf16, P, NT>, dim3(static_cast<unsigned>(blocks)), kJoinWarps * 32, 0, stream, a,
                          static_cast<int64_t>(sms) * kAttnWarps, split);
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
  if (tiles * columns * a.H * a.B > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  a.column_tiles = static_cast<int>(tiles);
  if (cache_columns(a.D) == 64) return bf16 ? attn_p<true, 64>(a, sms, stream) : attn_p<false, 64>(a, sms, stream);
  return bf16 ? attn_p<true, 128>(a, sms, stream) : attn_p<false, 128>(a, sms, stream);
}

}  // namespace rbf
