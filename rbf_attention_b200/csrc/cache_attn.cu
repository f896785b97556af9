// RBF attention of new tokens over the paged 8-bit cache (cache.cuh): softmax(2 g q.k - g |k|^2) V, or exp(-g |q - k|^2) V
// without the denominator, for tokens 0 .. held + i of a sequence as seen by its i-th new token.
//
// A step of generation reads the whole cache once and does two products per byte: the roofline is HBM, and what has to be cheap
// is making 16-bit operands of the bytes. So the products are mma.m16n8k16 with the *cache* as the 16-row operand (tokens of a
// block, then dims) and the queries - the new tokens of the query heads that share a key/value head - as the 8 columns, and a
// lane's bytes lie in the cache in the order in which the instruction wants them. A code becomes an exact fp16 number in one
// permute (the byte under 0x64 is 1024 + byte) and one subtraction, for two values. Scales stay outside: a block's scores are
// multiplied by its key scale in fp32, its weights by its value scale (see Running::refer). |k|^2 is the integer sum of the
// codes' squares.
//   S^T (16 tokens x 8 columns) = K Q^T,  P^T by exponentials in fp32,  O^T (16 dims x 8 columns) += V^T P^T
// Queries are multiplied by the power of two that brings their largest element to [1, 2) and rounded to fp16: exact for every
// element within 2^-14 of the largest in 16-bit types, off by 2^-25 of it below. P is rounded to fp16 (2^-11 of it), as the operand
// that the codes' products take; the sum that the outputs are divided by is of the weights in fp32, so that a row's roundings
// average out instead of moving its denominator with them. The exponentials are ex2.approx, two units of fp32 off. The block that is not
// complete yet is held in 16 bits and multiplied in its own type, P with it: of bfloat16 2^-8 of the weights of at most 15
// tokens, which is the output's own rounding, where fp16 operands would need the values scaled (the kernel for many
// columns, whose operands all are fp16, does that).
//
// Three kernels share this. Long sequences: work is split evenly whatever the lengths, all (sequence, head) segments in a row,
// cut into units of one load, are dealt to the warps of one wave in contiguous ranges. A warp works by itself - no barrier - with
// a running maximum (moved only when a score exceeds it by 2^8, which keeps P below 2^8) and writes its segment's output, or its
// part (unnormalised output, maximum, sum) where the segment is shared with other warps; a second kernel joins the parts in the
// order of the tokens. Joining a block's warps at the end of each segment instead, so that a segment has fewer parts, took 5 to 8
// us longer: the warps wait for the slowest. Short sequences: a segment per block or cluster, one launch. More than 8 columns:
// see cache_attn_rows_kernel.
//
// Bounds, one B200: 16 sequences of up to 32768 tokens, 8 key heads of 128, 32 query heads (549 MB): 100 us a call, the first
// kernel 93 us at 5.9 TB/s = 90 % of the copy bandwidth. 64 sequences of up to 1028 tokens, 8 heads of 64 (35.5 MB, 5.4 us at
// that bandwidth): 16.4 us, of which the chain of launch, lengths, pages, codes and join is the larger part.
#include <cstdint>
#include <cuda_runtime.h>

#include <type_traits>

#include "cache.cuh"
#include "launch.h"

namespace rbf {
namespace {

// Up to 8 columns: warps of a block (one per SM), blocks of a unit, and units of a warp that are loaded ahead, the current one
// among them: what registers (65536) and shared memory (227 KB) hold with 8 KB units. 16 x 32768 tokens of 128 columns took 115
// us with 8 warps and three units, 104 so; 8 x 16384 of 64 columns 36 and 33.5 us, with 16 warps and three units of 4 KB 35.5.
constexpr int kWarpsOf8 = 12, kStagesOf8 = 2;
template <int P> constexpr int kUnitBlocks = 256 / P;
constexpr int kShortWarps = 8;                     // of the kernel for short sequences, 4 where there are many
constexpr float kSlack = 8.f;                      // growth of a score, in powers of two, that does not move the maximum

// A warp's unit of work: UB blocks that are complete, or the one that is not
template <int P, int UB>
struct Tile {
  static constexpr int kUnit = UB * kBlockTokens;
  static constexpr int kBytes = (UB > 2 ? UB : 2) * cache_slot_bytes(P);
  static constexpr int kScales = kBytes;           // a stage: the rows, the scales, whether there is a page
  static constexpr int kFlag = kScales + 48;
  static constexpr int kStage = kScales + 64;
  static_assert(UB == 2 || UB == 4, "scales are loaded 16 bytes at a time into 32");
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
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}
// 8 x 8 16-bit matrix, row lane / 4 and columns 2 (lane % 4), + 1 in each lane, transposed
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Bytes 0, 1 (2, 3) of a word of codes as two fp16 numbers. `exponents` is 0x64 in every byte, from the kernel's arguments: of a
// constant that it knows the compiler makes a move before almost every permute (43 for 64).
__device__ __forceinline__ uint32_t codes_lo(uint32_t w, uint32_t exponents) {
  const uint32_t x = __byte_perm(w, exponents, 0x4140);
  const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&y);
}
__device__ __forceinline__ uint32_t codes_hi(uint32_t w, uint32_t exponents) {
  const uint32_t x = __byte_perm(w, exponents, 0x4342);
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
template <int UB>
struct Units {
  int held, fresh, groups, count;
  __device__ Units(const CacheAttnArgs& a, int b) {
    const CacheSpan s = cache_span(a.lengths, a.fresh, b, a.T, a.max_pages);
    held = s.held;
    fresh = s.fresh;
    const int total = held + fresh;
    groups = fresh == 0 ? 0 : (total / kBlockTokens + UB - 1) / UB;
    count = groups + (fresh != 0 && total % kBlockTokens != 0);
  }
};

// Groups of blocks, the incomplete one among them
template <int UB>
struct AllUnits {
  int held, fresh, count;
  __device__ AllUnits(const CacheAttnArgs& a, int b) {
    const CacheSpan s = cache_span(a.lengths, a.fresh, b, a.T, a.max_pages);
    held = s.held;
    fresh = s.fresh;
    count = fresh == 0 ? 0 : (held + fresh + UB * kBlockTokens - 1) / (UB * kBlockTokens);
  }
};

// Sum over the sequences of the units of a segment, by a whole warp
template <class U>
__device__ __forceinline__ int64_t sum_units(const CacheAttnArgs& a) {
  int64_t all = 0;
  for (int b = threadIdx.x & 31; b < a.B; b += 32) all += U(a, b).count;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
  return all;
}
// The sequence that unit `at` belongs to and its first unit, by a whole warp
template <class U>
__device__ __forceinline__ int find_sequence(const CacheAttnArgs& a, int segments, int64_t at, int64_t& begin) {
  const int lane = threadIdx.x & 31;
  begin = 0;
  for (int b = 0; b < a.B; b += 32) {
    const int64_t mine = b + lane < a.B ? static_cast<int64_t>(U(a, b + lane).count) * segments : 0;
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned past = __ballot_sync(0xffffffffu, begin + upto > at);
    if (past != 0) {
      const int l = __ffs(past) - 1;
      begin += __shfl_sync(0xffffffffu, upto - mine, l);
      return b + l;
    }
    begin += __shfl_sync(0xffffffffu, upto, 31);
  }
  return a.B;
}

// Element offset of output column c of a segment (new token c / G of query head h * G + c % G)
__device__ __forceinline__ int64_t out_offset(const CacheAttnArgs& a, int b, int h, int c) {
  return ((static_cast<int64_t>(b) * a.H * a.G + h * a.G + c % a.G) * a.T + c / a.G) * a.D;
}
__device__ __forceinline__ const uint16_t* q_row(const CacheAttnArgs& a, int b, int h, int c) {
  return static_cast<const uint16_t*>(a.q) + b * a.qs[0] + (h * a.G + c % a.G) * a.qs[1] + c / a.G * a.qs[2];
}

// The workspace: notes, one per segment or per warp, whichever are fewer, then two parts per warp. A warp that has the first
// units of a segment which goes on with the next warp leaves a note about it; its part of that segment is its second, the
// parts of the others are their first ones.
struct alignas(16) Note {
  int b, seg, first, last, fresh, unused[3];       // sequence (-1: nothing to join), segment in it, its warps, real new tokens
};
// One part: per column P outputs and three numbers, the maximum, the sum and what the variant without a denominator needs; of
// as many columns as a tile has at most
constexpr int part_pitch(int P) { return P + 4; }
template <int P>
__device__ __forceinline__ float* part_of(const CacheAttnArgs& a, int columns, int64_t index) {
  return a.parts + a.notes * (sizeof(Note) / sizeof(float)) + index * (min(columns, a.T * a.G) * part_pitch(P));
}

// 2^x for -126 <= x <= 127
__device__ __forceinline__ float power2(int x) { return __int_as_float((x + 127) << 23); }

// A warp's state for one segment
template <int P>
struct Running {
  float o[P / 16][4];                              // tile j: dims 32 (j / 2) + 4 g + 2 (j % 2), + 1 of columns 2t, 2t + 1
  float m[2], l[2];                                // of columns 2t, 2t + 1; l: this lane's share
  int unit;                                        // o is in units of 2^unit
  __device__ __forceinline__ void clear() {
    unit = 0;
#pragma unroll
    for (int j = 0; j < P / 16; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
  }
  // A block's value scale goes into its weights, so that all products add up in o: weights are at most 2^8, so the unit is
  // chosen to have the largest scale at hand in [2^6, 2^7), fp16 below its limit and its smallest normal number at 2^-20 of
  // a weight of 1. It is changed, by a power of two, where a scale is above that or below 2^-6, up or down; not so far down
  // that o would leave fp32's range (it is 2^100 of what is added then).
  __device__ __forceinline__ void refer(float scale) {
    const float now = scale * power2(-unit);
    if (now < 128.f && (now >= 0.015625f || scale == 0.f)) return;
    int to = max(static_cast<int>(__float_as_uint(scale) >> 23) - 127 - 6, -126);
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < P / 16; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(o[j][e]));
    const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
    if (bits != 0) {
      to = max(to, unit - min(120, max(0, 100 - (static_cast<int>(bits >> 23) - 127))));
      const float f = power2(max(unit - to, -126));
#pragma unroll
      for (int j = 0; j < P / 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] *= f;
    }
    unit = to;
  }
  // l of the whole warp, o in units of 1
  __device__ __forceinline__ void sum_up() {
    const float up = power2(unit);
#pragma unroll
    for (int j = 0; j < P / 16; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[j][e] *= up;
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], w);
  }
  // this lane's outputs of column 2t + e, in the order of the dims
  __device__ __forceinline__ void store(float* row, int e) const {
#pragma unroll
    for (int i = 0; i < P / 32; ++i)
      *reinterpret_cast<float4*>(row + 32 * i + (threadIdx.x & 31) / 4 * 4) =
          make_float4(o[2 * i][e], o[2 * i][2 + e], o[2 * i + 1][e], o[2 * i + 1][2 + e]);
  }
  // The maximum moves only if a score exceeds it by more than the slack; s becomes the weights, l their sum.
  template <int kBlocks>
  __device__ __forceinline__ void weigh(float (&s)[kBlocks][4]) {
    float top[2];
    bool over = false;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      top[e] = fmaxf(s[0][e], s[0][2 + e]);
#pragma unroll
      for (int k = 1; k < kBlocks; ++k) top[e] = fmaxf(top[e], fmaxf(s[k][e], s[k][2 + e]));
      over |= top[e] > m[e] + kSlack;
    }
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = fmaxf(top[e], m[e]);
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
        const float f = m[e] == x ? 1.f : attn_ex2(m[e] - x);
        m[e] = x;
        l[e] *= f;
#pragma unroll
        for (int j = 0; j < P / 16; ++j) {
          o[j][e] *= f;
          o[j][2 + e] *= f;
        }
      }
    }
    float ref[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) ref[e] = m[e] == -INFINITY ? 0.f : m[e];      // no token seen yet
#pragma unroll
    for (int k = 0; k < kBlocks; ++k) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[k][e] = attn_ex2(s[k][e] - ref[e % 2]);
      l[0] += s[k][0] + s[k][2];
      l[1] += s[k][1] + s[k][3];
    }
  }
};

// Operand words of query column c (lane g's of a tile) as they are in memory: k step i has dims 64 (i / 4) + 16 t + 4 (i % 4)
// to + 3
template <int P>
__device__ __forceinline__ void load_q(const CacheAttnArgs& a, int b, int h, int c, int t, uint32_t (&w)[P / 16][2]) {
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
}

// The query columns of a segment: operands, their scales, and how far each column sees
template <bool kBf16, int P>
struct Queries {
  uint32_t w[P / 16][2];                           // fp16, scaled
  float mul[2], sq[2];                             // of columns 2t, 2t + 1: what the scores are multiplied by, g log2(e) |q|^2
  int limit[2];                                // last token that the column sees
  int first_limit, last_limit;                     // every column of the tile sees at least, none sees more
  int b, h, total;
  uint32_t exponents;

  __device__ __forceinline__ void load(const CacheAttnArgs& a, int b_, int h_, int held, int total_) {
    b = b_, h = h_, total = total_;
    exponents = a.exponents;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint32_t raw[P / 16][2];
    load_q<P>(a, b, h, g, t, raw);
    uint32_t top = 0;
    float square = 0.f;
#pragma unroll
    for (int i = 0; i < P / 16; ++i) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 f = unpack2<kBf16>(raw[i][e]);
        top = max(top, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
        square = fmaf(f.x, f.x, fmaf(f.y, f.y, square));
      }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      square += __shfl_xor_sync(0xffffffffu, square, o);
    }
    uint32_t exponent = top >> 23;                 // of the largest element; zero and infinity keep their meaning
    exponent = exponent == 0 ? 127u : min(exponent, 253u);
    const float down = __uint_as_float((254u - exponent) << 23), up = __uint_as_float(exponent << 23);
#pragma unroll
    for (int i = 0; i < P / 16; ++i) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 f = unpack2<kBf16>(raw[i][e]);
        w[i][e] = pack2<false>(f.x * down, f.y * down);
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int from = (2 * t + e) * 4;
      mul[e] = 2.f * a.scale * __shfl_sync(0xffffffffu, up, from);
      sq[e] = a.scale * __shfl_sync(0xffffffffu, square, from);
      const int c = 2 * t + e;
      limit[e] = c < a.T * a.G ? held + c / a.G : total - 1;
    }
    first_limit = held;
    last_limit = held + 7 / a.G;
  }
};

// Asks for a unit's bytes; `what`: first complete block in the page | their count << 8, or tokens of the incomplete block | 1 << 16
template <int P, int UB>
__device__ __forceinline__ void fetch_unit(uint8_t* stage, const uint8_t* page, int what) {
  using T = Tile<P, UB>;
  constexpr int kSlot = cache_slot_bytes(P);
  const int lane = threadIdx.x & 31;
  const uint32_t to = smem_u32(stage);
  if (lane == 0) *reinterpret_cast<int*>(stage + T::kFlag) = page != nullptr;
  if (page == nullptr) return;
  if (what >> 16) {
    const uint8_t* src = page + kPageHeader + kPageBlocks * kSlot + lane * 16;
#pragma unroll
    for (int i = 0; i < 2 * kSlot / 512; ++i)              // keys, then values: the rows that there are
      if ((i % (kSlot / 512) * 512 + lane * 16) / (2 * P) < (what & 0xff)) copy16(to + i * 512 + lane * 16, src + i * 512);
    return;
  }
  const uint8_t* src = page + kPageHeader + (what & 0xff) * kSlot + lane * 16;
  const int bytes = (what >> 8) * kSlot;
  if (bytes == UB * kSlot) {
#pragma unroll
    for (int i = 0; i < UB * kSlot / 512; ++i) copy16(to + i * 512 + lane * 16, src + i * 512);
  } else {
#pragma unroll
    for (int i = 0; i < UB * kSlot / 512; ++i)
      if (i * 512 < bytes) copy16(to + i * 512 + lane * 16, src + i * 512);
  }
  if (lane < UB / 2) copy16(to + T::kScales + lane * 16, page + (what & 0xff) * 8 + lane * 16);
}

// A group of complete blocks, the first of them at token `begin`. kPlain: all of the unit's blocks are there, their scales are
// finite and every column sees them: the code has no branches, so that the blocks' chains of products overlap.
template <bool kPlain, bool kBf16, int P, int UB>
__device__ __forceinline__ void codes_blocks(const CacheAttnArgs& a, const Queries<kBf16, P>& q, Running<P>& run,
                                             const uint8_t* stage, int begin, int whole) {
  using T = Tile<P, UB>;
  constexpr int kSlot = cache_slot_bytes(P);
  const int lane = threadIdx.x & 31, g = lane >> 2;
  const float2* scales = reinterpret_cast<const float2*>(stage + T::kScales);
  float s[UB][4];
#pragma unroll
  for (int k = 0; k < UB; ++k) {
#pragma unroll
    for (int e = 0; e < 4; ++e) s[k][e] = -INFINITY;
    if (!kPlain && k >= whole) continue;
    const float key_scale = scales[k].x;
    const uint4* key = reinterpret_cast<const uint4*>(stage + k * kSlot) + lane;
    int sq0 = 0, sq1 = 0;
    float acc[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = 0.f;
#pragma unroll
    for (int d = 0; d < P / 64; ++d) {
      const uint4 w0 = key[2 * d * 32], w1 = key[(2 * d + 1) * 32];
      const uint32_t r0[4] = {w0.x, w0.y, w0.z, w0.w}, r1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sq0 += dot4(r0[i]);
        sq1 += dot4(r1[i]);
        const uint32_t A[4] = {codes_lo(r0[i], q.exponents), codes_lo(r1[i], q.exponents), codes_hi(r0[i], q.exponents),
                               codes_hi(r1[i], q.exponents)};
        mma16816<false>(acc, A, q.w[d * 4 + i][0], q.w[d * 4 + i][1]);
      }
    }
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) {
      sq0 += __shfl_xor_sync(0xffffffffu, sq0, x);
      sq1 += __shfl_xor_sync(0xffffffffu, sq1, x);
    }
    const float bias = a.scale * key_scale * key_scale;
    const float b0 = bias * static_cast<float>(sq0), b1 = bias * static_cast<float>(sq1);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float mul = q.mul[e] * key_scale;
      s[k][e] = fmaf(acc[e], mul, -b0);
      s[k][2 + e] = fmaf(acc[2 + e], mul, -b1);
    }
    if (!kPlain) {
      const int tok = begin + k * kBlockTokens + 4 * (g >> 1) + (g & 1);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (tok + 2 * (e / 2) > q.limit[e % 2]) s[k][e] = -INFINITY;
    }
  }
  run.weigh(s);
  float scale[UB], most = 0.f;
#pragma unroll
  for (int k = 0; k < UB; ++k) {
    scale[k] = kPlain || k < whole ? scales[k].y : 0.f;
    if (kPlain || scale[k] < INFINITY) most = fmaxf(most, scale[k]);
  }
  run.refer(most);
  const float down = power2(-run.unit);
#pragma unroll
  for (int k = 0; k < UB; ++k) {
    if (!kPlain && k >= whole) continue;
    uint32_t p[2];
    const float by = scale[k] * down;
    const bool finite = fabsf(scale[k]) < INFINITY;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[k][e] *= by;
      // a block that is not finite reaches the columns that see it, whatever its weight, and no other
      if (!kPlain && !finite) s[k][e] = begin + k * kBlockTokens <= q.limit[e % 2] ? __int_as_float(0x7fc00000) : 0.f;
    }
    p[0] = transpose8(pack2<false>(s[k][0], s[k][1]));
    p[1] = transpose8(pack2<false>(s[k][2], s[k][3]));
    const uint4* value = reinterpret_cast<const uint4*>(stage + k * kSlot + 16 * P) + lane;
#pragma unroll
    for (int i = 0; i < P / 32; ++i) {
      const uint4 w = value[i * 32];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t r0 = half ? w.z : w.x, r1 = half ? w.w : w.y;
        const uint32_t A[4] = {codes_lo(r0, q.exponents), codes_lo(r1, q.exponents), codes_hi(r0, q.exponents),
                               codes_hi(r1, q.exponents)};
        mma16816<false>(run.o[2 * i + half], A, p[0], p[1]);
      }
    }
  }
}

template <bool kBf16, int P, int UB>
__device__ __forceinline__ void codes_unit(const CacheAttnArgs& a, const Queries<kBf16, P>& q, Running<P>& run,
                                           const uint8_t* stage, int begin) {
  using T = Tile<P, UB>;
  if (begin > q.last_limit) return;
  const int whole = min(UB, q.total / kBlockTokens - begin / kBlockTokens);
  bool plain = whole == UB && begin + T::kUnit - 1 <= q.first_limit;
  const float2* scales = reinterpret_cast<const float2*>(stage + T::kScales);
#pragma unroll
  for (int k = 0; k < UB; ++k) plain &= scales[k].y < INFINITY;
  if (plain) codes_blocks<true, kBf16, P, UB>(a, q, run, stage, begin, whole);
  else codes_blocks<false, kBf16, P, UB>(a, q, run, stage, begin, whole);
}

// The block that is not complete, in 16 bits
template <bool kBf16, int P>
__device__ __forceinline__ void rest_unit(const CacheAttnArgs& a, const Queries<kBf16, P>& q, Running<P>& run,
                                          const uint8_t* stage) {
  constexpr int J = P / 16, KC = P / 32;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int total = q.total, base = total / kBlockTokens * kBlockTokens, tok = 4 * (g >> 1) + (g & 1);
  if (base > q.last_limit) return;
  const uint16_t* keys = reinterpret_cast<const uint16_t*>(stage);
  const uint16_t* values = keys + cache_slot_bytes(P) / 2;
  float s[1][4];
#pragma unroll
  for (int e = 0; e < 4; ++e) s[0][e] = 0.f;
  float sq[2] = {0.f, 0.f};
  uint32_t qt[P / 16][2];
  load_q<P>(a, q.b, q.h, g, t, qt);
#pragma unroll
  for (int d = 0; d < P / 64; ++d) {
    uint32_t r[2][8];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const bool there = base + tok + 2 * half < total;
      const uint4* row = reinterpret_cast<const uint4*>(keys + (tok + 2 * half) * P + d * 64 + t * 16);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint4 x = there ? row[e] : make_uint4(0, 0, 0, 0);
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
      mma16816<kBf16>(s[0], A, qt[d * 4 + i][0], qt[d * 4 + i][1]);
    }
  }
#pragma unroll
  for (int x = 1; x < 4; x <<= 1) {
    sq[0] += __shfl_xor_sync(0xffffffffu, sq[0], x);
    sq[1] += __shfl_xor_sync(0xffffffffu, sq[1], x);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int token = base + tok + 2 * (e / 2);
    s[0][e] = token <= q.limit[e % 2] && token < total ? fmaf(s[0][e], 2.f * a.scale, -a.scale * sq[e / 2]) : -INFINITY;
  }
  run.weigh(s);
  uint32_t p[2];
  p[0] = transpose8(pack2<kBf16>(s[0][0], s[0][1]));
  p[1] = transpose8(pack2<kBf16>(s[0][2], s[0][3]));
  uint2 x[KC][4];                                  // dims 32 i + 4 g ... + 3 of tokens 4 t + r
  uint32_t most = 0;                               // largest magnitudes of even and odd dims, as integers
#pragma unroll
  for (int i = 0; i < KC; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      x[i][r] = make_uint2(0, 0);
      if (base + 4 * t + r < total) x[i][r] = *reinterpret_cast<const uint2*>(values + (4 * t + r) * P + 32 * i + 4 * g);
      most = __vmaxu2(most, __vmaxu2(x[i][r].x & 0x7fff7fffu, x[i][r].y & 0x7fff7fffu));
    }
  most = __reduce_max_sync(0xffffffffu, max(most & 0xffffu, most >> 16));
  const bool finite = most < (kBf16 ? 0x7f80u : 0x7c00u);
  if (finite) run.refer(unpack2<kBf16>(most).x * 0.0078125f);
  // A product 0 * inf of a column that does not see the token must not reach it: such blocks go token by token.
  const bool slow = !finite && total - 1 > q.first_limit;
#pragma unroll 1
  for (int only = slow ? 0 : kBlockTokens - 1; only < kBlockTokens; ++only) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      uint32_t A[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {                // row g: dim 4 g + 2 (j % 2), row g + 8: the next; k: tokens 0, 1 then 2, 3
        uint32_t lo = j % 2 ? x[j / 2][e / 2 * 2].y : x[j / 2][e / 2 * 2].x;
        uint32_t hi = j % 2 ? x[j / 2][e / 2 * 2 + 1].y : x[j / 2][e / 2 * 2 + 1].x;
        if (slow) {
          if (only != 4 * t + e / 2 * 2) lo = 0;
          if (only != 4 * t + e / 2 * 2 + 1) hi = 0;
        }
        A[e] = __byte_perm(lo, hi, e % 2 ? 0x7632 : 0x5410);
      }
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      mma16816<kBf16>(acc, A, p[0], p[1]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (!slow || base + only <= q.limit[e % 2]) run.o[j][e] = fmaf(acc[e], power2(-run.unit), run.o[j][e]);
    }
  }
}

// 1 / l, or what the weights of the variant without a denominator lack; 0 where nothing was seen. m, l: of all its tokens.
__device__ __forceinline__ float last_factor(const CacheAttnArgs& a, float m, float l, float q_sq) {
  if (m == -INFINITY && l == 0.f) return 0.f;
  return a.softmax ? 1.f / l : attn_ex2((m == -INFINITY ? 0.f : m) - q_sq);
}

template <bool kBf16, int P>
__global__ void __launch_bounds__(kWarpsOf8 * 32) cache_attn_kernel(const CacheAttnArgs a) {
  constexpr int UB = kUnitBlocks<P>, KC = P / 32, kStages = kStagesOf8, kWarps = kWarpsOf8;
  using T = Tile<P, UB>;
  constexpr int kBytes = cache_page_bytes(P);
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + (threadIdx.x >> 5) * (kStages * T::kStage);       // a warp has its own
  const int64_t workers = static_cast<int64_t>(gridDim.x) * kWarps;
  const int64_t self = static_cast<int64_t>(threadIdx.x >> 5) * gridDim.x + blockIdx.x;    // neighbours on other SMs
  const int segments = a.column_tiles * a.H;       // of a sequence
  const Deal deal(sum_units<Units<UB>>(a) * segments, workers);
  int64_t at = deal.begin(self);
  const int64_t stop = deal.begin(self + 1);
  Note* const notes = reinterpret_cast<Note*>(a.parts);
  const bool by_segment = a.notes < workers;
  if (lane == 0 && !by_segment) notes[self].b = -1;
  for (int64_t empty = self; empty < a.B; empty += workers) {              // sequences without new tokens
    if (Units<UB>(a, static_cast<int>(empty)).count != 0) continue;
    const int64_t words = static_cast<int64_t>(a.H) * a.G * a.T * a.D / 8;
    uint4* out = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out)) + empty * words;
    for (int64_t i = lane; i < words; i += 32) out[i] = make_uint4(0, 0, 0, 0);
    if (by_segment)
      for (int i = lane; i < segments; i += 32) notes[empty * segments + i].b = -1;
  }
  if (at >= stop) return;

  int64_t seq_begin;
  int b = find_sequence<Units<UB>>(a, segments, at, seq_begin);

  // ---- loads: lane i looks up the i-th of the next 32 units, so that page numbers are waited for once in 32 units
  struct Lookup {
    const uint8_t* page;                           // the head's part, null where there is nothing to load
    int what;                                      // see fetch_unit
  };
  int look_b = b;                                  // this lane's sequence
  int64_t look_begin = seq_begin;
  auto look_up = [&](int64_t x) {
    Lookup r{nullptr, 0};
    while (x < stop && look_b < a.B) {
      const Units<UB> units(a, look_b);
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
      r.page = cache_page(a.pages, a.table, look_b, a.max_pages, a.num_pages, a.H, h, kBytes, first * kBlockTokens);
      r.what = u < units.groups ? first % kPageBlocks | min(UB, blocks - first) << 8 : total % kBlockTokens | 1 << 16;
      break;
    }
    return r;
  };
  const int64_t start = at, mine = stop - at;
  Lookup now = look_up(start + lane), next = look_up(start + 32 + lane);
  int64_t fetched = 0;                             // units asked for
  auto fetch = [&]() {
    if (fetched < mine) {
      const int from = static_cast<int>(fetched & 31);
      if (from == 0 && fetched != 0) {
        now = next;
        next = look_up(start + fetched + 32 + lane);
      }
      const uint64_t page = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(now.page), from);
      fetch_unit<P, UB>(ring + static_cast<int>(fetched % kStages) * T::kStage, reinterpret_cast<const uint8_t*>(page),
                        __shfl_sync(0xffffffffu, now.what, from));
      ++fetched;
    }
    copies_close();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch();

  int64_t taken = 0;                               // units worked on
  while (at < stop && b < a.B) {
    const Units<UB> units(a, b);
    if (at >= seq_begin + static_cast<int64_t>(units.count) * segments) {  // on to the next sequence (some have no units)
      seq_begin += static_cast<int64_t>(units.count) * segments;
      ++b;
      continue;
    }
    const int h = static_cast<int>((at - seq_begin) / units.count);
    const int u0 = static_cast<int>((at - seq_begin) % units.count);
    const int64_t left = stop - at;
    const int u1 = left < units.count - u0 ? u0 + static_cast<int>(left) : units.count;
    Queries<kBf16, P> q;
    q.load(a, b, h, units.held, units.held + units.fresh);
    Running<P> run;
    run.clear();
    for (int u = u0; u < u1; ++u) {
      const uint8_t* stage = ring + static_cast<int>(taken % kStages) * T::kStage;
      copies_wait<kStages - 2>();
      fetch();
      ++taken;
      if (*reinterpret_cast<const int*>(stage + T::kFlag) == 0) continue;  // a page outside the pool: its tokens are absent
      if (u < units.groups) codes_unit<kBf16, P, UB>(a, q, run, stage, u * T::kUnit);
      else rest_unit<kBf16, P>(a, q, run, stage);
    }

    // ---- the segment's output, or this warp's part of it
    run.sum_up();
    const bool complete = u0 == 0 && u1 == units.count;
    float* part = part_of<P>(a, 8, 2 * self + (u0 == 0));
    if (u0 == 0 && lane == 0 && (by_segment || !complete)) {
      const int last = static_cast<int>(min(deal.worker(at + units.count - 1), workers - 1));
      Note& note = notes[by_segment ? static_cast<int64_t>(b) * segments + h : self];
      note = {complete ? -1 : b, h, static_cast<int>(self), last, units.fresh, {}};
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int c = 2 * t + e;
      if (c >= a.T * a.G) continue;
      const float m = run.m[e], l = run.l[e];
      if (complete) {
        const float f = last_factor(a, m, l, q.sq[e]);
        const bool none = c / a.G >= units.fresh || (m == -INFINITY && l == 0.f);
        uint16_t* out = static_cast<uint16_t*>(a.out) + out_offset(a, b, h, c);
#pragma unroll
        for (int i = 0; i < KC; ++i) {
          const int d = 32 * i + 4 * g;
          if (d >= a.D) continue;
          uint2 y = make_uint2(pack2<kBf16>(run.o[2 * i][e] * f, run.o[2 * i][2 + e] * f),
                               pack2<kBf16>(run.o[2 * i + 1][e] * f, run.o[2 * i + 1][2 + e] * f));
          if (none) y = make_uint2(0, 0);
          *reinterpret_cast<uint2*>(out + d) = y;
        }
      } else {
        run.store(part + c * part_pitch(P), e);
        if (g == 0) *reinterpret_cast<float4*>(part + c * part_pitch(P) + P) = make_float4(m, l, q.sq[e], 0.f);
      }
    }
    at += u1 - u0;
  }
  grid_dependents_launch();
}

// (m, l, y) of a column from two sets of its tokens
template <int kCount>
__device__ __forceinline__ void join(float& m, float& l, float (&y)[kCount], float m2, float l2, const float (&y2)[kCount]) {
  const float x = fmaxf(m, m2), ref = x == -INFINITY ? 0.f : x;
  const float f = attn_ex2(m - ref), f2 = attn_ex2(m2 - ref);
  m = x;
  l = l * f + l2 * f2;
#pragma unroll
  for (int i = 0; i < kCount; ++i) y[i] = y[i] * f + y2[i] * f2;
}
template <int kCount>
__device__ __forceinline__ void load_floats(const float* from, float (&x)[kCount]) {
  if constexpr (kCount == 4) {
    const float4 v = *reinterpret_cast<const float4*>(from);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    const float2 v = *reinterpret_cast<const float2*>(from);
    x[0] = v.x, x[1] = v.y;
  }
}

// A segment per block, or per cluster of blocks, whose warps take its units in turn: for short sequences, whose time is the
// chain of one load after another. There is no dealing out, no second kernel and no workspace; the warps' parts are joined in
// shared memory, the blocks' through the cluster's, in a fixed order.
template <bool kBf16, int P, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, 16 / kWarps) cache_attn_short_kernel(const CacheAttnArgs a) {
  constexpr int UB = 2, kRing = 2;
  using T = Tile<P, UB>;
  constexpr int kBytes = cache_page_bytes(P);
  static_assert(kRing * T::kStage >= (8 * P + 48) * 4, "a warp's part, and the block's, take the place of a ring");
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, warp = threadIdx.x >> 5;
  uint8_t* ring = smem + warp * (kRing * T::kStage);
  uint32_t rank, ranks;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ranks));
  const int segment = static_cast<int>(blockIdx.x / ranks), b = segment / a.H, h = segment % a.H;
  // the row of the page table (at most 32 pages), asked for beside the lengths
  const int id_of_lane = lane < a.max_pages ? a.table[static_cast<int64_t>(b) * a.max_pages + lane] : -1;
  const Units<UB> units(a, b);
  const int total = units.held + units.fresh, blocks = total / kBlockTokens;
  const int each = kWarps * static_cast<int>(ranks), first = static_cast<int>(rank) * kWarps + warp;
  const int mine = units.count > first ? (units.count - first + each - 1) / each : 0;

  const uint8_t* page = nullptr;                   // of this lane's unit among the next 32 of the warp
  int what = 0;
  auto look_up = [&](int i) {
    page = nullptr;
    const int u = first + (i + lane) * each, block = u < units.groups ? u * UB : blocks;
    const int id = __shfl_sync(0xffffffffu, id_of_lane, block / kPageBlocks & 31);
    if (i + lane >= mine || id < 0 || id >= a.num_pages) return;
    page = a.pages + (static_cast<int64_t>(id) * a.H + h) * kBytes;
    what = u < units.groups ? block % kPageBlocks | min(UB, blocks - block) << 8 : total % kBlockTokens | 1 << 16;
  };
  int fetched = 0;
  auto fetch = [&]() {
    if (fetched < mine) {
      if (fetched % 32 == 0) look_up(fetched);
      const uint64_t p = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(page), fetched & 31);
      fetch_unit<P, UB>(ring + fetched % kRing * T::kStage, reinterpret_cast<const uint8_t*>(p),
                        __shfl_sync(0xffffffffu, what, fetched & 31));
      ++fetched;
    }
    copies_close();
  };
#pragma unroll
  for (int i = 0; i < kRing; ++i) fetch();
  Queries<kBf16, P> q;
  Running<P> run;
  run.clear();
  if (units.count > 0) q.load(a, b, h, units.held, total);
  for (int i = 0; i < mine; ++i) {
    const uint8_t* stage = ring + i % kRing * T::kStage;
    copies_wait<kRing - 1>();
    if (*reinterpret_cast<const int*>(stage + T::kFlag) != 0) {
      const int u = first + i * each;
      if (u < units.groups) codes_unit<kBf16, P, UB>(a, q, run, stage, u * T::kUnit);
      else rest_unit<kBf16, P>(a, q, run, stage);
    }
    __syncwarp();                                  // every lane has read the stage
    fetch();
  }

  // ---- join: the warps', then the blocks'
  run.sum_up();
  const int columns = a.T * a.G;
  float* part = reinterpret_cast<float*>(ring);    // 8 x P outputs, 8 maxima, 8 sums
  __syncwarp();
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    run.store(part + (2 * t + e) * P, e);
    if (g == 0) {
      part[8 * P + 2 * t + e] = run.m[e];
      part[8 * P + 8 + 2 * t + e] = run.l[e];
    }
  }
  __syncthreads();
  constexpr int kPart = kRing * T::kStage / 4;     // floats from one warp's part to the next
  float* parts = reinterpret_cast<float*>(smem);
  constexpr int kPerColumn = P / 4;                // threads of a column, four dims each
  const int used = columns * kPerColumn;
  struct Joined {
    float m = -INFINITY, l = 0.f, y[4] = {};
  };
  auto write = [&](int i, const Joined& j) {
    const int c = i / kPerColumn, d = i % kPerColumn * 4;
    if (d >= a.D) return;
    float f = 0.f;
    if (c / a.G < units.fresh) f = last_factor(a, j.m, j.l, parts[8 * P + 16 + c]);
    uint2 y = make_uint2(pack2<kBf16>(j.y[0] * f, j.y[1] * f), pack2<kBf16>(j.y[2] * f, j.y[3] * f));
    if (c / a.G >= units.fresh || (j.m == -INFINITY && j.l == 0.f)) y = make_uint2(0, 0);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + out_offset(a, b, h, c) + d) = y;
  };
  if (warp == 0 && g == 0)                         // |q|^2, which every warp has
    for (int e = 0; e < 2; ++e) parts[8 * P + 16 + 2 * t + e] = units.count > 0 ? q.sq[e] : 0.f;
  __syncthreads();
  for (int i = threadIdx.x; i < used; i += kWarps * 32) {
    const int c = i / kPerColumn, at = c * P + i % kPerColumn * 4;
    Joined j;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float* p = parts + w * kPart;
      float y2[4];
      load_floats(p + at, y2);
      join(j.m, j.l, j.y, p[8 * P + c], p[8 * P + 8 + c], y2);
    }
    if (ranks == 1) {
      write(i, j);
    } else {                                       // the block's part, where the second warp's was: read by this thread alone
      float* p = parts + kPart;
      *reinterpret_cast<float4*>(p + at) = make_float4(j.y[0], j.y[1], j.y[2], j.y[3]);
      if (i % kPerColumn == 0) {
        p[8 * P + 32 + c] = j.m;
        p[8 * P + 40 + c] = j.l;
      }
    }
  }
  if (ranks == 1) return;
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (rank == 0) {
    for (int i = threadIdx.x; i < used; i += kWarps * 32) {
      const int c = i / kPerColumn, at = c * P + i % kPerColumn * 4;
      Joined j;
      for (uint32_t r = 0; r < ranks; ++r) {
        uint32_t there;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(smem_u32(parts + kPart)), "r"(r));
        float m2, l2, y2[4];
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(m2) : "r"(there + (8 * P + 32 + c) * 4));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(l2) : "r"(there + (8 * P + 40 + c) * 4));
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(y2[0]), "=f"(y2[1]), "=f"(y2[2]), "=f"(y2[3]) : "r"(there + at * 4));
        join(j.m, j.l, j.y, m2, l2, y2);
      }
      write(i, j);
    }
  }
  __syncwarp();
  // blocks stay until they have been read
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---------------------------------------------------------------------------------------------------------------------
// Many columns: the queries are the 16-row operand
// ---------------------------------------------------------------------------------------------------------------------
// With more than 8 columns of queries (chunks of a prompt, many query heads to a key head) a byte's widening is shared by a
// block: its four warps widen a unit of four blocks of tokens, one each, into operand order in shared memory (the cache's order
// with two bytes for one: lane (g, t)'s 16 codes are the second operand of four products, of the keys' dims and of the values'
// tokens alike), and every warp multiplies 16 query rows with it: S (16 rows x 8 tokens) = Q K^T, O += P V, where the
// accumulators of S are in place as the operand P. RW warps have different rows; where fewer than four are needed the others
// have other blocks of the unit, and the warps with the same rows join at the end of the segment.
// The block that is not complete is brought to fp16 by powers of two, its largest key and value to [1, 2): exact but for
// elements below 2^-14 of it (off by 2^-25 of it), and is then a block like the others.
// What bounds it is the chain inside a unit - barrier, widening, barrier, products, exponentials, products - with 12 (8 at 128
// dims) warps on an SM: the tensor pipe is busy for 19 to 28 % of the time, the issue slots for 33 to 44 %. 37 new tokens on 6
// histories of up to 5003, 16 heads of 64: 39 to 41 us a call; 200 on 32 of up to 500, 8 heads: 76 (112 with the cache as the row operand and 32
// columns a warp). Three blocks of 168 registers on an SM, or two of 255, with spills of up to 92 bytes a thread (bfloat16,
// 64 rows of 64 columns; 72 in float16, 20 to 32 with fewer rows, at 128 columns 8 to 24 in float16 and none in bfloat16); four and
// three blocks spill more (50 and 93 us).
// Three units under way instead of two, the incomplete block's rows among them: 41 and 81 us; the next unit widened beside the
// products, with one barrier a unit instead of two: 40 and 79.
constexpr int kRowWarps = 4;
template <int P>
struct RowTile {
  static constexpr int kRaw = kRowWarps * cache_slot_bytes(P);             // codes as they come, two units
  static constexpr int kStage = kRaw + 64;                                 // and their scales
  static constexpr int kWide = 2 * kRaw;                                   // a unit's operands: keys, then values
  static constexpr int kSmem = 2 * kStage + kWide;
  static constexpr int kBlocks = P == 64 ? 3 : 2;                          // on an SM
};

// A warp's state for its 16 rows: rows g and g + 8 of a lane
template <int P>
struct RowState {
  float o[P / 32][4][4];                           // [c][i]: dims 32 c + 8 t + i and + 4 + i of row g, then of row g + 8
  float m[2], l[2];
  int unit;                                        // o is in units of 2^unit
  __device__ __forceinline__ void clear() {
    unit = 0;
#pragma unroll
    for (int c = 0; c < P / 32; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[c][i][e] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
  }
  __device__ __forceinline__ void times(float f0, float f1) {
#pragma unroll
    for (int c = 0; c < P / 32; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[c][i][0] *= f0;
        o[c][i][1] *= f0;
        o[c][i][2] *= f1;
        o[c][i][3] *= f1;
      }
  }
  // See Running::refer
  __device__ __forceinline__ void refer(float scale) {
    const float now = scale * power2(-unit);
    if (now < 128.f && (now >= 0.015625f || scale == 0.f)) return;
    int to = max(static_cast<int>(__float_as_uint(scale) >> 23) - 127 - 6, -126);
    float top = 0.f;
#pragma unroll
    for (int c = 0; c < P / 32; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(o[c][i][e]));
    const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
    if (bits != 0) {
      to = max(to, unit - min(120, max(0, 100 - (static_cast<int>(bits >> 23) - 127))));
      const float f = power2(max(unit - to, -126));
      times(f, f);
    }
    unit = to;
  }
};

// 16 codes of a lane as the second operands of four products
__device__ __forceinline__ void widen_codes(uint4 w, uint32_t exponents, uint4* to) {
  to[0] = make_uint4(codes_lo(w.x, exponents), codes_hi(w.x, exponents), codes_lo(w.y, exponents), codes_hi(w.y, exponents));
  to[32] = make_uint4(codes_lo(w.z, exponents), codes_hi(w.z, exponents), codes_lo(w.w, exponents), codes_hi(w.w, exponents));
}

template <bool kBf16>
__device__ __forceinline__ uint32_t rescale2(uint32_t w, float f) {
  const float2 x = unpack2<kBf16>(w);
  return pack2<false>(x.x * f, x.y * f);
}
// The power of two that brings a number of these bits (of a float's magnitude) to [1, 2), and its inverse
__device__ __forceinline__ float to_one(uint32_t bits, float& back) {
  uint32_t exponent = bits >> 23;
  exponent = exponent == 0 ? 127u : min(exponent, 253u);
  back = __uint_as_float(exponent << 23);
  return __uint_as_float((254u - exponent) << 23);
}

template <bool kBf16, int P, int RW>
__global__ void __launch_bounds__(kRowWarps * 32, RowTile<P>::kBlocks) cache_attn_rows_kernel(const CacheAttnArgs a) {
  using T = RowTile<P>;
  constexpr int KC = P / 32, UB = kRowWarps, kSlot = cache_slot_bytes(P), kBytes = cache_page_bytes(P);
  constexpr int kRows = 16 * RW, kUnitTokens = UB * kBlockTokens;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ alignas(16) float s_bias[UB][kBlockTokens];
  __shared__ float s_key[UB], s_value[UB];
  __shared__ int s_there;                          // blocks of the unit that are there
  __shared__ bool s_odd[UB];                       // the incomplete block has a value that is not finite
  uint8_t* const wide = smem + 2 * T::kStage;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, warp = threadIdx.x >> 5;
  const int row0 = warp % RW * 16, group = warp / RW;                      // its rows, its RW blocks of a unit
  const int workers = gridDim.x, self = blockIdx.x, segments = a.column_tiles * a.H;
  const Deal deal(sum_units<AllUnits<UB>>(a) * segments, workers);
  int64_t at = deal.begin(self);
  const int64_t stop = deal.begin(self + 1);
  Note* const notes = reinterpret_cast<Note*>(a.parts);
  const bool by_segment = a.notes < workers;
  if (threadIdx.x == 0 && !by_segment) notes[self].b = -1;
  for (int empty = self; empty < a.B; empty += workers) {                  // sequences without new tokens
    if (AllUnits<UB>(a, empty).count != 0) continue;
    const int64_t words = static_cast<int64_t>(a.H) * a.G * a.T * a.D / 8;
    uint4* out = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out)) + empty * words;
    for (int64_t i = threadIdx.x; i < words; i += kRowWarps * 32) out[i] = make_uint4(0, 0, 0, 0);
    if (by_segment)
      for (int i = threadIdx.x; i < segments; i += kRowWarps * 32) notes[static_cast<int64_t>(empty) * segments + i].b = -1;
  }
  if (at >= stop) return;

  int64_t seq_begin;
  int b = find_sequence<AllUnits<UB>>(a, segments, at, seq_begin);

  // ---- loads: two units ahead of their use, their page numbers one more, so that nothing waits for these
  int64_t look_left = stop - at;                   // units of the block whose page has not been looked up
  int look_b = b, look_seg = static_cast<int>((at - seq_begin) / AllUnits<UB>(a, b).count);
  int look_u = static_cast<int>((at - seq_begin) % AllUnits<UB>(a, b).count), look_count = 0, look_blocks = 0;
  auto look_at = [&](int sequence) {
    const AllUnits<UB> units(a, sequence);
    look_count = units.count;
    look_blocks = (units.held + units.fresh) / kBlockTokens;
  };
  look_at(b);
  int next_id = -1, next_h = 0, next_what = 0;     // page number, head, first block in the page | complete blocks << 8
  auto look_up = [&]() {
    next_id = -1;
    if (look_left == 0) return;
    --look_left;
    const int column = look_u * kUnitTokens / kPageTokens;
    if (column < a.max_pages) next_id = a.table[static_cast<int64_t>(look_b) * a.max_pages + column];
    next_h = look_seg % a.H;
    next_what = look_u * UB % kPageBlocks | max(0, min(UB, look_blocks - look_u * UB)) << 8;
    if (++look_u < look_count) return;
    look_u = 0;
    if (++look_seg < segments) return;
    look_seg = 0;
    do {
      if (++look_b == a.B) break;
      look_at(look_b);
    } while (look_count == 0);
    if (look_b == a.B) look_left = 0;
  };
  const uint8_t *page = nullptr, *next_page = nullptr;                     // of the unit at hand and of the next
  auto fetch = [&](int slot) {
    page = next_page;
    next_page = nullptr;
    if (next_id >= 0 && next_id < a.num_pages) {
      next_page = a.pages + (static_cast<int64_t>(next_id) * a.H + next_h) * kBytes;
      const uint8_t* src = next_page + kPageHeader + (next_what & 0xff) * kSlot + threadIdx.x * 16;
      const uint32_t to = smem_u32(smem + slot * T::kStage);
      const int bytes = (next_what >> 8) * kSlot;
#pragma unroll
      for (int i = 0; i < T::kRaw / (kRowWarps * 512); ++i)
        if (i * (kRowWarps * 512) + static_cast<int>(threadIdx.x) * 16 < bytes)
          copy16(to + i * (kRowWarps * 512) + threadIdx.x * 16, src + i * (kRowWarps * 512));
      if (threadIdx.x < 2 && bytes > 0)
        copy16(to + T::kRaw + threadIdx.x * 16, next_page + (next_what & 0xff) * 8 + threadIdx.x * 16);
    }
    copies_close();
    look_up();
  };
  look_up();
  fetch(0);
  fetch(1);

  int slot = 0;
  while (at < stop && b < a.B) {
    const AllUnits<UB> units(a, b);
    if (at >= seq_begin + static_cast<int64_t>(units.count) * segments) {
      seq_begin += static_cast<int64_t>(units.count) * segments;
      ++b;
      continue;
    }
    const int total = units.held + units.fresh;
    const int seg = static_cast<int>((at - seq_begin) / units.count);
    const int u0 = static_cast<int>((at - seq_begin) % units.count);
    const int64_t left = stop - at;
    const int u1 = left < units.count - u0 ? u0 + static_cast<int>(left) : units.count;
    const int h = seg % a.H, c0 = seg / a.H * kRows;
    const int columns = min(kRows, a.T * a.G - c0);

    // ---- queries, as in Queries::load; rows g and g + 8
    uint32_t q[P / 16][4];
    float mul[2], q_sq[2];
    int limit[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int c = c0 + row0 + g + 8 * e;
      uint32_t raw[P / 16][2];
      load_q<P>(a, b, h, c, t, raw);
      uint32_t top = 0;
      float square = 0.f;
#pragma unroll
      for (int i = 0; i < P / 16; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float2 f = unpack2<kBf16>(raw[i][k]);
          top = max(top, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
          square = fmaf(f.x, f.x, fmaf(f.y, f.y, square));
        }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        square += __shfl_xor_sync(0xffffffffu, square, o);
      }
      float up;
      const float down = to_one(top, up);
#pragma unroll
      for (int i = 0; i < P / 16; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) q[i][2 * k + e] = rescale2<kBf16>(raw[i][k], down);
      mul[e] = 2.f * a.scale * up;
      q_sq[e] = a.scale * square;
      limit[e] = c < a.T * a.G ? units.held + c / a.G : total - 1;
    }
    const int first_limit = units.held + (c0 + row0) / a.G, last_limit = units.held + (c0 + columns - 1) / a.G;
    const bool active = row0 < columns;            // some of the warp's rows are real

    RowState<P> run;
    run.clear();
    for (int u = u0; u < u1; ++u) {
      const int begin = u * kUnitTokens;
      const bool seen = begin <= last_limit;       // by some column of the tile
      copies_wait<1>();
      __syncthreads();                             // the unit is there, and the last one's operands have been read
      const uint8_t* raw = smem + slot * T::kStage;
      if (threadIdx.x == 0)
        s_there = page == nullptr || !seen ? 0 : min(UB, (total - begin + kBlockTokens - 1) / kBlockTokens);
      if (page != nullptr && seen) {
        const int base = begin + warp * kBlockTokens;
        uint4* keys = reinterpret_cast<uint4*>(wide) + warp * (2 * P / 64) * 64 + lane;
        uint4* values = reinterpret_cast<uint4*>(wide + T::kRaw) + warp * KC * 64 + lane;
        if (base + kBlockTokens <= total) {
          const uint4* from = reinterpret_cast<const uint4*>(raw + warp * kSlot) + lane;
          const float2 scale = reinterpret_cast<const float2*>(raw + T::kRaw)[warp];
          int sq[2] = {0, 0};
#pragma unroll
          for (int d = 0; d < P / 64; ++d)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint4 w = from[(2 * d + half) * 32];
              sq[half] += dot4(w.x) + dot4(w.y) + dot4(w.z) + dot4(w.w);
              widen_codes(w, a.exponents, keys + (half * (P / 64) + d) * 64);
            }
#pragma unroll
          for (int i = 0; i < KC; ++i) widen_codes(from[(KC + i) * 32], a.exponents, values + i * 64);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            sq[half] += __shfl_xor_sync(0xffffffffu, sq[half], 1);
            sq[half] += __shfl_xor_sync(0xffffffffu, sq[half], 2);
            if (t == 0)
              s_bias[warp][4 * (g >> 1) + 2 * half + (g & 1)] = a.scale * scale.x * scale.x * static_cast<float>(sq[half]);
          }
          if (lane == 0) {
            s_key[warp] = scale.x;
            s_value[warp] = scale.y;
            s_odd[warp] = false;
          }
        } else if (base < total) {
          const uint16_t* rest = reinterpret_cast<const uint16_t*>(page + kPageHeader + kPageBlocks * kSlot);
          uint32_t k[2][P / 64][8], top = 0;       // largest magnitude of the finite ones: rows may see these alone
          float sq[2] = {0.f, 0.f};
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int tok = 4 * (g >> 1) + 2 * half + (g & 1);
#pragma unroll
            for (int d = 0; d < P / 64; ++d) {
              const uint4* row = reinterpret_cast<const uint4*>(rest + tok * P + d * 64 + t * 16);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const uint4 x = base + tok < total ? row[e] : make_uint4(0, 0, 0, 0);
                k[half][d][4 * e] = x.x, k[half][d][4 * e + 1] = x.y, k[half][d][4 * e + 2] = x.z, k[half][d][4 * e + 3] = x.w;
              }
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float2 f = unpack2<kBf16>(k[half][d][i]);
                sq[half] = fmaf(f.x, f.x, fmaf(f.y, f.y, sq[half]));
                const uint32_t b0 = __float_as_uint(f.x) & 0x7fffffffu, b1 = __float_as_uint(f.y) & 0x7fffffffu;
                top = max(top, max(b0 < 0x7f800000u ? b0 : 0u, b1 < 0x7f800000u ? b1 : 0u));
              }
            }
            sq[half] += __shfl_xor_sync(0xffffffffu, sq[half], 1);
            sq[half] += __shfl_xor_sync(0xffffffffu, sq[half], 2);
            if (t == 0) s_bias[warp][tok] = a.scale * sq[half];
          }
          float up;
          float down = to_one(__reduce_max_sync(0xffffffffu, top), up);
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int d = 0; d < P / 64; ++d)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                keys[(half * (P / 64) + d) * 64 + e * 32] =
                    make_uint4(rescale2<kBf16>(k[half][d][4 * e], down), rescale2<kBf16>(k[half][d][4 * e + 1], down),
                               rescale2<kBf16>(k[half][d][4 * e + 2], down), rescale2<kBf16>(k[half][d][4 * e + 3], down));
          if (lane == 0) s_key[warp] = up;
          uint2 x[KC][4];                          // dims 32 i + 4 g ... + 3 of tokens 4 t + r
          bool odd = false;
          top = 0;                                 // of the finite ones
#pragma unroll
          for (int i = 0; i < KC; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              x[i][r] = make_uint2(0, 0);
              if (base + 4 * t + r < total)
                x[i][r] = *reinterpret_cast<const uint2*>(rest + kSlot / 2 + (4 * t + r) * P + 32 * i + 4 * g);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float2 f = unpack2<kBf16>(e ? x[i][r].y : x[i][r].x);
                const uint32_t b0 = __float_as_uint(f.x) & 0x7fffffffu, b1 = __float_as_uint(f.y) & 0x7fffffffu;
                odd |= b0 >= 0x7f800000u || b1 >= 0x7f800000u;
                top = max(top, max(b0 < 0x7f800000u ? b0 : 0u, b1 < 0x7f800000u ? b1 : 0u));
              }
            }
          down = to_one(__reduce_max_sync(0xffffffffu, top), up);
          odd = __any_sync(0xffffffffu, odd);
          if (lane == 0) {
            s_value[warp] = up;
            s_odd[warp] = odd;
          }
#pragma unroll
          for (int i = 0; i < KC; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {          // dims 4 g + 2 e, + 1: tokens 0, 1 and 2, 3 of each
              const uint32_t x0 = e ? x[i][0].y : x[i][0].x, x1 = e ? x[i][1].y : x[i][1].x;
              const uint32_t x2 = e ? x[i][2].y : x[i][2].x, x3 = e ? x[i][3].y : x[i][3].x;
              values[i * 64 + e * 32] =
                  make_uint4(rescale2<kBf16>(__byte_perm(x0, x1, 0x5410), down),
                             rescale2<kBf16>(__byte_perm(x2, x3, 0x5410), down),
                             rescale2<kBf16>(__byte_perm(x0, x1, 0x7632), down),
                             rescale2<kBf16>(__byte_perm(x2, x3, 0x7632), down));
            }
        }
      }
      __syncthreads();                             // the operands are there, the codes have been read
      fetch(slot);
      slot ^= 1;
      const int there = s_there;
      if (!active || there <= group * RW) continue;

      // Whole units whose tokens all rows see, with finite scales, are most: without a branch in them.
      auto work = [&](auto plain) {
        constexpr bool kPlain = decltype(plain)::value;
        // ---- scores of this warp's blocks
        float s[RW][2][4];
#pragma unroll
        for (int j = 0; j < RW; ++j) {
          const int k = group * RW + j;
          if (!kPlain && k >= there) {
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
              for (int e = 0; e < 4; ++e) s[j][half][e] = -INFINITY;
            continue;
          }
          const uint4* keys = reinterpret_cast<const uint4*>(wide) + k * (2 * P / 64) * 64 + lane;
          const float key = s_key[k], mul0 = mul[0] * key, mul1 = mul[1] * key;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float(&acc)[4] = s[j][half];
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = 0.f;
#pragma unroll
            for (int d = 0; d < P / 64; ++d) {
              const uint4 x = keys[(half * (P / 64) + d) * 64], y = keys[(half * (P / 64) + d) * 64 + 32];
              mma16816<false>(acc, q[d * 4], x.x, x.y);
              mma16816<false>(acc, q[d * 4 + 1], x.z, x.w);
              mma16816<false>(acc, q[d * 4 + 2], y.x, y.y);
              mma16816<false>(acc, q[d * 4 + 3], y.z, y.w);
            }
            const float2 bias = *reinterpret_cast<const float2*>(&s_bias[k][4 * t + 2 * half]);
            acc[0] = fmaf(acc[0], mul0, -bias.x);
            acc[1] = fmaf(acc[1], mul0, -bias.y);
            acc[2] = fmaf(acc[2], mul1, -bias.x);
            acc[3] = fmaf(acc[3], mul1, -bias.y);
            if (!kPlain) {
              const int tok = begin + k * kBlockTokens + 4 * t + 2 * half;
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (tok + e % 2 > limit[e / 2] || tok + e % 2 >= total) acc[e] = -INFINITY;
            }
          }
        }
        // ---- weights, as Running::weigh
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < RW; ++j)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            top[0] = fmaxf(top[0], fmaxf(s[j][half][0], s[j][half][1]));
            top[1] = fmaxf(top[1], fmaxf(s[j][half][2], s[j][half][3]));
          }
        if (__any_sync(0xffffffffu, top[0] > run.m[0] + kSlack || top[1] > run.m[1] + kSlack)) {
          float f[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = fmaxf(top[e], run.m[e]);
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
            f[e] = run.m[e] == x ? 1.f : attn_ex2(run.m[e] - x);
            run.m[e] = x;
            run.l[e] *= f[e];
          }
          run.times(f[0], f[1]);
        }
        const float ref[2] = {run.m[0] == -INFINITY ? 0.f : run.m[0], run.m[1] == -INFINITY ? 0.f : run.m[1]};
        float most = 0.f;
#pragma unroll
        for (int j = 0; j < RW; ++j)
          if (kPlain || (group * RW + j < there && s_value[group * RW + j] < INFINITY))
            most = fmaxf(most, s_value[group * RW + j]);
        run.refer(most);
        const float down = power2(-run.unit);
#pragma unroll
        for (int j = 0; j < RW; ++j) {
          const int k = group * RW + j;
          if (!kPlain && k >= there) continue;
          const float value = s_value[k], by = value * down;
          const bool finite = fabsf(value) < INFINITY;
          uint32_t p[4];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[j][half][e] = attn_ex2(s[j][half][e] - ref[e / 2]);
            run.l[0] += s[j][half][0] + s[j][half][1];
            run.l[1] += s[j][half][2] + s[j][half][3];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s[j][half][e] *= by;
              if (!kPlain && !finite)
                s[j][half][e] = begin + k * kBlockTokens <= limit[e / 2] ? __int_as_float(0x7fc00000) : 0.f;
            }
            p[2 * half] = pack2<false>(s[j][half][0], s[j][half][1]);
            p[2 * half + 1] = pack2<false>(s[j][half][2], s[j][half][3]);
          }
          const uint4* values = reinterpret_cast<const uint4*>(wide + T::kRaw) + k * KC * 64 + lane;
          if (kPlain || !s_odd[k]) {
#pragma unroll
            for (int c = 0; c < KC; ++c) {
              const uint4 x = values[c * 64], y = values[c * 64 + 32];
              mma16816<false>(run.o[c][0], p, x.x, x.y);
              mma16816<false>(run.o[c][1], p, x.z, x.w);
              mma16816<false>(run.o[c][2], p, y.x, y.y);
              mma16816<false>(run.o[c][3], p, y.z, y.w);
            }
          } else {                                   // token by token: 0 * inf must not reach rows that do not see it
#pragma unroll 1
            for (int only = 0; only < kBlockTokens; ++only) {
              const uint32_t mask = only % 2 ? 0xffff0000u : 0x0000ffffu;
              const uint32_t lo = t == only / 4 && only % 4 < 2 ? mask : 0u, hi = t == only / 4 && only % 4 >= 2 ? mask : 0u;
              const int token = begin + k * kBlockTokens + only;
#pragma unroll
              for (int c = 0; c < KC; ++c) {
                const uint4 x = values[c * 64], y = values[c * 64 + 32];
                const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  float acc[4] = {0.f, 0.f, 0.f, 0.f};
                  mma16816<false>(acc, p, w[2 * i] & lo, w[2 * i + 1] & hi);
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    if (token <= limit[e / 2]) run.o[c][i][e] += acc[e];
                }
              }
            }
          }
        }
      };
      const bool whole = begin + kUnitTokens - 1 <= first_limit && begin + kUnitTokens <= total;
      bool finite_values = true;
#pragma unroll
      for (int j = 0; j < RW; ++j) finite_values &= s_value[group * RW + j] < INFINITY;
      if (whole && finite_values) work(std::true_type{});
      else work(std::false_type{});
    }

    // ---- the rows' warps with other blocks join the first, in the operands' place; then the output, or a part of it
    const float up = power2(run.unit);
    run.times(up, up);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      run.l[e] += __shfl_xor_sync(0xffffffffu, run.l[e], 1);
      run.l[e] += __shfl_xor_sync(0xffffffffu, run.l[e], 2);
    }
    if constexpr (RW < kRowWarps) {
      constexpr int kState = KC * 4 + 1;           // 16-byte words of a lane
      static_assert((kRowWarps - RW) * kState * 512 <= T::kWide, "states in the operands' place");
      __syncthreads();
      float4* state = reinterpret_cast<float4*>(wide) + lane;
      if (group > 0) {
        float4* to = state + (warp - RW) * kState * 32;
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            to[(c * 4 + i) * 32] = make_float4(run.o[c][i][0], run.o[c][i][1], run.o[c][i][2], run.o[c][i][3]);
        to[KC * 4 * 32] = make_float4(run.m[0], run.m[1], run.l[0], run.l[1]);
      }
      __syncthreads();
      if (group == 0) {
#pragma unroll 1
        for (int other = warp; other < kRowWarps - RW; other += RW) {
          const float4* from = state + other * kState * 32;
          const float4 z = from[KC * 4 * 32];
          const float m2[2] = {z.x, z.y}, l2[2] = {z.z, z.w};
          float f[2], f2[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float x = fmaxf(run.m[e], m2[e]), r = x == -INFINITY ? 0.f : x;
            f[e] = attn_ex2(run.m[e] - r);
            f2[e] = attn_ex2(m2[e] - r);
            run.m[e] = x;
            run.l[e] = run.l[e] * f[e] + l2[e] * f2[e];
          }
#pragma unroll
          for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float4 y = from[(c * 4 + i) * 32];
              run.o[c][i][0] = run.o[c][i][0] * f[0] + y.x * f2[0];
              run.o[c][i][1] = run.o[c][i][1] * f[0] + y.y * f2[0];
              run.o[c][i][2] = run.o[c][i][2] * f[1] + y.z * f2[1];
              run.o[c][i][3] = run.o[c][i][3] * f[1] + y.w * f2[1];
            }
        }
      }
    }
    const bool complete = u0 == 0 && u1 == units.count;
    if (u0 == 0 && threadIdx.x == 0 && (by_segment || !complete)) {
      const int last = static_cast<int>(min(deal.worker(at + units.count - 1), static_cast<int64_t>(workers - 1)));
      notes[by_segment ? static_cast<int64_t>(b) * segments + seg : self] = {complete ? -1 : b, seg, self, last, units.fresh, {}};
    }
    if (group == 0) {
      float* part = part_of<P>(a, kRows, 2 * self + (u0 == 0));
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int in = row0 + g + 8 * e, c = c0 + in;
        if (c >= a.T * a.G) continue;
        const float m = run.m[e], l = run.l[e];
        const float f = complete ? last_factor(a, m, l, q_sq[e]) : 1.f;
        const bool none = c / a.G >= units.fresh || (m == -INFINITY && l == 0.f);
        uint16_t* out = static_cast<uint16_t*>(a.out) + out_offset(a, b, h, c);
#pragma unroll
        for (int i = 0; i < KC; ++i) {
          const float(&o)[4][4] = run.o[i];
          const int d = 32 * i + 8 * t;
          if (complete) {
            if (d >= a.D) continue;
            uint4 y = make_uint4(pack2<kBf16>(o[0][2 * e] * f, o[1][2 * e] * f), pack2<kBf16>(o[2][2 * e] * f, o[3][2 * e] * f),
                                 pack2<kBf16>(o[0][2 * e + 1] * f, o[1][2 * e + 1] * f),
                             pack2<kBf16>(o[2][2 * e + 1] * f, o[3][2 * e + 1] * f));
            if (none) y = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(out + d) = y;
          } else {
            float4* to = reinterpret_cast<float4*>(part + in * part_pitch(P) + d);
            to[0] = make_float4(o[0][2 * e], o[1][2 * e], o[2][2 * e], o[3][2 * e]);
            to[1] = make_float4(o[0][2 * e + 1], o[1][2 * e + 1], o[2][2 * e + 1], o[3][2 * e + 1]);
          }
        }
        if (!complete && t == 0) *reinterpret_cast<float4*>(part + in * part_pitch(P) + P) = make_float4(m, l, q_sq[e], 0.f);
      }
    }
    at += u1 - u0;
  }
  grid_dependents_launch();
}

constexpr int kJoinWarps = 32;                     // of a block at most

// Joins the parts of the segments that several warps worked on: blocks (i, ...) the segment of note i, a block's warps its
// columns in groups of `split` to a column.
template <bool kBf16, int P, int kColumns>
__global__ void __launch_bounds__(kJoinWarps * 32) cache_join_kernel(const CacheAttnArgs a, const int workers, const int split) {
  __shared__ float s_y[kJoinWarps][P], s_m[kJoinWarps], s_l[kJoinWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, share = warp % split;
  constexpr int kPer = P / 32;
  grid_dependency_wait();
  const int in = static_cast<int>(blockIdx.y) * (static_cast<int>(blockDim.x) / 32 / split) + warp / split;
  const Note note = reinterpret_cast<const Note*>(a.parts)[blockIdx.x];
  // nothing to join; and lengths that changed while the kernels ran must not lead outside of the tensors
  if (note.b < 0 || note.b >= a.B || static_cast<unsigned>(note.seg) >= static_cast<unsigned>(a.column_tiles * a.H) ||
      note.first < 0 || note.first > note.last || note.last >= workers)
    return;
  const int first = note.first;
  const int h = note.seg % a.H, c = note.seg / a.H * kColumns + in;
  const bool real = in < kColumns && c < a.T * a.G, some = real && c / a.G < note.fresh;
  float y[kPer] = {}, m = -INFINITY, l = 0.f, q_sq = 0.f;
  if (some) {
    const int64_t pitch = min(kColumns, a.T * a.G) * part_pitch(P);
    const float* part = part_of<P>(a, kColumns, 2 * (first + share) + (share == 0)) + in * part_pitch(P);
    if (share == 0) q_sq = part[P + 2];
#pragma unroll 4
    for (int w = first + share; w <= note.last; w += split) {
      float y2[kPer];
      load_floats(part + lane * kPer, y2);
      const float4 of_column = *reinterpret_cast<const float4*>(part + P);
      join(m, l, y, of_column.x, of_column.y, y2);
      part += (2 * split - (w == first)) * pitch;
    }
  }
  if (split > 1) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) s_y[warp][lane * kPer + i] = y[i];
    if (lane == 0) {
      s_m[warp] = m;
      s_l[warp] = l;
    }
    __syncthreads();
    if (share != 0) return;
    for (int w = warp + 1; w < warp + split; ++w) {
      float y2[kPer];
      load_floats(s_y[w] + lane * kPer, y2);
      join(m, l, y, s_m[w], s_l[w], y2);
    }
  }
  if (!real || lane * kPer >= a.D) return;
  const float f = some ? last_factor(a, m, l, q_sq) : 0.f;
  const bool none = !some || (m == -INFINITY && l == 0.f);
  uint32_t packed[kPer / 2];
#pragma unroll
  for (int i = 0; i < kPer / 2; ++i) packed[i] = none ? 0u : pack2<kBf16>(y[2 * i] * f, y[2 * i + 1] * f);
  uint16_t* to = static_cast<uint16_t*>(a.out) + out_offset(a, note.b, h, c) + lane * kPer;
  if constexpr (kPer == 4) *reinterpret_cast<uint2*>(to) = make_uint2(packed[0], packed[1]);
  else *reinterpret_cast<uint32_t*>(to) = packed[0];
}

template <bool kBf16, int P, int kColumns>
cudaError_t join_t(const CacheAttnArgs& a, int workers, cudaStream_t stream) {
  const int64_t segments = static_cast<int64_t>(a.B) * a.column_tiles * a.H;
  // a warp for every eight of the parts that a segment has on average, and eight warps or more to a block
  const int width = static_cast<int64_t>(a.T) * a.G < kColumns ? a.T * a.G : kColumns;
  const int64_t parts = workers / segments;
  int split = 1;
  while (split < kJoinWarps && split * 8 < parts) split *= 2;
  const int warps = split > 8 ? split : 8, each = warps / split;
  return launch_dependent(cache_join_kernel<kBf16, P, kColumns>, dim3(a.notes, (width + each - 1) / each), warps * 32, 0, stream, a,
                          workers, split);
}

int64_t cache_attn_notes(int64_t segments, int64_t workers) { return segments < workers ? segments : workers; }

template <bool kBf16, int P>
cudaError_t attn_t(CacheAttnArgs a, int sms, cudaStream_t stream) {
  constexpr int kSmem = kWarpsOf8 * kStagesOf8 * Tile<P, kUnitBlocks<P>>::kStage;
  const int workers = sms * kWarpsOf8;
  const int64_t segments = static_cast<int64_t>(a.B) * a.column_tiles * a.H;
  a.notes = static_cast<int>(cache_attn_notes(segments, workers));
  static PerDeviceFlags flags;
  cudaError_t e = ensure_dynamic_smem(cache_attn_kernel<kBf16, P>, kSmem, flags);
  if (e != cudaSuccess) return e;
  cache_attn_kernel<kBf16, P><<<sms, kWarpsOf8 * 32, kSmem, stream>>>(a);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  return join_t<kBf16, P, 8>(a, workers, stream);
}

// Blocks of a cluster that share a segment in the kernel for short sequences, 0: not that kernel. What the lengths are is known on
// the device alone, so the rule goes by the page table's width: up to 4096 tokens, up to 8192 where the segments are no more than
// the SMs (columns: 8 at most). Calls with 8 heads of 64, this kernel and the dealing one: 1 x 1000 tokens 7.8 and 11.4 us,
// 64 x 1028 16.8 and 24.3, 200 x 400 21.0 and 28.4, 4 x 4000 10.8 and 14.7, 16 x 4000 20.7 and 23.1, but 64 x 4000 43.6 and 41.7
// (128 columns: 67.9 and 61.8). A segment has more blocks where that leaves none of the SMs without one and its units suffice.
constexpr int kShort = 4096, kShortOfFew = 8192;
int short_ranks(int64_t segments, int64_t columns, int max_pages, int sms) {
  static_assert(kShortOfFew / kPageTokens <= 32, "a lane holds a page number");
  if (columns > 8 || max_pages > (segments <= sms ? kShortOfFew : kShort) / kPageTokens) return 0;
  const int64_t units = static_cast<int64_t>(max_pages) * kPageBlocks / 2;
  int ranks = 1;
  while (ranks < 8 && segments * ranks * 2 <= sms && units > kShortWarps * ranks) ranks *= 2;
  return ranks;
}

template <bool kBf16, int P, int kWarps>
cudaError_t short_t(const CacheAttnArgs& a, int ranks, cudaStream_t stream) {
  constexpr int kSmem = kWarps * 2 * Tile<P, 2>::kStage;
  static PerDeviceFlags flags;
  const cudaError_t e = ensure_dynamic_smem(cache_attn_short_kernel<kBf16, P, kWarps>, kSmem, flags);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ranks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(a.B) * a.H * ranks);
  config.blockDim = dim3(kWarps * 32);
  config.dynamicSmemBytes = kSmem;
  config.stream = stream;
  config.attrs = &attr;
  config.numAttrs = ranks > 1 ? 1 : 0;             // a cluster of one block takes longer to launch than a block
  const cudaError_t launched = cudaLaunchKernelEx(&config, cache_attn_short_kernel<kBf16, P, kWarps>, a);
  if (launched != cudaSuccess) cudaGetLastError();
  return launched;
}

template <bool kBf16, int P, int RW>
cudaError_t rows_t(CacheAttnArgs a, int sms, cudaStream_t stream) {
  using T = RowTile<P>;
  const int workers = sms * T::kBlocks;
  a.notes = static_cast<int>(cache_attn_notes(static_cast<int64_t>(a.B) * a.column_tiles * a.H, workers));
  static PerDeviceFlags flags;
  cudaError_t e = ensure_dynamic_smem(cache_attn_rows_kernel<kBf16, P, RW>, T::kSmem, flags);
  if (e != cudaSuccess) return e;
  cache_attn_rows_kernel<kBf16, P, RW><<<workers, kRowWarps * 32, T::kSmem, stream>>>(a);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  return join_t<kBf16, P, 16 * RW>(a, workers, stream);
}

template <bool kBf16, int P>
cudaError_t attn_p(const CacheAttnArgs& a, int sms, cudaStream_t stream) {
  const int64_t segments = static_cast<int64_t>(a.B) * a.H;
  if (const int ranks = short_ranks(segments, static_cast<int64_t>(a.T) * a.G, a.max_pages, sms))
    return segments > 2 * sms ? short_t<kBf16, P, 4>(a, ranks, stream) : short_t<kBf16, P, kShortWarps>(a, ranks, stream);
  // more than 8 columns: tiles of 64, or the one tile that holds them
  switch (cache_attn_columns(a.T, a.G)) {
    case 8: return attn_t<kBf16, P>(a, sms, stream);
    case 16: return rows_t<kBf16, P, 1>(a, sms, stream);
    case 32: return rows_t<kBf16, P, 2>(a, sms, stream);
    default: return rows_t<kBf16, P, 4>(a, sms, stream);
  }
}

}  // namespace

// Columns of a tile: new tokens of the query heads that share a key/value head
int cache_attn_columns(int T, int G) {
  const int64_t columns = static_cast<int64_t>(T) * G;
  return columns <= 8 ? 8 : columns <= 16 ? 16 : columns <= 32 ? 32 : 64;
}

size_t cache_attn_workspace_bytes(int B, int H, int G, int T, int D, int max_pages, int sms) {
  const int P = cache_columns(D);
  if (short_ranks(static_cast<int64_t>(B) * H, static_cast<int64_t>(T) * G, max_pages, sms)) return 0;
  const int tile = cache_attn_columns(T, G), width = static_cast<int64_t>(T) * G < tile ? T * G : tile;
  const int each = tile == 8 ? kWarpsOf8 : P == 64 ? RowTile<64>::kBlocks : RowTile<128>::kBlocks;
  const int64_t workers = static_cast<int64_t>(sms) * each;
  return static_cast<size_t>(workers) * (sizeof(Note) + 2 * width * part_pitch(P) * sizeof(float));
}

cudaError_t launch_cache_attn(CacheAttnArgs a, bool bf16, int sms, cudaStream_t stream) {
  if (a.B == 0 || a.T == 0) return cudaSuccess;
  const int64_t columns = cache_attn_columns(a.T, a.G), tiles = (static_cast<int64_t>(a.T) * a.G + columns - 1) / columns;
  if (tiles * columns * a.H * a.B > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  a.column_tiles = static_cast<int>(tiles);
  a.exponents = 0x64646464u;
  if (cache_columns(a.D) == 64) return bf16 ? attn_p<true, 64>(a, sms, stream) : attn_p<false, 64>(a, sms, stream);
  return bf16 ? attn_p<true, 128>(a, sms, stream) : attn_p<false, 128>(a, sms, stream);
}

}  // namespace rbf
