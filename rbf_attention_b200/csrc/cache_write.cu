// Tokens into the paged 8-bit cache (cache.cuh), out of it again, and pages to other places. All three move bytes once:
// writing a token reads 4 D bytes per head (a key and a value of 16 bits) and writes 2 D, reading is the reverse, a copied page
// is read and written. Roofline: HBM.
#include <cstdint>
#include <cuda_runtime.h>

#include "cache.cuh"
#include "launch.h"

namespace rbf {
namespace {

constexpr int kWriteThreads = 128;                 // four warps, a block of 16 tokens of one head each
// Blocks on an SM: a warp waits for one round of loads, eight of 16 bytes a lane, so as many as registers allow without much
// spilling. 8 x 16 heads x 8190 tokens written, of 128 columns and of 64: 124 us (6.5 TB/s) and 75 so, 134 and 84 with six blocks,
// 144 and 83 with ten.
constexpr int kWriteBlocks = 8;

template <bool kBf16>
__device__ __forceinline__ uint4 narrow8(const float (&x)[8]) {
  return make_uint4(pack2<kBf16>(x[0], x[1]), pack2<kBf16>(x[2], x[3]), pack2<kBf16>(x[4], x[5]), pack2<kBf16>(x[6], x[7]));
}

// code + 128 of four 16-bit numbers: nearest integers of x * (127 / amax), ties to even, both steps in fp32 (|code| <= 127: x / amax
// is at most 1, and the two roundings cannot lift 127 by half). Adding 1.5 * 2^23 leaves the integer in the low bits: a conversion
// runs at an eighth of the rate.
template <bool kBf16>
__device__ __forceinline__ uint32_t codes_of(uint32_t lo, uint32_t hi, float inverse) {
  constexpr float kLift = 12582912.f + 128.f;
  float2 x = unpack2<kBf16>(lo), y = unpack2<kBf16>(hi);
  fmul2(x.x, x.y, x.x, x.y, inverse, inverse);
  fmul2(y.x, y.y, y.x, y.y, inverse, inverse);
  // single additions: the compiler makes one rounding of a product and an addition of pairs
  auto lift = [&](float f) { return __float_as_uint(__fadd_rn(f, kLift)); };
  return __byte_perm(__byte_perm(lift(x.x), lift(x.y), 0x0040), __byte_perm(lift(y.x), lift(y.y), 0x0040), 0x5410);
}

// A warp's share of a block's keys or values: lane (r, c) has tokens r, r + kRows, ... of 8-column group c; of values, four tokens
// of a quad, which it transposes
template <int P, bool kValues>
struct Share {
  static constexpr int kGroups = P / 8, kRows = 32 / kGroups, kPer = kBlockTokens / kRows;
  uint4 raw[kPer];
  static __device__ __forceinline__ int column() { return (threadIdx.x & 31) % kGroups; }
  static __device__ __forceinline__ int token(int i) {
    const int r = static_cast<int>(threadIdx.x & 31) / kGroups;
    return kValues ? (i / 4) * 4 * kRows + r * 4 + i % 4 : i * kRows + r;
  }
  // The first `old` tokens are rows of `tail`, the others rows of `src`, `ld` apart (`src` is where the block's first token would be).
  __device__ __forceinline__ void load(const uint16_t* src, int64_t ld, const uint16_t* tail, int old, int D) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int t = token(i), col = column() * 8;
      const uint16_t* from = t < old ? tail + t * P : src + t * ld;
      raw[i] = col < D ? *reinterpret_cast<const uint4*>(from + col) : make_uint4(0, 0, 0, 0);
    }
  }
};

// Its codes and the block's scale into the cache
template <bool kBf16, int P, bool kValues>
__device__ __forceinline__ void write_block(const Share<P, kValues>& in, uint8_t* slot, float* scale_out) {
  using S = Share<P, kValues>;
  constexpr int kPer = S::kPer;
  const uint4(&raw)[kPer] = in.raw;
  const int lane = threadIdx.x & 31, c = S::column();
  auto token = [](int i) { return S::token(i); };
  uint32_t top = 0;                                 // magnitudes as integers: NaN is above infinity is above every number
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) top = __vmaxu2(top, w[e] & 0x7fff7fffu);
  }
  top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
  const float amax = unpack2<kBf16>(top).x;
  const bool finite = top < (kBf16 ? 0x7f80u : 0x7c00u), held = amax >= kSmallestHeld;
  const float inverse = finite && held ? __fdiv_rn(127.f, amax) : 0.f;
#pragma unroll
  for (int i = 0; i < kPer; i += 4) {               // four tokens at a time
    uint2 code[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint4 w = raw[i + k];
      // a block with a number that is not finite has codes of zero, and its scale makes them NaN
      code[k] = finite ? make_uint2(codes_of<kBf16>(w.x, w.y, inverse), codes_of<kBf16>(w.z, w.w, inverse))
                       : make_uint2(0x80808080u, 0x80808080u);
    }
    if constexpr (!kValues) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int tok = token(i + k), half = (tok >> 1) & 1, g = (tok >> 2) * 2 + (tok & 1);
        *reinterpret_cast<uint2*>(slot + ((c / 8) * 2 + half) * 512 + g * 64 + (c % 8) * 8) = code[k];
      }
    } else {
      const int t = token(i) / 4;
#pragma unroll
      for (int e = 0; e < 2; ++e) {                 // four tokens x four dims, transposed
        const uint32_t r0 = e ? code[0].y : code[0].x, r1 = e ? code[1].y : code[1].x;
        const uint32_t r2 = e ? code[2].y : code[2].x, r3 = e ? code[3].y : code[3].x;
        const uint32_t lo01 = __byte_perm(r0, r1, 0x5140), hi01 = __byte_perm(r0, r1, 0x7362);
        const uint32_t lo23 = __byte_perm(r2, r3, 0x5140), hi23 = __byte_perm(r2, r3, 0x7362);
        const uint4 out = make_uint4(__byte_perm(lo01, lo23, 0x5410), __byte_perm(lo01, lo23, 0x7632),
                                     __byte_perm(hi01, hi23, 0x5410), __byte_perm(hi01, hi23, 0x7632));
        const int d4 = c * 2 + e;                   // group of four dims
        *reinterpret_cast<uint4*>(slot + 16 * P + (d4 / 8) * 512 + ((d4 % 8) * 4 + t) * 16) = out;
      }
    }
  }
  if (lane == 0) scale_out[kValues] = !finite ? __uint_as_float(0x7fc00000u) : held ? __fdiv_rn(amax, 127.f) : 0.f;
}

// One warp per block of 16 tokens that the new tokens touch, of one head's keys or values - of 64 columns both, so that a warp
// has eight loads under way. Neighbours have the heads of a block, which are beside one another in what a projection writes (with
// the blocks of a head as neighbours 138 and 86 us). The warp of the first block also stores what is left behind the last
// complete one: both use the rows of the incomplete block, which are read first.
template <int P> constexpr bool kBothOf = P == 64;
template <bool kBf16, int P>
__global__ void __launch_bounds__(kWriteThreads, kWriteBlocks) cache_append_kernel(const CacheAppendArgs a) {
  constexpr bool kBoth = kBothOf<P>;
  constexpr int kBytes = cache_page_bytes(P), kSlot = cache_slot_bytes(P);
  const int lane = threadIdx.x & 31;
  const unsigned unit = blockIdx.x * (kWriteThreads / 32) + (threadIdx.x >> 5);          // below 2^31: 32-bit divisions
  const unsigned columns = kBoth ? a.H : 2 * a.H, slow = unit / columns, fast = unit - slow * columns;
  const bool values = !kBoth && fast >= static_cast<unsigned>(a.H);
  const int h = static_cast<int>(values ? fast - a.H : fast), b = static_cast<int>(slow / a.blocks);
  const int j = static_cast<int>(slow - static_cast<unsigned>(b) * a.blocks);
  if (b >= a.B) return;
  const CacheSpan span = cache_span(a.lengths, a.fresh, b, a.T, a.max_pages);
  if (span.fresh == 0) return;
  const int end = span.held + span.fresh, block = span.held / kBlockTokens + j;
  const uint16_t* k = static_cast<const uint16_t*>(a.k) + b * a.ks[0] + h * a.ks[1];
  const uint16_t* v = static_cast<const uint16_t*>(a.v) + b * a.vs[0] + h * a.vs[1];
  if ((block + 1) * static_cast<int64_t>(kBlockTokens) <= end) {
    uint8_t* page = const_cast<uint8_t*>(
        cache_page(a.pages, a.table, b, a.max_pages, a.num_pages, a.H, h, kBytes, block * kBlockTokens));
    if (page != nullptr) {
      const uint16_t* tail = reinterpret_cast<const uint16_t*>(page + kPageHeader + kPageBlocks * kSlot);
      uint8_t* slot = page + kPageHeader + (block % kPageBlocks) * kSlot;
      float* scales = reinterpret_cast<float*>(page) + (block % kPageBlocks) * 2;
      const int64_t at = static_cast<int64_t>(block) * kBlockTokens - span.held;
      const int old = static_cast<int>(at < 0 ? -at : 0);
      Share<P, false> keys;
      Share<P, true> vals;
      if (!values) keys.load(k + at * a.ks[2], a.ks[2], tail, old, a.D);
      if (kBoth || values) vals.load(v + at * a.vs[2], a.vs[2], tail + kSlot / 2, old, a.D);
      if (!values) write_block<kBf16>(keys, slot, scales);
      if (kBoth || values) write_block<kBf16>(vals, slot, scales);
    }
  }
  if (j != 0 || end % kBlockTokens == 0) return;
  __syncwarp();                                     // the incomplete block's rows have been read
  const int last = end / kBlockTokens * kBlockTokens;
  uint8_t* page = const_cast<uint8_t*>(cache_page(a.pages, a.table, b, a.max_pages, a.num_pages, a.H, h, kBytes, last));
  if (page == nullptr) return;
  const int from = last > span.held ? last : span.held;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    if (!kBoth && kv != values) continue;
    uint8_t* tail = page + kPageHeader + (kPageBlocks + kv) * kSlot;
    const uint16_t* src = kv ? v : k;
    const int64_t ld = kv ? a.vs[2] : a.ks[2];
    for (int i = lane; i < (end - from) * (P / 8); i += 32) {
      const int pos = from + i / (P / 8), col = i % (P / 8) * 8;
      uint4 x = make_uint4(0, 0, 0, 0);
      if (col < a.D) x = *reinterpret_cast<const uint4*>(src + static_cast<int64_t>(pos - span.held) * ld + col);
      *reinterpret_cast<uint4*>(tail + ((pos % kBlockTokens) * P + col) * 2) = x;
    }
  }
}

// (x0, x1) of two codes that are held as 2^23 + 128 + code, times the scale
__device__ __forceinline__ void scaled2(float& x0, float& x1, float a0, float a1, float scale) {
  fadd2(a0, a1, a0, a1, -8388736.f, -8388736.f);
  fmul2(x0, x1, a0, a1, scale, scale);
}

// Four tokens (a quad of a block) x eight columns of one head's keys and values per thread
template <bool kBf16, int P>
__global__ void __launch_bounds__(256) cache_read_kernel(const CacheReadArgs a) {
  constexpr int kBytes = cache_page_bytes(P), kSlot = cache_slot_bytes(P);
  const unsigned head = blockIdx.x / a.chunks;      // 32-bit divisions, these the same for the block
  const unsigned at = (blockIdx.x - head * a.chunks) * 256 + threadIdx.x, groups = a.D / 8, quad = at / groups;
  const int b = static_cast<int>(head / a.H), h = static_cast<int>(head - b * a.H), d = static_cast<int>(at - quad * groups) * 8;
  if (quad >= static_cast<unsigned>(a.quads)) return;
  const int n = cache_span(a.lengths, nullptr, b, 0, a.max_pages).held;
  const int first = a.first != nullptr ? a.first[b] : 0;
  const int64_t begin = first < 0 ? 0 : first;      // (a negative start reads from the first token on)
  const int64_t pos64 = (begin / 4 + quad) * 4;
  // byte i of a word under the exponent of 2^23: the float 2^23 + byte (a conversion runs at a quarter of the rate)
  auto lifted = [&](uint32_t word, int i) { return __uint_as_float(__byte_perm(word, a.exponent, 0x7440 + i)); };
  uint4 k[4], v[4];                                 // eight columns of four tokens
#pragma unroll
  for (int r = 0; r < 4; ++r) k[r] = v[r] = make_uint4(0, 0, 0, 0);
  const int pos = static_cast<int>(pos64 < n ? pos64 : 0);
  const uint8_t* page = pos64 < n ? cache_page(a.pages, a.table, b, a.max_pages, a.num_pages, a.H, h, kBytes, pos) : nullptr;
  if (page != nullptr) {
    const int block = pos / kBlockTokens, in_block = pos % kBlockTokens;
    if (block < n / kBlockTokens) {
      const uint8_t* slot = page + kPageHeader + (block % kPageBlocks) * kSlot;
      const float2 scale = reinterpret_cast<const float2*>(page)[block % kPageBlocks];
      uint4 w[2];                                   // word i: dim i of four tokens
      uint2 kw[4];                                  // of each token eight dims
#pragma unroll
      for (int e = 0; e < 2; ++e)
        w[e] = *reinterpret_cast<const uint4*>(slot + 16 * P + d / 32 * 512 + ((d % 32 / 4 + e) * 4 + in_block / 4) * 16);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int tok = in_block + r, half = (tok >> 1) & 1, g = (tok >> 2) * 2 + (tok & 1);
        kw[r] = *reinterpret_cast<const uint2*>(slot + ((d / 64) * 2 + half) * 512 + g * 64 + d % 64);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float kx[8], vx[8];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t words[4] = {w[e].x, w[e].y, w[e].z, w[e].w}, key = e ? kw[r].y : kw[r].x;
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            scaled2(kx[4 * e + i], kx[4 * e + i + 1], lifted(key, i), lifted(key, i + 1), scale.x);
            scaled2(vx[4 * e + i], vx[4 * e + i + 1], lifted(words[i], r), lifted(words[i + 1], r), scale.y);
          }
        }
        k[r] = narrow8<kBf16>(kx);
        v[r] = narrow8<kBf16>(vx);
      }
    } else {
      const uint8_t* tail = page + kPageHeader + kPageBlocks * kSlot;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (pos + r >= n) break;
        k[r] = *reinterpret_cast<const uint4*>(tail + ((in_block + r) * P + d) * 2);
        v[r] = *reinterpret_cast<const uint4*>(tail + kSlot + ((in_block + r) * P + d) * 2);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int64_t i = pos64 + r - begin;
    if (i < 0 || i >= a.count) continue;
    const int64_t to = (static_cast<int64_t>(head) * a.count + i) * a.D + d;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.k) + to) = k[r];
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.v) + to) = v[r];
  }
}

constexpr int kCopyThreads = 256;
constexpr int kCopyChunk = kCopyThreads * 4;        // 16-byte words that a block moves

__global__ void __launch_bounds__(kCopyThreads) cache_copy_kernel(const __grid_constant__ CacheCopyArgs a) {
  const int chunk = blockIdx.x % a.chunks, pair = blockIdx.x / a.chunks % a.count, layer = blockIdx.x / a.chunks / a.count;
  const uint4* src = reinterpret_cast<const uint4*>(a.pages) + (layer * a.num_pages + a.pair[pair].src) * a.words;
  uint4* dst = reinterpret_cast<uint4*>(a.pages) + (layer * a.num_pages + a.pair[pair].dst) * a.words;
  uint4 x[4];
  const int64_t i = static_cast<int64_t>(chunk) * kCopyChunk + threadIdx.x;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (i + j * kCopyThreads < a.words) x[j] = __ldcs(src + i + j * kCopyThreads);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (i + j * kCopyThreads < a.words) __stcs(dst + i + j * kCopyThreads, x[j]);
}

template <bool kBf16, int P>
cudaError_t append_t(const CacheAppendArgs& a, cudaStream_t stream) {
  const int64_t units = static_cast<int64_t>(a.B) * a.H * (kBothOf<P> ? 1 : 2) * a.blocks, per = kWriteThreads / 32;
  if (units > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  cache_append_kernel<kBf16, P><<<static_cast<unsigned>((units + per - 1) / per), kWriteThreads, 0, stream>>>(a);
  return cudaGetLastError();
}
template <bool kBf16, int P>
cudaError_t read_t(CacheReadArgs a, cudaStream_t stream) {
  const int64_t chunks = (static_cast<int64_t>(a.quads) * (a.D / 8) + 255) / 256, blocks = chunks * a.B * a.H;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  a.chunks = static_cast<unsigned>(chunks);
  a.exponent = 0x4b000000u;
  cache_read_kernel<kBf16, P><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_cache_append(const CacheAppendArgs& a, bool bf16, cudaStream_t stream) {
  if (a.B == 0 || a.T == 0) return cudaSuccess;
  if (cache_columns(a.D) == 64) return bf16 ? append_t<true, 64>(a, stream) : append_t<false, 64>(a, stream);
  return bf16 ? append_t<true, 128>(a, stream) : append_t<false, 128>(a, stream);
}

cudaError_t launch_cache_read(const CacheReadArgs& a, bool bf16, cudaStream_t stream) {
  if (a.B == 0 || a.count == 0) return cudaSuccess;
  if (cache_columns(a.D) == 64) return bf16 ? read_t<true, 64>(a, stream) : read_t<false, 64>(a, stream);
  return bf16 ? read_t<true, 128>(a, stream) : read_t<false, 128>(a, stream);
}

cudaError_t launch_cache_copy(CacheCopyArgs a, int layers, cudaStream_t stream) {
  if (a.count == 0 || layers == 0) return cudaSuccess;
  a.chunks = static_cast<int>((a.words + kCopyChunk - 1) / kCopyChunk);
  const int64_t blocks = static_cast<int64_t>(layers) * a.count * a.chunks;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  cache_copy_kernel<<<static_cast<unsigned>(blocks), kCopyThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace rbf
