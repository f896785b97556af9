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

// Two 16-bit numbers as fp32
template <bool kBf16>
__device__ __forceinline__ void widen8(const uint4& raw, float (&x)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<kBf16>(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

// code + 128 of a value: nearest integer of x * (127 / amax), ties to even, both steps in fp32 (|code| <= 127: x / amax is at
// most 1, and the two roundings cannot lift 127 by half). Non-finite products have code 0; their block's scale is not finite.
__device__ __forceinline__ uint32_t code_of(float x, float inverse) {
  return static_cast<uint32_t>(__float2int_rn(__fmul_rn(x, inverse)) + 128) & 0xffu;
}

// One warp per block of 16 tokens that the new tokens touch, of one head's keys or values. The warp of the first block also
// stores what is left behind the last complete one: both use the rows of the incomplete block, which are read first.
template <bool kBf16, int P>
__global__ void __launch_bounds__(kWriteThreads) cache_append_kernel(const CacheAppendArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * (kWriteThreads / 32) + (threadIdx.x >> 5);
  const int j = static_cast<int>(unit % a.blocks);
  const int64_t head = unit / a.blocks;
  const int kv = static_cast<int>(head & 1);
  const int h = static_cast<int>((head >> 1) % a.H);
  const int64_t b64 = (head >> 1) / a.H;
  if (b64 >= a.B) return;
  const int b = static_cast<int>(b64);
  const CacheSpan span = cache_span(a.lengths, a.fresh, b, a.T, a.max_pages);
  if (span.fresh == 0) return;
  const int end = span.held + span.fresh;
  const int first = span.held / kBlockTokens;
  const uint16_t* src = static_cast<const uint16_t*>(kv ? a.v : a.k);
  const int64_t* st = kv ? a.vs : a.ks;
  src += b * st[0] + h * st[1];
  constexpr int kBytes = cache_page_bytes(P), kSlot = cache_slot_bytes(P);
  const int D = a.D;

  // columns 8 x ... of token `pos`: from the incomplete block or from the call's tokens
  auto load8 = [&](const uint8_t* tail, int pos, int col) -> uint4 {
    if (col >= D) return make_uint4(0, 0, 0, 0);
    if (pos < span.held) return *reinterpret_cast<const uint4*>(tail + ((pos % kBlockTokens) * P + col) * 2);
    return *reinterpret_cast<const uint4*>(src + static_cast<int64_t>(pos - span.held) * st[2] + col);
  };

  const int block = first + j;
  if ((block + 1) * static_cast<int64_t>(kBlockTokens) <= end) {
    uint8_t* page = const_cast<uint8_t*>(cache_page(a.pages, a.table, b, a.max_pages, a.num_pages, a.H, h, kBytes, block * kBlockTokens));
    if (page != nullptr) {
      const uint8_t* tail = page + kPageHeader + (kPageBlocks + kv) * kSlot;
      // lane (r, c): tokens r, r + kRows, ... of 8-column group c
      constexpr int kGroups = P / 8, kRows = 32 / kGroups, kPer = kBlockTokens / kRows;
      const int r = lane / kGroups, c = lane % kGroups;
      // keys: tokens r + i * kRows; values: four tokens of a quad belong to one lane, which transposes them in registers
      auto token = [&](int i) { return kv ? (i / 4) * 4 * kRows + r * 4 + i % 4 : i * kRows + r; };
      uint4 raw[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) raw[i] = load8(tail, block * kBlockTokens + token(i), c * 8);
      uint32_t top = 0;                             // magnitudes as integers: NaN is above infinity is above every number
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        float x[8];
        widen8<kBf16>(raw[i], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
      }
      top = __reduce_max_sync(0xffffffffu, top);
      const float amax = __uint_as_float(top);
      const bool finite = top < 0x7f800000u, held = amax >= kSmallestHeld;
      const float scale = !finite ? __uint_as_float(0x7fc00000u) : held ? __fdiv_rn(amax, 127.f) : 0.f;
      const float inverse = finite && held ? __fdiv_rn(127.f, amax) : 0.f;
      uint8_t* slot = page + kPageHeader + (block % kPageBlocks) * kSlot + kv * 16 * P;
      uint2 code[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        float x[8];
        widen8<kBf16>(raw[i], x);
        uint32_t w[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          w[e] = 0;
#pragma unroll
          for (int f = 0; f < 4; ++f) w[e] |= code_of(x[4 * e + f], inverse) << (8 * f);
        }
        code[i] = make_uint2(w[0], w[1]);
      }
      if (kv == 0) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int tok = token(i), half = (tok >> 1) & 1, g = (tok >> 2) * 2 + (tok & 1);
          *reinterpret_cast<uint2*>(slot + ((c / 8) * 2 + half) * 512 + g * 64 + (c % 8) * 8) = code[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < kPer; i += 4) {
          const int t = token(i) / 4;
#pragma unroll
          for (int e = 0; e < 2; ++e) {             // four tokens x four dims, transposed
            const uint32_t r0 = e ? code[i].y : code[i].x, r1 = e ? code[i + 1].y : code[i + 1].x;
            const uint32_t r2 = e ? code[i + 2].y : code[i + 2].x, r3 = e ? code[i + 3].y : code[i + 3].x;
            const uint32_t lo01 = __byte_perm(r0, r1, 0x5140), hi01 = __byte_perm(r0, r1, 0x7362);
            const uint32_t lo23 = __byte_perm(r2, r3, 0x5140), hi23 = __byte_perm(r2, r3, 0x7362);
            const uint4 out = make_uint4(__byte_perm(lo01, lo23, 0x5410), __byte_perm(lo01, lo23, 0x7632),
                                         __byte_perm(hi01, hi23, 0x5410), __byte_perm(hi01, hi23, 0x7632));
            const int d4 = c * 2 + e;               // group of four dims
            *reinterpret_cast<uint4*>(slot + (d4 / 8) * 512 + ((d4 % 8) * 4 + t) * 16) = out;
          }
        }
      }
      if (lane == 0) reinterpret_cast<float*>(page)[(block % kPageBlocks) * 2 + kv] = scale;
    }
  }
  if (j != 0 || end % kBlockTokens == 0) return;
  __syncwarp();                                     // the incomplete block's rows have been read
  const int last = end / kBlockTokens * kBlockTokens;
  uint8_t* page = const_cast<uint8_t*>(cache_page(a.pages, a.table, b, a.max_pages, a.num_pages, a.H, h, kBytes, last));
  if (page == nullptr) return;
  uint8_t* tail = page + kPageHeader + (kPageBlocks + kv) * kSlot;
  const int from = last > span.held ? last : span.held;
  for (int i = lane; i < (end - from) * (P / 8); i += 32) {
    const int pos = from + i / (P / 8), col = i % (P / 8) * 8;
    *reinterpret_cast<uint4*>(tail + ((pos % kBlockTokens) * P + col) * 2) = load8(tail, pos, col);
  }
}

// Four tokens (a quad of a block) x four columns of one head's keys and values per thread
template <bool kBf16, int P>
__global__ void __launch_bounds__(256) cache_read_kernel(const CacheReadArgs a) {
  constexpr int kBytes = cache_page_bytes(P), kSlot = cache_slot_bytes(P);
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int groups = a.D / 4;
  const int d = static_cast<int>(at % groups) * 4;
  const int quad = static_cast<int>(at / groups % a.quads);
  const int64_t head = at / groups / a.quads;
  if (head >= static_cast<int64_t>(a.B) * a.H) return;
  const int b = static_cast<int>(head / a.H), h = static_cast<int>(head % a.H);
  const int n = cache_span(a.lengths, nullptr, b, 0, a.max_pages).held;
  int first = a.first != nullptr ? a.first[b] : 0;
  const int64_t begin = first < 0 ? 0 : first;      // (a negative start reads from the first token on)
  const int64_t pos64 = (begin / 4 + quad) * 4;
  uint2 k[4], v[4];                                 // four columns of four tokens
#pragma unroll
  for (int r = 0; r < 4; ++r) k[r] = v[r] = make_uint2(0, 0);
  const int pos = static_cast<int>(pos64 < n ? pos64 : 0);
  const uint8_t* page = pos64 < n ? cache_page(a.pages, a.table, b, a.max_pages, a.num_pages, a.H, h, kBytes, pos) : nullptr;
  if (page != nullptr) {
    const int block = pos / kBlockTokens, in_block = pos % kBlockTokens;
    if (block < n / kBlockTokens) {
      const uint8_t* slot = page + kPageHeader + (block % kPageBlocks) * kSlot;
      const float2 scale = reinterpret_cast<const float2*>(page)[block % kPageBlocks];
      const uint4 w4 = *reinterpret_cast<const uint4*>(slot + 16 * P + d / 32 * 512 + (d % 32 / 4 * 4 + in_block / 4) * 16);
      const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int tok = in_block + r, half = (tok >> 1) & 1, g = (tok >> 2) * 2 + (tok & 1);
        const uint32_t kw = *reinterpret_cast<const uint32_t*>(slot + ((d / 64) * 2 + half) * 512 + g * 64 + d % 64);
        float kx[4], vx[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          kx[i] = static_cast<float>(static_cast<int>(kw >> (8 * i) & 0xffu) - 128) * scale.x;
          vx[i] = static_cast<float>(static_cast<int>(w[i] >> (8 * r) & 0xffu) - 128) * scale.y;
        }
        k[r] = make_uint2(pack2<kBf16>(kx[0], kx[1]), pack2<kBf16>(kx[2], kx[3]));
        v[r] = make_uint2(pack2<kBf16>(vx[0], vx[1]), pack2<kBf16>(vx[2], vx[3]));
      }
    } else {
      const uint8_t* tail = page + kPageHeader + kPageBlocks * kSlot;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (pos + r >= n) break;
        k[r] = *reinterpret_cast<const uint2*>(tail + ((in_block + r) * P + d) * 2);
        v[r] = *reinterpret_cast<const uint2*>(tail + kSlot + ((in_block + r) * P + d) * 2);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int64_t i = pos64 + r - begin;
    if (i < 0 || i >= a.count) continue;
    const int64_t to = (head * a.count + i) * a.D + d;
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.k) + to) = k[r];
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.v) + to) = v[r];
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
  const int64_t units = static_cast<int64_t>(a.B) * a.H * 2 * a.blocks, per = kWriteThreads / 32;
  cache_append_kernel<kBf16, P><<<static_cast<unsigned>((units + per - 1) / per), kWriteThreads, 0, stream>>>(a);
  return cudaGetLastError();
}
template <bool kBf16, int P>
cudaError_t read_t(const CacheReadArgs& a, cudaStream_t stream) {
  const int64_t threads = static_cast<int64_t>(a.B) * a.H * a.quads * (a.D / 4);
  cache_read_kernel<kBf16, P><<<static_cast<unsigned>((threads + 255) / 256), 256, 0, stream>>>(a);
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
