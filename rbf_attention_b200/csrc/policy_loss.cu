// Log-probabilities of given tokens and the clipped policy loss with a KL term, for fine-tuning the language model on rewards:
//   lp = z[t] - lse(z),  r = e^(lp - old),  gain = min(r A, clip(r, 1 - low, 1 + high) A),
//   kl = e^(ref - lp) - (ref - lp) - 1,     loss = sum over rows of w (kl_weight kl - gain)
//   d loss / d lp = w (kl_weight (1 - e^(ref - lp)) - [r A <= clipped] r A) = c,   d loss / d z = c (onehot(t) - softmax(z))
// Everything but the row's lse is a handful of scalars per row, so the gradient is known as soon as the row has been read once:
// one kernel reads the logits and writes the gradient of the loss, as the cross entropy does. (Not of float16 logits, whose numbers
// end at 2^-24: there the factor that the loss is scaled by comes before the rounding, see loss_gradient_kernel.) Roofline: HBM. A block owns a
// row, reads it with an online maximum and sum and keeps it in shared memory where it fits; longer rows come a second time out
// of L2. The rows' bases may have any alignment: a row is a head of single elements up to the first 16-byte
// boundary, 16-byte words, and a tail. Sums over rows are in 64 bits and in the order of the rows of a block, then of the blocks.
// 16384 x 50304 bfloat16: 581 to 588 us, 5.6 TB/s = 86 % of a copy. The special-function unit is busy for 60 % of that, the issue slots
// for 47; a quarter of the exponentials by polynomials took 599 us, fetching the next row into shared memory word by word behind
// the gradient 616.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "launch.h"

namespace rbf {
namespace {

// A block's threads, and blocks of the loss kernel on an SM: a short row is little work between two barriers, so many small
// blocks share an SM (8000 rows of 8192 bfloat16: 100 us with 512 threads, 59 with 128). The threads go by the row's length alone:
// they decide the order of its sum, and a row has the same log-probability from both operators, with or without a gradient,
// among any number of rows.
constexpr int kLong = 512, kShort = 128;
constexpr int kShortBytes = 24 * 1024;              // of a row
constexpr int kBlocksOfShort = 8, kBlocksOfLong = 2;
// A staged row leaves room for a second block on the SM: of its 228 KB every block has 1 KB that is the system's, and its static arrays.
constexpr int kStageBytes = 228 * 1024 / 2 - 1024 - 512;
// Longer ones have the SM alone, unless all rows run at once two to an SM and unstaged (float32 x 50257: 5000 rows 396 us, read a
// second time by two blocks on an SM 453; 200 rows 26 and 23; 3000 x 100000 bfloat16 242 and 295).
constexpr int kAloneBytes = 226 * 1024;
constexpr double kLn2 = 0.6931471805599453;
constexpr int kCountHere = 8192;                    // rows up to which every block counts them by itself

__device__ __forceinline__ float pl_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int kDtype> struct Number;                // 0 bfloat16, 1 float16, 2 float32
template <> struct Number<0> {
  using type = uint16_t;
  static __device__ __forceinline__ float widen(uint16_t x) { return __uint_as_float(static_cast<uint32_t>(x) << 16); }
  static __device__ __forceinline__ uint16_t narrow(float x) { return __bfloat16_as_ushort(__float2bfloat16_rn(x)); }
};
template <> struct Number<1> {
  using type = uint16_t;
  static __device__ __forceinline__ float widen(uint16_t x) { return __half2float(__ushort_as_half(x)); }
  static __device__ __forceinline__ uint16_t narrow(float x) { return __half_as_ushort(__float2half_rn(x)); }
};
template <> struct Number<2> {
  using type = float;
  static __device__ __forceinline__ float widen(float x) { return x; }
  static __device__ __forceinline__ float narrow(float x) { return x; }
};

// The numbers of a 16-byte word
template <int kDtype>
__device__ __forceinline__ void widen16(const uint4& raw, float (&x)[kDtype == 2 ? 4 : 8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kDtype == 2) {
      x[i] = __uint_as_float(w[i]);
    } else {
      const float2 f = unpack2<kDtype == 0>(w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}

// sum of 2^(y - m) over values y = x * log2(e); m = -inf and s = 0 before any of them is above -inf
struct Online {
  float m = -INFINITY, s = 0.f;
  __device__ __forceinline__ void merge(float m2, float s2) {
    const float top = fmaxf(m, m2);
    if (top == -INFINITY) {                         // nothing above -inf yet; a NaN has to stay
      s += s2;
      return;
    }
    s = s * pl_ex2(m - top) + s2 * pl_ex2(m2 - top);
    m = top;
  }
  template <int kCount>
  __device__ __forceinline__ void add(const float (&x)[kCount]) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < kCount; ++i) top = fmaxf(top, x[i]);
    top *= kLog2e;
    if (top > m) {
      s *= pl_ex2(m - top);
      m = top;
    }
    const float neg = m == -INFINITY ? 0.f : -m;    // 2^-inf is zero, 2^NaN is NaN
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int i = 0; i + 1 < kCount; i += 2) {
      float y0, y1;
      ffma2_bcast(y0, y1, x[i], x[i + 1], kLog2e, neg);
      fadd2(s0, s1, s0, s1, pl_ex2(y0), pl_ex2(y1));
    }
    if constexpr (kCount % 2) s0 += pl_ex2(fmaf(x[kCount - 1], kLog2e, neg));
    s += s0 + s1;
  }
};

// Where a row's 16-byte words are: elements [0, head) and [body, cols) are single ones
template <typename T>
struct Cut {
  static constexpr int kPer = 16 / sizeof(T);
  int head, words, body;
  __device__ Cut(const T* row, int cols) {
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(row) / sizeof(T) % kPer);
    head = min(cols, off == 0 ? 0 : kPer - off);
    words = (cols - head) / kPer;
    body = head + words * kPer;
  }
};

// The row's maximum and sum, by all threads of the block; on return thread 0 (and every thread of warp 0) has them.
template <int kDtype, bool kStage, int kThreads>
__device__ __forceinline__ Online row_sum(const typename Number<kDtype>::type* x, int cols, uint4* stage) {
  using T = typename Number<kDtype>::type;
  __shared__ float s_m[kThreads / 32], s_s[kThreads / 32];
  const Cut<T> cut(x, cols);
  const uint4* words = reinterpret_cast<const uint4*>(x + cut.head);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Online sum;
#pragma unroll 4
  for (int c = tid; c < cut.words; c += kThreads) {
    const uint4 raw = kStage ? __ldcs(words + c) : words[c];
    if constexpr (kStage) stage[c] = raw;
    float v[Cut<T>::kPer];
    widen16<kDtype>(raw, v);
    sum.add(v);
  }
  const int single = tid < cut.head ? tid : cut.body + tid - cut.head;
  if (tid < cut.head + cols - cut.body) {
    const float v[1] = {Number<kDtype>::widen(x[single])};
    sum.add(v);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    sum.merge(__shfl_xor_sync(0xffffffffu, sum.m, o), __shfl_xor_sync(0xffffffffu, sum.s, o));
  if (lane == 0) {
    s_m[warp] = sum.m;
    s_s[warp] = sum.s;
  }
  __syncthreads();
  if (warp == 0) {
    sum.m = lane < kThreads / 32 ? s_m[lane] : -INFINITY;
    sum.s = lane < kThreads / 32 ? s_s[lane] : 0.f;
#pragma unroll
    for (int o = kThreads / 64; o > 0; o >>= 1)
      sum.merge(__shfl_xor_sync(0xffffffffu, sum.m, o), __shfl_xor_sync(0xffffffffu, sum.s, o));
  }
  return sum;
}

// Log-probability of a row's token in 64 bits: numbers of the size of the logits and of log2(cols) nearly cancel in it, and the
// loss compares it with others like it. The logits' factor is the one of the sum's terms, so that a shift of all logits cancels.
__device__ __forceinline__ double log_prob(float x, const Online& sum, float& lse2) {
  int e;
  const float f = frexpf(sum.s, &e);                // log2f is off by units of its result's last place: of [0.5, 1) it is small
  const double l = static_cast<double>(sum.m) + e + static_cast<double>(log2f(f));
  lse2 = static_cast<float>(l);
  return (static_cast<double>(x) * static_cast<double>(kLog2e) - l) * kLn2;
}

// Brings a row's 16-byte words into L2; nothing waits for it.
__device__ __forceinline__ void prefetch_l2(const void* p, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

__device__ __forceinline__ bool counts(const PolicyArgs& a, int64_t token) {
  return token != a.ignore_index && token >= 0 && token < a.cols;
}

template <int kDtype, int kThreads>
__global__ void __launch_bounds__(kThreads, 2048 / kThreads) token_log_probs_kernel(const PolicyArgs a) {
  using N = Number<kDtype>;
  using T = typename N::type;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t token = a.tokens[row];
    if (!counts(a, token)) {
      if (threadIdx.x == 0) a.log_probs[row] = 0.f;
      continue;
    }
    const T* x = static_cast<const T*>(a.logits) + row * a.ld;
    const Online sum = row_sum<kDtype, false, kThreads>(x, a.cols, nullptr);
    float lse2;
    if (threadIdx.x == 0) a.log_probs[row] = static_cast<float>(log_prob(N::widen(x[token]), sum, lse2));
    __syncthreads();                                // the warps' slots are used again
  }
}

// How many rows count: one number per block
__global__ void __launch_bounds__(kLong) policy_count_kernel(const PolicyArgs a) {
  constexpr int kThreads = kLong;
  grid_dependents_launch();
  __shared__ int s_n[kThreads / 32];
  int n = 0;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; r < a.rows; r += step)
    n += counts(a, a.tokens[r]);
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) s_n[threadIdx.x >> 5] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; ++w) n += s_n[w];
    a.counts[blockIdx.x] = n;
  }
}

template <int kDtype, bool kStage, int kThreads, int kBlocks>
__global__ void __launch_bounds__(kThreads, kBlocks) policy_loss_kernel(const PolicyArgs a) {
  using N = Number<kDtype>;
  using T = typename N::type;
  constexpr int V = Cut<T>::kPer;
  extern __shared__ uint4 s_row[];                  // kStage: the row's words, each kept by the thread that read it
  __shared__ float s_shift, s_slope;
  __shared__ int s_count;
  const int tid = threadIdx.x;
  grid_dependency_wait();
  if (a.weights == nullptr) {
    if (tid == 0) s_count = 0;
    __syncthreads();
    int n = 0;
    if (a.count_blocks > 0) {
      for (int i = tid; i < a.count_blocks; i += kThreads) n += a.counts[i];
    } else {
      for (int64_t r = tid; r < a.rows; r += kThreads) n += counts(a, a.tokens[r]);
    }
    n = __reduce_add_sync(0xffffffffu, n);
    if ((tid & 31) == 0 && n != 0) atomicAdd(&s_count, n);
    __syncthreads();
  }
  double loss = 0.0;                                // of this block's rows, thread 0
  if (a.weights == nullptr && s_count == 0) loss = __longlong_as_double(0x7ff8000000000000ll);      // the mean of nothing
  int64_t next_token = blockIdx.x < a.rows ? a.tokens[blockIdx.x] : 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.logits) + row * a.ld;
    T* dx = static_cast<T*>(a.dlogits) + row * a.ld_out;
    const Cut<T> cut(x, a.cols);
    const int64_t token = next_token;
    const bool counted = counts(a, token), more = row + gridDim.x < a.rows;
    if (more) next_token = a.tokens[row + gridDim.x];
    if (counted) {
      float mine = 0.f, A = 0.f, old = 0.f, ref = 0.f, w = 0.f;
      if (tid == 0) {                               // asked for before the row, not after its sum (16384 x 50304: 600 -> 581 us)
        mine = N::widen(x[token]);
        A = a.advantages[row];
        old = a.old_log_probs[row];
        if (a.ref_log_probs != nullptr) ref = a.ref_log_probs[row];
        w = a.weights != nullptr ? a.weights[row] : 1.f / static_cast<float>(s_count);
      }
      const Online sum = row_sum<kDtype, kStage, kThreads>(x, a.cols, s_row);
      // a staged row has been read: the block's next one comes into L2 while this one is reduced and its gradient written
      if (kStage && tid == kThreads - 32 && more && counts(a, next_token)) {
        const T* next = x + static_cast<int64_t>(gridDim.x) * a.ld;
        const Cut<T> next_cut(next, a.cols);
        if (next_cut.words > 0) prefetch_l2(next + next_cut.head, next_cut.words * 16);
      }
      if (tid == 0) {
        float lse2;
        const double lp = log_prob(mine, sum, lse2);
        const float r = expf(static_cast<float>(lp - old));
        const float plain = r * A, clipped = fminf(fmaxf(r, 1.f - a.clip_low), 1.f + a.clip_high) * A;
        float value = -fminf(plain, clipped), slope = plain <= clipped ? -plain : 0.f;
        if (plain != plain) value = slope = plain;  // fminf would pass over it
        if (a.ref_log_probs != nullptr) {
          const float gap = static_cast<float>(ref - lp), away = expf(gap);
          value = fmaf(a.kl_weight, away - gap - 1.f, value);
          slope = fmaf(a.kl_weight, 1.f - away, slope);
        }
        a.log_probs[row] = static_cast<float>(lp);
        loss += static_cast<double>(w) * static_cast<double>(value);
        s_slope = w * slope;
        s_shift = -lse2;
        if (a.row_stats != nullptr) a.row_stats[row] = make_float2(-lse2, w * slope);
      }
    } else if (tid == 0) {
      a.log_probs[row] = 0.f;
      if (a.row_stats != nullptr) a.row_stats[row] = make_float2(0.f, 0.f);
    }
    if (a.dlogits == nullptr) {
      __syncthreads();                              // the warps' slots are used again
      continue;
    }
    uint4* out = reinterpret_cast<uint4*>(dx + cut.head);
    const int single = tid < cut.head ? tid : cut.body + tid - cut.head;
    const bool has_single = tid < cut.head + a.cols - cut.body;
    if (!counted) {
      for (int c = tid; c < cut.words; c += kThreads) out[c] = make_uint4(0, 0, 0, 0);
      if (has_single) dx[single] = N::narrow(0.f);
      continue;
    }
    __syncthreads();
    const float shift = s_shift, slope = s_slope;
    const int at = static_cast<int>(token) - cut.head, word = at >= 0 ? at / V : -1, in_word = at >= 0 ? at % V : 0;
    const uint4* words = reinterpret_cast<const uint4*>(x + cut.head);
#pragma unroll 2
    for (int c = tid; c < cut.words; c += kThreads) {
      uint4 raw;
      if constexpr (kStage) raw = s_row[c];
      else raw = words[c];
      float v[V];
      widen16<kDtype>(raw, v);
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        float y0, y1;
        ffma2_bcast(y0, y1, v[i], v[i + 1], kLog2e, shift);
        fmul2(v[i], v[i + 1], pl_ex2(y0), pl_ex2(y1), -slope, -slope);
      }
      if (c == word) {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (i == in_word) v[i] += slope;
      }
      uint4 y;
      if constexpr (kDtype == 2) {
        y = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
      } else {
        constexpr bool kBf16 = kDtype == 0;
        y = make_uint4(pack2<kBf16>(v[0], v[1]), pack2<kBf16>(v[2], v[3]), pack2<kBf16>(v[4 % V], v[5 % V]),
                       pack2<kBf16>(v[6 % V], v[7 % V]));
      }
      __stcs(out + c, y);
    }
    if (has_single) {
      float v = -slope * pl_ex2(fmaf(N::widen(x[single]), kLog2e, shift));
      if (single == token) v += slope;
      dx[single] = N::narrow(v);
    }
    __syncthreads();                                // s_shift, s_slope and the warps' slots are used again
  }
  if (tid == 0) a.sums[blockIdx.x] = loss;
  grid_dependents_launch();
}

// The blocks' sums in their order
__global__ void __launch_bounds__(32) policy_finish_kernel(const PolicyArgs a, const int blocks) {
  grid_dependency_wait();
  double sum = 0.0;
  for (int i = threadIdx.x; i < blocks; i += 32) sum += a.sums[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (threadIdx.x != 0) return;
  *a.loss = static_cast<float>(sum);
}

// The gradient of a loss whose rows are c (onehot(t) - softmax(z)), from a number pair per row (-log2 of the row's sum of e^z, c) and
// the factor that reaches the loss, which is multiplied in before the rounding: float16's numbers end at 2^-24, and the elements
// of a mean over many rows are smaller than that (16384 rows of 50257: 99.5 % of them) until a loss scale lifts them. Roofline: HBM,
// a read and a write: 16384 x 50304 in 525 us, 6.3 TB/s = 96 % of a copy; forward and backward 888 us, where a gradient that is
// rounded first takes 646. A block has 16 KB of a row; rows that do not count are zeros and are not read.
constexpr int kGradThreads = 256, kGradPer = 4, kGradWords = kGradPer * kGradThreads;
__global__ void __launch_bounds__(kGradThreads) loss_gradient_kernel(const LossGradientArgs a) {
  using N = Number<1>;
  using T = N::type;
  constexpr int V = Cut<T>::kPer;
  const int tid = threadIdx.x;
  const float factor = *a.factor;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const T* x = static_cast<const T*>(a.logits) + row * a.ld;
    T* dx = static_cast<T*>(a.dlogits) + row * a.ld_out;
    const int64_t token = a.tokens[row];
    const float2 stats = a.row_stats[row];
    const bool counted = token != a.ignore_index && token >= 0 && token < a.cols;
    const float shift = stats.x, slope = stats.y * factor;
    const Cut<T> cut(x, a.cols);
    const uint4* words = reinterpret_cast<const uint4*>(x + cut.head);
    uint4* out = reinterpret_cast<uint4*>(dx + cut.head);
    const int at = static_cast<int>(token) - cut.head, word = counted && at >= 0 ? at / V : -1, in_word = at % V;
    const int first = static_cast<int>(blockIdx.x) * kGradWords + tid;
    uint4 raw[kGradPer];
#pragma unroll
    for (int k = 0; k < kGradPer; ++k)
      if (counted && first + k * kGradThreads < cut.words) raw[k] = __ldcs(words + first + k * kGradThreads);
#pragma unroll
    for (int k = 0; k < kGradPer; ++k) {
      const int c = first + k * kGradThreads;
      uint4 y = make_uint4(0, 0, 0, 0);
      if (c >= cut.words) break;
      if (counted) {
        float v[V];
        widen16<1>(raw[k], v);
#pragma unroll
        for (int i = 0; i < V; i += 2) {
          float y0, y1;
          ffma2_bcast(y0, y1, v[i], v[i + 1], kLog2e, shift);
          fmul2(v[i], v[i + 1], pl_ex2(y0), pl_ex2(y1), -slope, -slope);
        }
        if (c == word) {
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (i == in_word) v[i] += slope;
        }
        y = make_uint4(pack2<false>(v[0], v[1]), pack2<false>(v[2], v[3]), pack2<false>(v[4], v[5]), pack2<false>(v[6], v[7]));
      }
      __stcs(out + c, y);
    }
    if (blockIdx.x == 0 && tid < cut.head + a.cols - cut.body) {
      const int single = tid < cut.head ? tid : cut.body + tid - cut.head;
      float v = 0.f;
      if (counted) {
        v = -slope * pl_ex2(fmaf(N::widen(x[single]), kLog2e, shift));
        if (single == token) v += slope;
      }
      dx[single] = N::narrow(v);
    }
  }
}

template <int kDtype, int kThreads>
cudaError_t log_probs_t(const PolicyArgs& a, int sms, cudaStream_t stream) {
  const int64_t most = static_cast<int64_t>(sms) * (2048 / kThreads);
  token_log_probs_kernel<kDtype, kThreads><<<static_cast<unsigned>(a.rows < most ? a.rows : most), kThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

template <int kDtype, bool kStage, int kThreads, int kBlocks>
cudaError_t policy_t(PolicyArgs a, int sms, cudaStream_t stream) {
  const int64_t most = static_cast<int64_t>(sms) * kBlocks;
  const int blocks = a.rows == 0 ? 1 : static_cast<int>(a.rows < most ? a.rows : most);
  const int64_t wanted = (a.rows + kLong - 1) / kLong;
  a.count_blocks = a.rows <= kCountHere ? 0 : static_cast<int>(wanted < sms ? wanted : sms);
  cudaError_t e;
  if (a.weights == nullptr && a.count_blocks > 0) {
    policy_count_kernel<<<a.count_blocks, kLong, 0, stream>>>(a);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
  }
  size_t smem = 0;
  if constexpr (kStage) {
    constexpr int kMost = kBlocks == 1 ? kAloneBytes : kStageBytes;
    static PerDeviceFlags flags;
    if ((e = ensure_dynamic_smem(policy_loss_kernel<kDtype, kStage, kThreads, kBlocks>, kMost, flags)) != cudaSuccess) return e;
    smem = (static_cast<size_t>(a.cols) * sizeof(typename Number<kDtype>::type) + 15) / 16 * 16;
  }
  e = launch_dependent(policy_loss_kernel<kDtype, kStage, kThreads, kBlocks>, dim3(blocks), kThreads, smem, stream, a);
  if (e != cudaSuccess) return e;
  return launch_dependent(policy_finish_kernel, dim3(1), 32, 0, stream, a, blocks);
}

template <int kDtype>
cudaError_t log_probs_of(const PolicyArgs& a, int sms, cudaStream_t stream) {
  const int64_t bytes = static_cast<int64_t>(a.cols) * sizeof(typename Number<kDtype>::type);
  return bytes <= kShortBytes ? log_probs_t<kDtype, kShort>(a, sms, stream) : log_probs_t<kDtype, kLong>(a, sms, stream);
}
template <int kDtype>
cudaError_t policy_of(const PolicyArgs& a, int sms, cudaStream_t stream) {
  const int64_t bytes = static_cast<int64_t>(a.cols) * sizeof(typename Number<kDtype>::type);
  const bool stage = a.dlogits != nullptr;
  if (bytes <= kShortBytes)
    return stage ? policy_t<kDtype, true, kShort, kBlocksOfShort>(a, sms, stream)
                 : policy_t<kDtype, false, kShort, kBlocksOfShort>(a, sms, stream);
  if (stage && bytes <= kStageBytes) return policy_t<kDtype, true, kLong, kBlocksOfLong>(a, sms, stream);
  if (stage && bytes <= kAloneBytes && a.rows > kBlocksOfLong * sms) return policy_t<kDtype, true, kLong, 1>(a, sms, stream);
  return policy_t<kDtype, false, kLong, kBlocksOfLong>(a, sms, stream);
}

}  // namespace

int policy_blocks(int sms) { return sms * kBlocksOfShort; }

cudaError_t launch_token_log_probs(const PolicyArgs& a, int dtype, int sms, cudaStream_t stream) {
  if (a.rows == 0) return cudaSuccess;
  switch (dtype) {
    case 0: return log_probs_of<0>(a, sms, stream);
    case 1: return log_probs_of<1>(a, sms, stream);
    case 2: return log_probs_of<2>(a, sms, stream);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_loss_gradient(const LossGradientArgs& a, cudaStream_t stream) {
  if (a.rows == 0) return cudaSuccess;
  const int words = a.cols / 8, chunks = words / kGradWords + 1;
  const dim3 grid(chunks, static_cast<unsigned>(a.rows < 65535 ? a.rows : 65535));
  loss_gradient_kernel<<<grid, kGradThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_policy_loss(const PolicyArgs& a, int dtype, int sms, cudaStream_t stream) {
  switch (dtype) {
    case 0: return policy_of<0>(a, sms, stream);
    case 1: return policy_of<1>(a, sms, stream);
    case 2: return policy_of<2>(a, sms, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace rbf
