// Log-probabilities of given tokens, entropy and best alternatives of rows of logits, and their gradient.
//
//   d_j = (z_j - m) scale, m = max z;  s = sum exp(d_j);  w = sum exp(d_j) d_j
//   log-probability of t: d_t - log s;  entropy: log s - w / s;  alternatives: the largest z, equal ones in their order
//   dz_j = scale ( sum_i g_i [j = t_i] - p_j ( sum_i g_i + h (d_j - log s + H) ) ),  p_j = exp(d_j) / s
// with g_i the gradients of the log-probabilities of the token and of the alternatives t_i, h that of the entropy H.
//
// A block per row, which reads it once for the maximum, once for the sums and once for every alternative.
#include "common.cuh"

namespace axb {

constexpr int TP_THREADS = 256, TP_MOST = 32;

struct TokenProbsArgs {
  const void* logits;
  long long batch_stride, row_stride;       // of logits, in values
  const long long* tokens;                  // or null
  long long token_batch_stride, token_stride;
  long long start, total;
  int per_batch, V, top, whole;
  float scale;
  long long ignored;
};

template <typename T> __device__ __forceinline__ float tp_value(const T* z, int j) {
  if constexpr (__is_same(T, float)) return z[j];
  else if constexpr (__is_same(T, __half)) return __half2float(z[j]);
  else return __bfloat162float(z[j]);
}
template <typename T> __device__ __forceinline__ T tp_store(float x) {
  if constexpr (__is_same(T, float)) return x;
  else if constexpr (__is_same(T, __half)) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}
// 32-bit key with the order of the numbers, a NaN above all of them; -0 counts as 0.
__device__ __forceinline__ uint32_t tp_key(float x) {
  if (x != x) return 0xff800001u;           // +inf has 0xff800000
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float tp_key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

__device__ __forceinline__ unsigned long long tp_block_max(unsigned long long v, unsigned long long* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  for (int i = 0; i < TP_THREADS / 32; ++i) v = max(v, red[i]);
  return v;
}
__device__ __forceinline__ float tp_block_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int i = 0; i < TP_THREADS / 32; ++i) v += red[i];
  return v;
}

template <typename T>
__global__ void __launch_bounds__(TP_THREADS)
token_probs_kernel(const TokenProbsArgs a, float* log_probs, float* entropy, float* top_log_probs, long long* top_tokens, float4* stats) {
  __shared__ unsigned long long red[TP_THREADS / 32];
  __shared__ float redf[TP_THREADS / 32];
  const int row = blockIdx.x, b = row / a.per_batch, r = row - b * a.per_batch;
  const T* z = static_cast<const T*>(a.logits) + b * a.batch_stride + r * a.row_stride;
  const long long token = a.tokens ? a.tokens[b * a.token_batch_stride + r * a.token_stride] : 0;
  if (a.tokens && token == a.ignored) {
    if (threadIdx.x == 0) {
      if (log_probs) log_probs[row] = 0.f;
      if (entropy) entropy[row] = 0.f;
      stats[row] = make_float4(0.f, 1.f, 0.f, 0.f);
    }
    if (threadIdx.x < a.top) {
      top_log_probs[static_cast<long long>(row) * a.top + threadIdx.x] = 0.f;
      top_tokens[static_cast<long long>(row) * a.top + threadIdx.x] = -1;
    }
    return;
  }
  // key of the largest number, NaN left out
  unsigned long long most = 0ull;
  for (int j = threadIdx.x; j < a.V; j += TP_THREADS) {
    const float x = tp_value(z, j);
    if (x == x) most = max(most, static_cast<unsigned long long>(tp_key(x)));
  }
  most = tp_block_max(most, red);
  const float m = most ? tp_key_value(static_cast<uint32_t>(most)) : -INFINITY, ref = m == -INFINITY ? 0.f : m;
  float s = 0.f, w = 0.f;
  for (int j = threadIdx.x; j < a.V; j += TP_THREADS) {
    const float d = (tp_value(z, j) - ref) * a.scale, e = __expf(d);
    s += e;
    if (e > 0.f) w += e * d;
  }
  s = tp_block_sum(s, redf);
  w = tp_block_sum(w, redf);
  const double log_s = log(static_cast<double>(s));
  const float H = static_cast<float>(log_s - static_cast<double>(w) / s);
  if (threadIdx.x == 0) {
    const long long t = token - a.start;
    float zt = a.tokens && t >= 0 && t < a.V ? tp_value(z, static_cast<int>(t)) : 0.f;
    if (a.tokens && (token < 0 || token >= a.total)) zt = __int_as_float(0x7fffffff);
    if (a.whole) {
      if (log_probs) log_probs[row] = static_cast<float>((static_cast<double>(zt) - m) * a.scale - log_s);
      if (entropy) entropy[row] = H;
    }
    stats[row] = make_float4(m, s, a.whole ? H : w, zt);
  }
  unsigned long long before = ~0ull;
  for (int i = 0; i < a.top; ++i) {
    unsigned long long best = 0ull;
    for (int j = threadIdx.x; j < a.V; j += TP_THREADS) {
      const unsigned long long k = static_cast<unsigned long long>(tp_key(tp_value(z, j))) << 32 | (0xffffffffu - j);
      if (k < before) best = max(best, k);
    }
    before = tp_block_max(best, red);
    if (threadIdx.x == 0) {
      const int j = static_cast<int>(0xffffffffu - static_cast<uint32_t>(before));
      const float x = tp_value(z, j);
      top_log_probs[static_cast<long long>(row) * a.top + i] = a.whole ? static_cast<float>((static_cast<double>(x) - m) * a.scale - log_s) : x;
      top_tokens[static_cast<long long>(row) * a.top + i] = a.start + j;
    }
  }
}

// out [rows, V] dense; stats (m, s, H) of the whole vocabulary; null gradients are zeros
template <typename T>
__global__ void __launch_bounds__(TP_THREADS)
token_probs_bwd_kernel(const TokenProbsArgs a, const float4* stats, const float* d_log_probs, const float* d_entropy, const float* d_top,
                       const long long* top_tokens, T* out) {
  __shared__ float s_g[TP_MOST + 1];
  __shared__ long long s_t[TP_MOST + 1];
  const int row = blockIdx.x, b = row / a.per_batch, r = row - b * a.per_batch;
  const T* z = static_cast<const T*>(a.logits) + b * a.batch_stride + r * a.row_stride;
  T* dz = out + static_cast<long long>(row) * a.V;
  const long long token = a.tokens ? a.tokens[b * a.token_batch_stride + r * a.token_stride] : 0;
  if (a.tokens && token == a.ignored) {
    for (int j = threadIdx.x; j < a.V; j += TP_THREADS) dz[j] = tp_store<T>(0.f);
    return;
  }
  const int n = 1 + (d_top ? a.top : 0);
  if (threadIdx.x < n) {
    const long long i = static_cast<long long>(row) * a.top + threadIdx.x - 1;
    float g = threadIdx.x ? d_top[i] : d_log_probs ? d_log_probs[row] : 0.f;
    if (threadIdx.x == 0 && d_log_probs && (token < 0 || token >= a.total)) g = __int_as_float(0x7fffffff);
    s_g[threadIdx.x] = g;
    s_t[threadIdx.x] = threadIdx.x ? top_tokens[i] - a.start : a.tokens ? token - a.start : -1;
  }
  __syncthreads();
  const float4 st = stats[row];
  const float log_s = static_cast<float>(log(static_cast<double>(st.y))), h = d_entropy ? d_entropy[row] : 0.f;
  float all = 0.f;
  for (int i = 0; i < n; ++i) all += s_g[i];
  for (int j = threadIdx.x; j < a.V; j += TP_THREADS) {
    const float d = (tp_value(z, j) - st.x) * a.scale, p = __expf(d) / st.y;
    float g = -p * (all + (p > 0.f ? h * (d - log_s + st.z) : 0.f));
    for (int i = 0; i < n; ++i) if (s_t[i] == j) g += s_g[i];
    dz[j] = tp_store<T>(g * a.scale);
  }
}

static int fill(TokenProbsArgs& a, const char* what, const void* logits, long long batch_stride, long long row_stride, const long long* tokens,
                long long token_batch_stride, long long token_stride, int batches, int per_batch, int V, long long start, long long total, int top,
                float scale, long long ignored, int whole, int dtype) {
  if (batches < 1 || per_batch < 1 || static_cast<long long>(batches) * per_batch > 0x7fffffffll || V < 1 || V > (1 << 30) || top < 0 ||
      top > TP_MOST || top > V || !(scale > 0.f) || dtype < 0 || dtype > 2) {
    set_error("%s: %d x %d rows of %d values, %d alternatives, scale %g, type %d", what, batches, per_batch, V, top, scale, dtype);
    return -1;
  }
  a = {logits, batch_stride, row_stride, tokens, token_batch_stride, token_stride, start, total, per_batch, V, top, whole, scale, ignored};
  return 0;
}

}  // namespace axb

using namespace axb;

extern "C" int axb_token_log_probs(const void* logits, long long batch_stride, long long row_stride, const long long* tokens,
                                   long long token_batch_stride, long long token_stride, float* log_probs, float* entropy,
                                   float* top_log_probs, long long* top_tokens, float* stats, int batches, int per_batch, int V, long long start,
                                   long long total, int top, float scale, long long ignored, int whole, int dtype, void* stream) {
  TokenProbsArgs a;
  if (fill(a, "token log-probabilities", logits, batch_stride, row_stride, tokens, token_batch_stride, token_stride, batches, per_batch, V,
           start, total, top, scale, ignored, whole, dtype)) return -1;
  const int rows = batches * per_batch;
  auto kernel = dtype == 0 ? token_probs_kernel<__nv_bfloat16> : dtype == 1 ? token_probs_kernel<__half> : token_probs_kernel<float>;
  kernel<<<rows, TP_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(a, log_probs, entropy, top_log_probs, top_tokens,
                                                                   reinterpret_cast<float4*>(stats));
  AXB_CUDA(cudaGetLastError());
  return 0;
}

extern "C" int axb_token_log_probs_bwd(const void* logits, long long batch_stride, long long row_stride, const long long* tokens,
                                       long long token_batch_stride, long long token_stride, const float* stats, const float* d_log_probs,
                                       const float* d_entropy, const float* d_top, const long long* top_tokens, void* out, int batches,
                                       int per_batch, int V, long long start, long long total, int top, float scale, long long ignored, int dtype,
                                       void* stream) {
  TokenProbsArgs a;
  if (fill(a, "gradient of token log-probabilities", logits, batch_stride, row_stride, tokens, token_batch_stride, token_stride, batches,
           per_batch, V, start, total, top, scale, ignored, 1, dtype)) return -1;
  const int rows = batches * per_batch;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const float4* st = reinterpret_cast<const float4*>(stats);
  if (dtype == 0) token_probs_bwd_kernel<<<rows, TP_THREADS, 0, s>>>(a, st, d_log_probs, d_entropy, d_top, top_tokens, static_cast<__nv_bfloat16*>(out));
  else if (dtype == 1) token_probs_bwd_kernel<<<rows, TP_THREADS, 0, s>>>(a, st, d_log_probs, d_entropy, d_top, top_tokens, static_cast<__half*>(out));
  else token_probs_bwd_kernel<<<rows, TP_THREADS, 0, s>>>(a, st, d_log_probs, d_entropy, d_top, top_tokens, static_cast<float*>(out));
  AXB_CUDA(cudaGetLastError());
  return 0;
}
