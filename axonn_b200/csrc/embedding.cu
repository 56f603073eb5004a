// Rows of a table by token, scaled, and the gradient of the table: the sums of the rows of equal tokens.
//
//   out_i = scale table[t_i];   dtable_v = scale sum_{i: t_i = v} dy_i   (nothing of the padding token)
// A token outside the table gives a row of NaN and has no gradient.  Sums are 32-bit, in the order of the tokens, and rounded once.
//
// A block per looked-up row; a block per 1024 columns of a row of the gradient, which goes over all tokens.
#include "common.cuh"

namespace axb {

constexpr int EMB_THREADS = 128, EMB_COLS = 8;

template <typename T> __device__ __forceinline__ float emb_value(T x) {
  if constexpr (__is_same(T, float)) return x;
  else if constexpr (__is_same(T, __half)) return __half2float(x);
  else return __bfloat162float(x);
}
template <typename T> __device__ __forceinline__ T emb_store(float x) {
  if constexpr (__is_same(T, float)) return x;
  else if constexpr (__is_same(T, __half)) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}

template <typename T, typename I>
__global__ void __launch_bounds__(EMB_THREADS)
embedding_kernel(const I* __restrict__ tokens, const T* __restrict__ table, long long pitch, int V, int H, float scale, T* __restrict__ out) {
  const long long t = tokens[blockIdx.x];
  T* to = out + static_cast<long long>(blockIdx.x) * H;
  const bool there = t >= 0 && t < V;
  const T* from = table + (there ? t : 0) * pitch;
  for (int c = threadIdx.x; c < H; c += EMB_THREADS) to[c] = there ? emb_store<T>(emb_value(from[c]) * scale) : emb_store<T>(__int_as_float(0x7fffffff));
}

template <typename T, typename I>
__global__ void __launch_bounds__(EMB_THREADS)
embedding_grad_kernel(const I* __restrict__ tokens, int n, const T* __restrict__ dy, long long pitch, int H, float scale, long long padding,
                      T* __restrict__ dtable) {
  __shared__ int s_at[EMB_THREADS];
  __shared__ int s_count[EMB_THREADS / 32];
  const long long v = blockIdx.x;
  const int first = blockIdx.y * EMB_THREADS * EMB_COLS + threadIdx.x, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  float sum[EMB_COLS] = {};
  for (int i = 0; i < n && v != padding; i += EMB_THREADS) {
    const int at = i + threadIdx.x;
    const bool mine = at < n && tokens[at] == v;
    const unsigned met = __ballot_sync(0xffffffffu, mine);
    __syncthreads();
    if (lane == 0) s_count[w] = __popc(met);
    __syncthreads();
    int base = 0, count = 0;
    for (int k = 0; k < EMB_THREADS / 32; ++k) { if (k < w) base += s_count[k]; count += s_count[k]; }
    if (count == 0) continue;
    if (mine) s_at[base + __popc(met & ((1u << lane) - 1u))] = at;
    __syncthreads();
    for (int k = 0; k < count; ++k) {
      const T* from = dy + s_at[k] * pitch;
#pragma unroll
      for (int c = 0; c < EMB_COLS; ++c) if (first + c * EMB_THREADS < H) sum[c] += emb_value(from[first + c * EMB_THREADS]);
    }
  }
#pragma unroll
  for (int c = 0; c < EMB_COLS; ++c) if (first + c * EMB_THREADS < H) dtable[v * H + first + c * EMB_THREADS] = emb_store<T>(sum[c] * scale);
}

template <typename T, typename I>
static int embedding(const void* tokens, long long n, const void* table, long long pitch, int V, int H, float scale, void* out, cudaStream_t s) {
  embedding_kernel<T, I><<<static_cast<unsigned>(n), EMB_THREADS, 0, s>>>(static_cast<const I*>(tokens), static_cast<const T*>(table), pitch, V, H,
                                                                        scale, static_cast<T*>(out));
  AXB_CUDA(cudaGetLastError());
  return 0;
}
template <typename T, typename I>
static int embedding_grad(const void* tokens, long long n, const void* dy, long long pitch, int V, int H, float scale, long long padding,
                          void* dtable, cudaStream_t s) {
  const dim3 grid(V, (H + EMB_THREADS * EMB_COLS - 1) / (EMB_THREADS * EMB_COLS));
  embedding_grad_kernel<T, I><<<grid, EMB_THREADS, 0, s>>>(static_cast<const I*>(tokens), static_cast<int>(n), static_cast<const T*>(dy), pitch, H,
                                                         scale, padding, static_cast<T*>(dtable));
  AXB_CUDA(cudaGetLastError());
  return 0;
}

}  // namespace axb

using namespace axb;

static int refused(const char* what, long long n, int V, int H, int dtype, int token_bytes) {
  if (n >= 0 && n <= 0x7fffffffll && V >= 1 && V <= (1 << 30) && H >= 1 && H <= (1 << 25) && dtype >= 0 && dtype <= 2 && (token_bytes == 4 || token_bytes == 8)) return 0;
  set_error("%s: %lld tokens of %d bytes, table %d x %d of type %d", what, n, token_bytes, V, H, dtype);
  return -1;
}

extern "C" int axb_embedding(const void* tokens, int token_bytes, long long n, const void* table, long long pitch, int V, int H, float scale,
                             void* out, int dtype, void* stream) {
  if (refused("embedding", n, V, H, dtype, token_bytes)) return -1;
  if (n == 0) return 0;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const auto go = token_bytes == 8 ? (dtype == 0 ? embedding<__nv_bfloat16, long long> : dtype == 1 ? embedding<__half, long long> : embedding<float, long long>)
                                   : (dtype == 0 ? embedding<__nv_bfloat16, int> : dtype == 1 ? embedding<__half, int> : embedding<float, int>);
  return go(tokens, n, table, pitch, V, H, scale, out, s);
}

extern "C" long long axb_embedding_grad_words(long long n, int V, int H) { return 1; }

extern "C" int axb_embedding_grad(const void* tokens, int token_bytes, long long n, const void* dy, long long pitch, int V, int H, float scale,
                                  long long padding, void* dtable, void* work, int dtype, void* stream) {
  if (refused("gradient of an embedding", n, V, H, dtype, token_bytes)) return -1;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const auto go = token_bytes == 8 ? (dtype == 0 ? embedding_grad<__nv_bfloat16, long long> : dtype == 1 ? embedding_grad<__half, long long> : embedding_grad<float, long long>)
                                   : (dtype == 0 ? embedding_grad<__nv_bfloat16, int> : dtype == 1 ? embedding_grad<__half, int> : embedding_grad<float, int>);
  return go(tokens, n, dy, pitch, V, H, scale, padding, dtable, s);
}
