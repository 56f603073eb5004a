// Selection of beam search: of all continuations of the beams of a prompt, value = score + logit - log sum exp(logits of the beam), the
// `beams` best, equal values in the order of (beam, token).
//
// Bound by reading the logits once.  A first launch cuts every beam's row into parts: each warp keeps a running maximum and sum of
// exponentials per lane and the best logits of what it has seen, sorted, one per lane; a value that does not beat the worst of them costs
// a comparison per eight.  The order within a beam is that of its logits, so that nothing has to be known of the sum.  A second launch
// puts the parts of a beam together and merges the beams' lists.  Sums and values there are 64-bit: the order of two beams' tokens
// depends on differences of their sums' logarithms that 32-bit values of twenty or so round away.
//
// A value that is not a number counts as -inf, and so do a score of +inf and every value of a beam whose sum is none.  Of a beam that has ended only the
// end token goes on, with the beam's score.
#include "common.cuh"

namespace axb {

constexpr int BEAM_MOST = 32;            // beams: a warp's list has one entry per lane
constexpr int BEAM_WARPS = 8;
constexpr int BEAM_PARTS = 32;           // of a row, at most: one per lane
constexpr float LOG2E = 1.4426950408889634f;

struct BeamArgs {
  const void* logits;                    // [B, K, V]
  const float* scores;                   // [B, K]
  const unsigned char* done;             // [B, K] or null
  float* out_scores;
  long long* out_tokens;
  int* out_parents;
  unsigned char* out_done;
  // of every row and part: K keys and K tokens, best first, and (maximum, sum)
  uint32_t* keys;
  int* tokens;
  float2* sums;
  int B, K, V, eos, parts, part_steps;   // part_steps: steps of 256 values of a warp in a part
};

// 32-bit key with the order of the numbers; 0 is below all of them.  -0 counts as 0.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// A warp's list: lane i has the i-th best (larger key, then lower token); key 0: none.
struct BestList {
  uint32_t key = 0u;
  int token = -1;
  __device__ __forceinline__ void insert(uint32_t k, int t, int lane) {
    const uint32_t better = __ballot_sync(0xffffffffu, key > k || (key == k && key != 0u && token < t));
    const int at = __popc(better);
    const uint32_t up_key = __shfl_up_sync(0xffffffffu, key, 1);
    const int up_token = __shfl_up_sync(0xffffffffu, token, 1);
    if (lane > at) { key = up_key; token = up_token; }
    else if (lane == at) { key = k; token = t; }
  }
};

template <typename T> __device__ __forceinline__ float logit_value(T x);
template <> __device__ __forceinline__ float logit_value(float x) { return x; }
template <> __device__ __forceinline__ float logit_value(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float logit_value(__half x) { return __half2float(x); }

// One step of a warp is 256 values.  VEC: every row starts on 16 bytes, lane has values 8 lane ..; otherwise lane has values lane, lane +
// 32 ... - for all rows of a call alike, so that equal rows have equal sums.
template <typename T, bool VEC> __device__ __forceinline__ int value_index(int lane, int j) { return VEC ? lane * 8 + j : j * 32 + lane; }
template <typename T, bool VEC> __device__ __forceinline__ void load_step(const T* row, int base, int V, int lane, float (&x)[8]) {
  if (VEC && base + 256 <= V) {
    T t[8];
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
      reinterpret_cast<uint4*>(t)[i] = __ldg(reinterpret_cast<const uint4*>(row + base + lane * 8) + i);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = logit_value(t[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = base + value_index<T, VEC>(lane, j);
      x[j] = i < V ? logit_value(row[i]) : __int_as_float(0xff800000);
    }
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * BEAM_WARPS) beam_rows_kernel(const BeamArgs a) {
  __shared__ uint32_t s_key[BEAM_WARPS][BEAM_MOST];
  __shared__ int s_token[BEAM_WARPS][BEAM_MOST];
  __shared__ float2 s_sum[BEAM_WARPS];
  pdl_launch_next();
  pdl_wait();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, K = a.K, V = a.V;
  const long long row_at = blockIdx.x;
  if (a.done && a.done[row_at]) return;
  const T* row = static_cast<const T*>(a.logits) + row_at * V;
  const int first = blockIdx.y * a.part_steps * BEAM_WARPS * 256, last = min(static_cast<long long>(V), first + a.part_steps * BEAM_WARPS * 256ll);
  float m = -3.4028234663852886e38f, sum = 0.f;
  BestList best;
  uint32_t worst = 0u;                   // key of the list's last entry: 0 while it is not full
  bool begun = false;
  int base = first + w * 256;
  float next[8];
  if (base < last) load_step<T, VEC>(row, base, V, lane, next);
  for (; base < last; base += BEAM_WARPS * 256) {
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = next[j];
    if (base + BEAM_WARPS * 256 < last) load_step<T, VEC>(row, base + BEAM_WARPS * 256, V, lane, next);
    float top = x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) top = fmaxf(top, x[j]);
    if (top > m) { sum *= exp2f((m - top) * LOG2E); m = top; }
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += exp2f((x[j] - m) * LOG2E);
    uint32_t above = worst;              // keys above this are looked at
    if (!begun) {
      // the K-th largest of the lanes' maxima: at least K values reach it, and few others do
      begun = true;
      uint32_t k = order_key(top);
#pragma unroll
      for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int o = size >> 1; o > 0; o >>= 1) {
          const uint32_t other = __shfl_xor_sync(0xffffffffu, k, o);
          const bool larger_here = ((lane & size) == 0) == ((lane & o) == 0);
          k = larger_here ? max(k, other) : min(k, other);
        }
      above = __shfl_sync(0xffffffffu, k, K - 1);
      above -= above != 0u;
    }
    if (__any_sync(0xffffffffu, order_key(top) > above)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int t = base + value_index<T, VEC>(lane, j);
        const uint32_t k = t < V ? order_key(x[j]) : 0u;
        uint32_t hits = __ballot_sync(0xffffffffu, k > above);
        while (hits) {
          const int from = __ffs(hits) - 1;
          hits &= hits - 1;
          best.insert(__shfl_sync(0xffffffffu, k, from), __shfl_sync(0xffffffffu, t, from), lane);
        }
      }
      // what came in at an equal key keeps the order of the tokens: insert compares both
      worst = __shfl_sync(0xffffffffu, best.key, K - 1);
    }
  }
  // the warps' lists, one by one: a list ends where its entries no longer come in
  if (lane < K) { s_key[w][lane] = best.key; s_token[w][lane] = best.token; }
  float top = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  sum *= exp2f((m - top) * LOG2E);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_sum[w] = make_float2(top, sum);
  __syncthreads();
  if (w) return;
  for (int i = 1; i < BEAM_WARPS; ++i)
    for (int e = 0; e < K; ++e) {
      const uint32_t k = s_key[i][e], k_worst = __shfl_sync(0xffffffffu, best.key, K - 1);
      const int t = s_token[i][e], t_worst = __shfl_sync(0xffffffffu, best.token, K - 1);
      if (k == 0u || k < k_worst || (k == k_worst && t > t_worst)) break;
      best.insert(k, t, lane);
    }
  const size_t o = (row_at * a.parts + blockIdx.y) * K;
  if (lane < K) { a.keys[o + lane] = best.key; a.tokens[o + lane] = best.token; }
  float2 s = lane < BEAM_WARPS ? s_sum[lane] : make_float2(-3.4028234663852886e38f, 0.f);
  top = s.x;
#pragma unroll
  for (int d = 4; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  sum = s.y * exp2f((s.x - top) * LOG2E);
#pragma unroll
  for (int d = 4; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (lane == 0) a.sums[row_at * a.parts + blockIdx.y] = make_float2(top, sum);
}

// One block per prompt.  A warp per beam: the beam's sum, its parts' lists merged; then the beams' lists, K rounds, a lane per beam.
__global__ void __launch_bounds__(32 * BEAM_WARPS) beam_select_kernel(const BeamArgs a) {
  __shared__ double s_value[BEAM_MOST][BEAM_MOST];
  __shared__ int s_token[BEAM_MOST][BEAM_MOST];
  pdl_launch_next();
  pdl_wait();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, K = a.K, V = a.V, b = blockIdx.x;
  const double none = -__longlong_as_double(0x7ff0000000000000ll);
  for (int row = w; row < K; row += BEAM_WARPS) {
    const size_t at = static_cast<size_t>(b) * K + row;
    const double score = a.scores[at] < -none ? a.scores[at] : none;      // no sum of logarithms of probabilities is +inf
    double value = none;
    int token = -1;                      // this lane's entry of the beam's list
    if (a.done && a.done[at]) {
      if (score > none) {                // the end token, then the others in their order
        value = lane == 0 ? score : none;
        token = lane == 0 ? a.eos : lane - (lane <= a.eos);
      }
    } else {
      float2 s = lane < a.parts ? a.sums[at * a.parts + lane] : make_float2(-3.4028234663852886e38f, 0.f);
      float top = s.x;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      double sum = static_cast<double>(s.y) * static_cast<double>(exp2f((s.x - top) * LOG2E));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const double log_sum = log(sum) + static_cast<double>(top);
      BestList best;
      if (lane < K) { best.key = a.keys[at * a.parts * K + lane]; best.token = a.tokens[at * a.parts * K + lane]; }
      for (int p = 1; p < a.parts; ++p) {
        // the part's list, an entry per lane; those that come in are its first ones
        const uint32_t k = lane < K ? a.keys[(at * a.parts + p) * K + lane] : 0u;
        const int t = lane < K ? a.tokens[(at * a.parts + p) * K + lane] : -1;
        for (int e = 0; e < K; ++e) {
          const uint32_t ke = __shfl_sync(0xffffffffu, k, e), k_worst = __shfl_sync(0xffffffffu, best.key, K - 1);
          const int te = __shfl_sync(0xffffffffu, t, e), t_worst = __shfl_sync(0xffffffffu, best.token, K - 1);
          if (ke == 0u || ke < k_worst || (ke == k_worst && te > t_worst)) break;
          best.insert(ke, te, lane);
        }
      }
      if (best.key) { value = score + (static_cast<double>(key_value(best.key)) - log_sum); token = best.token; }
      if (!(value == value)) value = none;
    }
    if (__shfl_sync(0xffffffffu, value, 0) == none) token = lane;      // nothing of this beam counts: its first tokens
    if (token >= V) token = -1;
    if (lane < K) { s_value[row][lane] = value; s_token[row][lane] = token; }
  }
  __syncthreads();
  if (w) return;
  int at = 0;                            // of this lane's beam
  for (int i = 0; i < K; ++i) {
    const bool left = lane < K && at < K && s_token[lane][at] >= 0;
    double value = left ? s_value[lane][at] : none;
    // the best value, then the lowest beam: within a beam the list has the order of the tokens
    unsigned candidates = __ballot_sync(0xffffffffu, left);
    double top = value;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { const double v = __shfl_xor_sync(0xffffffffu, top, o); top = v > top ? v : top; }
    candidates &= __ballot_sync(0xffffffffu, left && value == top);
    const int row = __ffs(candidates) - 1;
    if (lane == row) {
      const size_t o = static_cast<size_t>(b) * K + i;
      const int token = s_token[lane][at];
      a.out_scores[o] = static_cast<float>(value);
      a.out_tokens[o] = token;
      a.out_parents[o] = lane;
      if (a.done) a.out_done[o] = a.done[static_cast<size_t>(b) * K + lane] || token == a.eos;
      ++at;
    }
  }
}

static int beam_parts(int rows, int V) {
  // enough blocks for every SM to have a few, of at least a step per warp
  const int most = (V + BEAM_WARPS * 256 - 1) / (BEAM_WARPS * 256);
  int parts = (4 * sm_count_current() + rows - 1) / rows;
  if (parts > BEAM_PARTS) parts = BEAM_PARTS;
  return parts < most ? parts : most;
}

}  // namespace axb

using namespace axb;

// 32-bit words of the workspace: two per row and part, then two per entry of their lists
extern "C" long long axb_beam_select_words(int B, int K, int V) {
  return 2ll * B * K * beam_parts(B * K, V) * (1 + K);
}

extern "C" int axb_beam_select(const void* logits, const float* scores, const void* done, int eos, float* out_scores, long long* out_tokens,
                               int* out_parents, void* out_done, void* work, int B, int K, int V, int dtype, void* stream) {
  if (B <= 0 || K <= 0 || V <= 0 || K > BEAM_MOST || static_cast<long long>(B) * K > 0x7fffffffll) {
    set_error("beam_select: 1 to %d beams, not %d", BEAM_MOST, K);
    return -1;
  }
  if (V > 1 << 30) { set_error("beam_select: a vocabulary of at most %d", 1 << 30); return -1; }
  if (dtype < 0 || dtype > 2) { set_error("beam_select: bf16, fp16 or fp32 logits"); return -1; }
  if (reinterpret_cast<uintptr_t>(work) & 7) { set_error("beam_select: the workspace must be 8-byte aligned"); return -1; }
  const int rows = B * K, parts = beam_parts(rows, V), size = dtype == 2 ? 4 : 2;
  const long long steps = (V + 256ll * BEAM_WARPS - 1) / (256ll * BEAM_WARPS);
  BeamArgs a{logits, scores, (const unsigned char*)done, out_scores, out_tokens, out_parents, (unsigned char*)out_done};
  const size_t lists = static_cast<size_t>(rows) * parts;
  a.sums = (float2*)work;
  a.keys = (uint32_t*)work + 2 * lists;
  a.tokens = (int*)a.keys + lists * K;
  a.B = B; a.K = K; a.V = V; a.eos = eos; a.parts = parts;
  a.part_steps = static_cast<int>((steps + parts - 1) / parts);
  const bool vec = (reinterpret_cast<uintptr_t>(logits) & 15) == 0 && static_cast<long long>(V) * size % 16 == 0;
  void (*kern)(BeamArgs) = dtype == 0 ? (vec ? beam_rows_kernel<__nv_bfloat16, true> : beam_rows_kernel<__nv_bfloat16, false>)
                           : dtype == 1 ? (vec ? beam_rows_kernel<__half, true> : beam_rows_kernel<__half, false>)
                                        : (vec ? beam_rows_kernel<float, true> : beam_rows_kernel<float, false>);
  AXB_CUDA(pdl_launch(kern, dim3(rows, parts), dim3(32 * BEAM_WARPS), 0, (cudaStream_t)stream, a));
  AXB_CUDA(pdl_launch(beam_select_kernel, dim3(B), dim3(32 * BEAM_WARPS), 0, (cudaStream_t)stream, a));
  return 0;
}
