// Rows of a table by token, scaled, and the gradient of the table: the sums of the rows of equal tokens.
//
//   out_i = scale table[t_i];   dtable_v = scale sum_{i: t_i = v} dy_i   (nothing of the padding token)
// A token outside the table gives a row of NaN and has no gradient.  Sums are 32-bit, in an order that the tokens alone decide, and
// rounded once; numbers below 2^-126 are kept.
//
// Both are bound by the rows' bytes.  The gradient sorts (token, place) pairs and sums along the sorted list, so that every row of the
// gradient is written once, by one block, and no addition depends on when a block runs:
//   1. One cluster sorts by a stable radix sort; its CTAs exchange counts, and up to 32,768 pairs, through distributed shared memory.  It
//      also notes which tokens there are.
//   2. Blocks sum chunks of 32 pairs, columns split over blocks; other blocks of the same launch zero the rows of the tokens that
//      there are not.  A chunk is summed with what the last token of it has in the next one, unless that token fills the whole next
//      chunk: then its sum so far goes to the workspace.  A segment of any length so takes many blocks, and one of up to 32 pairs
//      no extra traffic.
//   3. The partial sums of long segments, which the blocks of the sums have noted, are joined: every eighth by one warp, then the warps'.
// Up to 256 tokens are looked through by every block instead: one launch, for steps that are bound by the host's launches.
//
// One B200, device time: 16,384 tokens, 50,304 x 2,048 bf16, lookup and gradient 83 us, of which the lookup 20 to 22 (a copy of its 67 MB
// 22), the sums 40 (273 MB: 6.8 TB/s), the join 5 to 8; 128,256 x 4,096 225 us (1.38 GB: 210 at the copy's rate).  The sort takes 9 to 13
// us beside the lookup.  Rows of 1001 fp32 values (4-byte pieces), 6,001 tokens of which 40 % are padding, 32,000 rows: 52 us (28).
#include <atomic>
#include <initializer_list>

#include "common.cuh"

namespace axb {

constexpr int SORT_THREADS = 512, SORT_WARPS = SORT_THREADS / 32, SORT_DIGIT = 9, SORT_BINS = 1 << SORT_DIGIT;
constexpr int SORT_CTAS = 16, SORT_PORTABLE = 8, SORT_KEEP = 4;      // KEEP: pairs of a thread that stay in registers
constexpr int SORT_SHARE = SORT_THREADS * SORT_KEEP;
constexpr int SORT_ALONE = 2 * SORT_THREADS;      // tokens that one CTA sorts
constexpr int SORT_SMEM = SORT_WARPS * SORT_BINS * 4, SORT_SMEM_SMALL = SORT_SMEM + 2 * SORT_SHARE * 8;
constexpr int CHUNK = 32;                     // pairs of a block of sums: a warp's lanes look one chunk ahead
// rows that are loaded before the first is added: 4 and 16 take 1 % more (16,384 tokens, 50,304 x 2,048)
constexpr int SUM_THREADS = 128, SUM_AHEAD = 8;
constexpr int ZERO_BYTES = 1 << 17;           // of the table, of a block that zeroes
// A launch less for the sort and one for the join, 3 us of host time each; 256 equal tokens are summed by one block per 2 KB of columns.
constexpr int FEW = 256, FEW_ZERO = 4096;     // tokens that are not sorted; rows of a block that zeroes, then
constexpr int JOIN_THREADS = 256, JOIN_COLS = 128, JOIN_BLOCKS = 64;
// Rows at a time and blocks per SM of a lookup: 4 rows and 6 blocks 26.7 us, 8 rows and 4 blocks 34.7, these 24.2 (16,384 rows of 4 KB).
constexpr int ROW_THREADS = 256, ROW_AHEAD = 2, ROW_BLOCKS = 8;

template <typename T> __device__ __forceinline__ float to_float(T x) {
  if constexpr (__is_same(T, float)) return x;
  else if constexpr (__is_same(T, __half)) return __half2float(x);
  else return __bfloat162float(x);
}
template <typename T> __device__ __forceinline__ T from_float(float x) {
  if constexpr (__is_same(T, float)) return x;
  else if constexpr (__is_same(T, __half)) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}
// Sums and products that keep numbers below 2^-126, which the build's fast mathematics flushes to zero.
__device__ __forceinline__ float plus(float a, float b) {
  float c;
  asm("add.rn.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}
__device__ __forceinline__ float times(float a, float b) {
  float c;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}

// N values that are moved at once
template <typename T, int N> struct alignas(sizeof(T) * N) Piece { T v[N]; };

// ------------------------------------------------------------------------------------------------------------------------ lookup
// `group` threads (a power of two) a row, ROWS rows for each of them at a time, 16 bytes of each in pieces of N values.  Tokens are read a
// step ahead.  `beside` the sorting of the same tokens, which lets this kernel begin when all work before both has ended, it waits for
// that at its end only.
template <typename T, typename I, int N, int ROWS>
__global__ void __launch_bounds__(ROW_THREADS, ROW_BLOCKS)
embedding_kernel(const I* __restrict__ tokens, long long n, const T* __restrict__ table, long long pitch, int V, int H, float scale,
                 T* __restrict__ out, int group, bool beside) {
  using P = Piece<T, N>;
  constexpr int PIECES = 16 / sizeof(P);
  pdl_launch_next();
  if (!beside) pdl_wait();
  const int groups = ROW_THREADS / group, at = threadIdx.x & (group - 1);
  long long first = (static_cast<long long>(blockIdx.x) * groups + threadIdx.x / group) * ROWS;
  const long long step = static_cast<long long>(gridDim.x) * groups * ROWS;
  const bool as_is = scale == 1.f;
  I next[ROWS];
  const auto fetch = [&](long long i) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) next[r] = i + r < n ? tokens[i + r] : I(-1);
  };
  fetch(first);
  for (; first < n; first += step) {
    const T* from[ROWS];
    bool there[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      there[r] = next[r] >= 0 && next[r] < V;
      from[r] = table + (there[r] ? static_cast<long long>(next[r]) * pitch : 0ll);
    }
    fetch(first + step);
    T* to = out + first * H;
    const int rows = static_cast<int>(min(static_cast<long long>(ROWS), n - first));
    for (int c0 = at * N; c0 < H; c0 += group * N * PIECES) {
      P p[ROWS][PIECES];
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int k = 0; k < PIECES; ++k)
          if (c0 + k * group * N < H) p[r][k] = *reinterpret_cast<const P*>(from[r] + c0 + k * group * N);
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        if (r >= rows) break;
        if (!as_is || !there[r]) {
          const float by = there[r] ? scale : __int_as_float(0x7fffffff);
#pragma unroll
          for (int k = 0; k < PIECES; ++k)
#pragma unroll
            for (int i = 0; i < N; ++i) p[r][k].v[i] = from_float<T>(times(to_float(p[r][k].v[i]), by));
        }
#pragma unroll
        for (int k = 0; k < PIECES; ++k)
          if (c0 + k * group * N < H) *reinterpret_cast<P*>(to + static_cast<long long>(r) * H + c0 + k * group * N) = p[r][k];
      }
    }
  }
  if (beside) pdl_wait();                        // this kernel's end stands for the sorting kernel's too
}

// ------------------------------------------------------------------------------------------------------------------------ gradient
struct Digits { int passes, bits[4]; };

__device__ __forceinline__ uint32_t cluster_ctas() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t read_of_cta(const uint32_t* p, uint32_t cta) {
  uint32_t addr, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(p)), "r"(cta));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// Lanes of the warp with the same digit, of those that are there.  (__match_any_sync takes as many steps as there are digits.)
__device__ __forceinline__ uint32_t same_digit(uint32_t d, bool there) {
  uint32_t same = __ballot_sync(0xffffffffu, there);
#pragma unroll
  for (int b = 0; b < SORT_DIGIT; ++b) {
    const uint32_t set = __ballot_sync(0xffffffffu, d >> b & 1u);
    same &= d >> b & 1u ? set : ~set;
  }
  return same;
}

__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ void give_to_cta(uint2* p, uint32_t cta, uint2 v) {
  uint32_t addr;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(p)), "r"(cta));
  asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(addr), "r"(v.x), "r"(v.y) : "memory");
}

// One cluster.  Tokens without a gradient have the key V.  A warp has a contiguous run of pairs and counts of its own, so that equal
// digits keep their order.  SMALL: a warp's pairs stay in registers, and the CTAs hand them to one another through shared memory, of which
// each has two parts of the whole list.  Otherwise they go through `a` and `b` in turns.  The result is in `a` if SMALL or after an even
// number of passes, and in `b` after an odd one.
template <typename I, bool SMALL>
__global__ void __launch_bounds__(SORT_THREADS)
sort_tokens_kernel(const I* __restrict__ tokens, int n, int V, long long padding, Digits digits, uint2* a, uint2* b, uint8_t* met) {
  extern __shared__ uint4 s_memory[];
  uint32_t* const s_count = reinterpret_cast<uint32_t*>(s_memory);         // [SORT_WARPS][SORT_BINS]
  uint2* const s_pairs = reinterpret_cast<uint2*>(s_count + SORT_WARPS * SORT_BINS);
  __shared__ uint32_t s_total[SORT_BINS], s_base[SORT_BINS], s_warp[SORT_BINS / 32];
  pdl_wait();
  pdl_launch_next();                             // the lookup beside this reads what was there before
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const uint32_t cta = cluster_cta_rank(), ctas = cluster_ctas(), lower = (1u << lane) - 1u;
  // n is below 2^31, and what is added to it below 2^14: unsigned numbers do
  const uint32_t end = n, warps = ctas * SORT_WARPS, run = ((end + warps - 1u) / warps + 31u) / 32u * 32u;
  const uint32_t from = (cta * SORT_WARPS + w) * run, to = min(from + run, end), share = run * SORT_WARPS;      // share: of a CTA
  uint32_t* mine = s_count + w * SORT_BINS;
  const auto key_of = [&](uint32_t i) {
    const long long t = tokens[i];
    return make_uint2(t >= 0 && t < V && t != padding ? static_cast<uint32_t>(t) : static_cast<uint32_t>(V), i);
  };
  uint2 kept[SORT_KEEP];
#pragma unroll
  for (int k = 0; k < SORT_KEEP; ++k) kept[k] = from + 32 * k + lane < to ? key_of(from + 32 * k + lane) : make_uint2(0u, 0u);
  for (uint32_t i = cta * SORT_THREADS + tid; i < (V + 15u) / 16u; i += ctas * SORT_THREADS) reinterpret_cast<uint4*>(met)[i] = make_uint4(0u, 0u, 0u, 0u);
  const uint2* in = nullptr;
  uint2* out = b;
  int shift = 0;
  for (int pass = 0; pass < digits.passes; ++pass) {
    const int bits = digits.bits[pass], bins = 1 << bits;
    const uint32_t mask = bins - 1u;
    const bool last = pass + 1 == digits.passes;
    uint32_t kept_same[SORT_KEEP];
    const auto pair_at = [&](uint32_t i) {
      if (i >= to) return make_uint2(0u, 0u);
      return in ? __ldcg(in + i) : key_of(i);
    };
    const auto count = [&](uint2 p, bool there) {
      const uint32_t d = p.x >> shift & mask, same = same_digit(d, there);
      if (there && (same & lower) == 0u) mine[d] += __popc(same);
      __syncwarp();
      return same;
    };
    const auto place = [&](uint2 p, uint32_t same, bool there) {
      const uint32_t d = p.x >> shift & mask;
      uint32_t at = 0u;
      if (there) at = s_base[d] + mine[d] + __popc(same & lower);
      __syncwarp();
      if (there) {
        if ((same & lower) == 0u) mine[d] += __popc(same);
        if (last && p.x < static_cast<uint32_t>(V)) met[p.x] = 1;          // of equal tokens, all write the same
        if (!SMALL) out[at] = p;
        else if (last) a[at] = p;
        else {
          uint32_t to_cta = 0u;
#pragma unroll
          for (uint32_t k = 1; k < SORT_CTAS; ++k) to_cta += at >= k * share;
          give_to_cta(s_pairs + (pass & 1) * SORT_SHARE + at - to_cta * share, to_cta, p);
        }
      }
      __syncwarp();
    };
    for (int i = lane; i < bins; i += 32) mine[i] = 0u;
    __syncwarp();
    if (!SMALL && pass > 0) {
#pragma unroll
      for (int k = 0; k < SORT_KEEP; ++k) kept[k] = pair_at(from + 32 * k + lane);
    }
#pragma unroll
    for (int k = 0; k < SORT_KEEP; ++k)
      if (from + 32 * k < to) kept_same[k] = count(kept[k], from + 32 * k + lane < to);
    if (!SMALL)
      for (uint32_t i = from + 32 * SORT_KEEP; i < to; i += 32) count(pair_at(i + lane), i + lane < to);
    __syncthreads();
    // counts of the warps before, then those of the CTAs before and of the smaller digits
    if (tid < bins) {
      uint32_t of[SORT_WARPS], sum = 0u;
#pragma unroll
      for (int k = 0; k < SORT_WARPS; ++k) of[k] = s_count[k * SORT_BINS + tid];
#pragma unroll
      for (int k = 0; k < SORT_WARPS; ++k) {
        s_count[k * SORT_BINS + tid] = sum;
        sum += of[k];
      }
      s_total[tid] = sum;
    }
    __syncwarp();
    cluster_sync_all();                          // also: `met` is zero
    uint32_t before = 0u, all = 0u, upto = 0u;
    if (tid < SORT_BINS) {
      if (tid < bins) {
#pragma unroll
        for (uint32_t k = 0; k < SORT_CTAS; ++k) {
          const uint32_t c = k < ctas ? read_of_cta(s_total + tid, k) : 0u;
          if (k < cta) before += c;
          all += c;
        }
      }
      upto = all;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      if (lane == 31) s_warp[w] = upto;
    }
    __syncthreads();
    if (tid < bins) {
#pragma unroll
      for (int k = 0; k < SORT_BINS / 32; ++k) if (k < w) upto += s_warp[k];
      s_base[tid] = upto - all + before;
    }
    __syncthreads();
    if (last) cluster_arrive_relaxed();          // this CTA has read the others' totals; nobody reads what it stores from here on
#pragma unroll
    for (int k = 0; k < SORT_KEEP; ++k)
      if (from + 32 * k < to) place(kept[k], kept_same[k], from + 32 * k + lane < to);
    if (!SMALL)
      for (uint32_t i = from + 32 * SORT_KEEP; i < to; i += 32) {
        const uint2 p = pair_at(i + lane);
        const bool there = i + lane < to;
        place(p, same_digit(p.x >> shift & mask, there), there);
      }
    __syncwarp();
    if (last) {
      cluster_wait();                            // no CTA ends before its totals have been read
      return;
    }
    cluster_sync_all();                          // the pairs are there, and the totals have been read
    if (SMALL) {
#pragma unroll
      for (int k = 0; k < SORT_KEEP; ++k)
        if (from + 32 * k + lane < to) kept[k] = s_pairs[(pass & 1) * SORT_SHARE + w * run + 32 * k + lane];
    }
    in = out;
    out = out == b ? a : b;
    shift += bits;
  }
}

// Rows [v0, v1) but those that are `met`, a warp a row: the values in front of the first 16-byte boundary, whole words, the values
// behind the last.
template <typename T, int N, typename Met> __device__ __forceinline__ void zero_rows_of(T* dtable, int v0, int v1, int H, Met met) {
  constexpr int COUNT = 16 / sizeof(T);
  const int lane = threadIdx.x & 31;
  for (int v = v0 + threadIdx.x / 32; v < v1; v += SUM_THREADS / 32) {
    if (met(v)) continue;
    T* row = dtable + static_cast<long long>(v) * H;
    const int head = N == COUNT ? 0 : min(static_cast<int>((16u - (reinterpret_cast<unsigned long long>(row) & 15u)) % 16u / sizeof(T)), H);
    const int words = (H - head) / COUNT;
    uint4* to = reinterpret_cast<uint4*>(row + head);
    for (int i = lane; i < words; i += 32) to[i] = make_uint4(0u, 0u, 0u, 0u);
    if (N < COUNT) {
      if (lane < head) row[lane] = from_float<T>(0.f);
      if (head + words * COUNT + lane < H) row[head + words * COUNT + lane] = from_float<T>(0.f);
    }
  }
}

// Few tokens: a block and 16 bytes of columns per thread for each of them, which sums the rows of its token if it is the first with it;
// the other blocks zero the rows of the tokens that there are not.
template <typename T, typename I, int N>
__global__ void __launch_bounds__(SUM_THREADS)
sum_few_rows_kernel(const I* __restrict__ tokens, int n, const T* __restrict__ dy, long long pitch, int V, int H, float scale, long long padding,
                    T* __restrict__ dtable, int slices, int zero_rows) {
  using P = Piece<T, N>;
  constexpr int PIECES = 16 / sizeof(P), STEP = SUM_THREADS * N;
  __shared__ int s_token[FEW];                   // -1: without a gradient
  __shared__ uint32_t s_met[FEW_ZERO / 32];
  __shared__ int s_at[FEW], s_count[SUM_THREADS / 32];
  pdl_launch_next();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  for (int i = tid; i < n; i += SUM_THREADS) {
    const long long t = tokens[i];
    s_token[i] = t >= 0 && t < V && t != padding ? static_cast<int>(t) : -1;
  }
  const int sums = n * slices;
  if (static_cast<int>(blockIdx.x) >= sums) {
    const int v0 = (static_cast<int>(blockIdx.x) - sums) * zero_rows, v1 = min(v0 + zero_rows, V);
    for (int i = tid; i < (zero_rows + 31) / 32; i += SUM_THREADS) s_met[i] = 0u;
    __syncthreads();
    for (int i = tid; i < n; i += SUM_THREADS)
      if (s_token[i] >= v0 && s_token[i] < v1) atomicOr(&s_met[(s_token[i] - v0) / 32], 1u << (s_token[i] - v0) % 32);
    __syncthreads();
    zero_rows_of<T, N>(dtable, v0, v1, H, [&](int v) { return (s_met[(v - v0) / 32] >> (v - v0) % 32 & 1u) != 0u; });
    return;
  }
  __syncthreads();
  const int own = static_cast<int>(blockIdx.x) / slices, slice = static_cast<int>(blockIdx.x) - own * slices, token = s_token[own];
  if (token < 0) return;
  // the places of the token, in their order; none in front of this one
  int count = 0;
  for (int i0 = 0; i0 < n; i0 += SUM_THREADS) {
    const bool mine = i0 + tid < n && s_token[i0 + tid] == token;
    if (__syncthreads_or(mine && i0 + tid < own)) return;
    const unsigned met = __ballot_sync(0xffffffffu, mine);
    if (lane == 0) s_count[w] = __popc(met);
    __syncthreads();
    int before = count;
    for (int k = 0; k < SUM_THREADS / 32; ++k) { if (k < w) before += s_count[k]; count += s_count[k]; }
    if (mine) s_at[before + __popc(met & ((1u << lane) - 1u))] = i0 + tid;
    __syncthreads();
  }
  const int col = slice * STEP * PIECES + tid * N;
  if (col >= H) return;
  float sum[PIECES][N] = {};
  for (int i = 0; i < count; i += SUM_AHEAD) {
    P p[SUM_AHEAD][PIECES];
#pragma unroll
    for (int k = 0; k < SUM_AHEAD; ++k) {
      const T* row = dy + s_at[min(i + k, count - 1)] * pitch + col;
#pragma unroll
      for (int c = 0; c < PIECES; ++c) if (col + c * STEP < H) p[k][c] = *reinterpret_cast<const P*>(row + c * STEP);
    }
#pragma unroll
    for (int k = 0; k < SUM_AHEAD; ++k) {
      if (i + k >= count) break;
#pragma unroll
      for (int c = 0; c < PIECES; ++c)
#pragma unroll
        for (int j = 0; j < N; ++j) sum[c][j] = plus(sum[c][j], to_float(p[k][c].v[j]));
    }
  }
#pragma unroll
  for (int c = 0; c < PIECES; ++c) {
    P p;
#pragma unroll
    for (int j = 0; j < N; ++j) p.v[j] = from_float<T>(times(sum[c][j], scale));
    if (col + c * STEP < H) *reinterpret_cast<P*>(dtable + static_cast<long long>(token) * H + col + c * STEP) = p;
  }
}

// Sums of a chunk, 16 bytes of columns per thread in pieces of N values; behind the blocks of the sums those that zero rows.
template <typename T, int N>
__global__ void __launch_bounds__(SUM_THREADS)
sum_rows_kernel(const uint2* __restrict__ pairs, int n, const T* __restrict__ dy, long long pitch, int V, int H, int Hp, float scale,
                const uint8_t* __restrict__ met, T* __restrict__ dtable, float* __restrict__ partial, int* __restrict__ pieces, int slices,
                long long sum_blocks, int zero_rows) {
  using P = Piece<T, N>;
  constexpr int PIECES = 16 / sizeof(P), STEP = SUM_THREADS * N;
  __shared__ uint2 s_pair[2 * CHUNK + 1];
  pdl_launch_next();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31;
  if (blockIdx.x >= sum_blocks) {
    const int v0 = static_cast<int>(blockIdx.x - sum_blocks) * zero_rows, v1 = min(v0 + zero_rows, V);
    zero_rows_of<T, N>(dtable, v0, v1, H, [&](int v) { return __ldg(met + v) != 0; });
    return;
  }
  const int chunk = static_cast<int>(blockIdx.x / slices), slice = static_cast<int>(blockIdx.x - static_cast<long long>(chunk) * slices);
  const long long base = static_cast<long long>(chunk) * CHUNK;
  if (tid <= 2 * CHUNK) {
    const long long i = base - 1 + tid;
    s_pair[tid] = i >= 0 && i < n ? pairs[i] : make_uint2(0xffffffffu, 0u);
  }
  __syncthreads();
  const auto key = [&](int i) { return s_pair[1 + i].x; };          // of the pair `i` behind the chunk's first
  const int here = static_cast<int>(min(static_cast<long long>(CHUNK), n - base));
  const uint32_t first = key(0), last = key(here - 1);
  const bool goes_on = key(-1) == first, all_one = here == CHUNK && first == last;
  int from = 0, to = here;
  bool open = false;                             // the last segment has pieces in other blocks
  const unsigned ahead = __ballot_sync(0xffffffffu, key(CHUNK + lane) == last);      // of the next chunk, those of the last token
  if (here == CHUNK) {
    if (ahead == 0xffffffffu) open = true;
    else to += __ffs(~ahead) - 1;
  }
  if (goes_on) {
    if (all_one) open = true;
    else from = __ffs(~__ballot_sync(0xffffffffu, lane < here && key(lane) == first)) - 1;
  }
  // tokens without a gradient are the last ones
  if (last >= static_cast<uint32_t>(V)) {
    to = min(to, from + __popc(__ballot_sync(0xffffffffu, from + lane < here && key(from + lane) < static_cast<uint32_t>(V))));
    open = false;
  }
  if (slice == 0) {
    // of a long segment that begins here: how many chunks it takes, this one and those that it fills
    int count = 0;
    if (open && !(goes_on && all_one)) {
      count = 1;
      for (int more = SUM_THREADS; more == SUM_THREADS; count += more) {
        const long long end = base + static_cast<long long>(count + tid + 1) * CHUNK;
        more = __syncthreads_count(end <= n && pairs[end - 1].x == last);
      }
    }
    if (tid == 0) pieces[chunk] = count;
  }
  if (from >= to) return;
  const int col = slice * STEP * PIECES + tid * N;
  if (col >= H) return;
  float sum[PIECES][N] = {};
  uint32_t now = key(from);
  const auto store = [&] {
#pragma unroll
    for (int c = 0; c < PIECES; ++c) {
      P p;
#pragma unroll
      for (int i = 0; i < N; ++i) { p.v[i] = from_float<T>(times(sum[c][i], scale)); sum[c][i] = 0.f; }
      if (col + c * STEP < H) *reinterpret_cast<P*>(dtable + static_cast<long long>(now) * H + col + c * STEP) = p;
    }
  };
  for (int i = from; i < to; i += SUM_AHEAD) {
    P p[SUM_AHEAD][PIECES];
#pragma unroll
    for (int k = 0; k < SUM_AHEAD; ++k) {
      const T* row = dy + s_pair[1 + min(i + k, to - 1)].y * pitch + col;
#pragma unroll
      for (int c = 0; c < PIECES; ++c) if (col + c * STEP < H) p[k][c] = *reinterpret_cast<const P*>(row + c * STEP);
    }
#pragma unroll
    for (int k = 0; k < SUM_AHEAD; ++k) {
      if (i + k >= to) break;
      if (key(i + k) != now) { store(); now = key(i + k); }
#pragma unroll
      for (int c = 0; c < PIECES; ++c)
#pragma unroll
        for (int j = 0; j < N; ++j) sum[c][j] = plus(sum[c][j], to_float(p[k][c].v[j]));
    }
  }
  if (!open || now != last) { store(); return; }
  float* to_part = partial + static_cast<long long>(chunk) * Hp + col;
#pragma unroll
  for (int c = 0; c < PIECES; ++c)
#pragma unroll
    for (int j = 0; j < N; ++j) if (col + c * STEP < H) to_part[c * STEP + j] = sum[c][j];
}

// The pieces of long segments: every eighth one by the same warp, then the warps' sums.  blockIdx.x: columns (there may be more than the 65,535
// that the grid's other dimensions have), blockIdx.y: segments.
template <typename T>
__global__ void __launch_bounds__(JOIN_THREADS)
join_rows_kernel(const uint2* __restrict__ pairs, const int* __restrict__ pieces, int chunks, int H, int Hp, float scale,
                 const float* __restrict__ partial, T* __restrict__ dtable) {
  __shared__ int2 s_begin[JOIN_THREADS];         // chunk, pieces
  __shared__ int s_warp[JOIN_THREADS / 32];
  __shared__ float4 s_sum[JOIN_THREADS / 32][32];
  pdl_launch_next();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, col = blockIdx.x * JOIN_COLS + lane * 4;
  unsigned seen = 0;
  for (int c0 = 0; c0 < chunks; c0 += JOIN_THREADS) {
    const int own = c0 + tid < chunks ? pieces[c0 + tid] : 0;
    const unsigned flags = __ballot_sync(0xffffffffu, own > 0);
    if (lane == 0) s_warp[w] = __popc(flags);
    __syncthreads();
    int before = 0, count = 0;
#pragma unroll
    for (int i = 0; i < JOIN_THREADS / 32; ++i) { if (i < w) before += s_warp[i]; count += s_warp[i]; }
    if (own > 0) s_begin[before + __popc(flags & ((1u << lane) - 1u))] = make_int2(c0 + tid, own);
    __syncthreads();
    // every gridDim.y-th of all
    for (int i = static_cast<int>((blockIdx.y + gridDim.y - seen % gridDim.y) % gridDim.y); i < count; i += gridDim.y) {
      const int2 begin = s_begin[i];
      const uint32_t token = pairs[static_cast<long long>(begin.x) * CHUNK + CHUNK - 1].x;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      if (col < Hp) {
        const float* from = partial + static_cast<long long>(begin.x) * Hp + col;
#pragma unroll 8
        for (int r = w; r < begin.y; r += JOIN_THREADS / 32) {
          const float4 p = *reinterpret_cast<const float4*>(from + static_cast<long long>(r) * Hp);
          sum.x = plus(sum.x, p.x); sum.y = plus(sum.y, p.y); sum.z = plus(sum.z, p.z); sum.w = plus(sum.w, p.w);
        }
      }
      s_sum[w][lane] = sum;
      __syncthreads();
      if (w == 0) {
#pragma unroll
        for (int g = 1; g < JOIN_THREADS / 32; ++g) {
          const float4 p = s_sum[g][lane];
          sum.x = plus(sum.x, p.x); sum.y = plus(sum.y, p.y); sum.z = plus(sum.z, p.z); sum.w = plus(sum.w, p.w);
        }
        const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
        for (int g = 0; g < 4; ++g) if (col + g < H) dtable[static_cast<long long>(token) * H + col + g] = from_float<T>(times(v[g], scale));
      }
      __syncthreads();
    }
    seen += count;
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------------------------------ launches
// Bytes that are moved at once: what divides every address and pitch, 16 at most.
static int piece_bytes(int value, std::initializer_list<unsigned long long> of) {
  unsigned long long all = 16;
  for (unsigned long long x : of) all |= x;
  const int bytes = static_cast<int>(all & (~all + 1));
  return bytes < value ? value : bytes;
}
static unsigned long long address(const void* p) { return reinterpret_cast<unsigned long long>(p); }

template <typename T, typename I, int N>
static int look_up(const void* tokens, long long n, const void* table, long long pitch, int V, int H, float scale, void* out, bool beside,
                   cudaStream_t s) {
  constexpr int COUNT = 16 / sizeof(T);
  const int words = (H + COUNT - 1) / COUNT;
  int group = 32;
  while (group < ROW_THREADS && group < words) group *= 2;
  const int groups = ROW_THREADS / group;
  // several rows at a time where there are blocks enough for all SMs without
  const long long room = static_cast<long long>(ROW_BLOCKS) * sm_count_current();
  const bool ahead = n / groups >= room * ROW_AHEAD;
  const long long per = static_cast<long long>(groups) * (ahead ? ROW_AHEAD : 1), blocks = (n + per - 1) / per;
  AXB_CUDA(pdl_launch(ahead ? embedding_kernel<T, I, N, ROW_AHEAD> : embedding_kernel<T, I, N, 1>, dim3(static_cast<unsigned>(blocks < room ? blocks : room)),
                      dim3(ROW_THREADS), 0, s, static_cast<const I*>(tokens), n, static_cast<const T*>(table), pitch, V, H, scale,
                      static_cast<T*>(out), group, beside));
  return 0;
}

// What the gradient needs of more than a few tokens: a byte for every token of the table, and the sorted pairs (a second list for many: they take turns).
struct Sorted {
  long long met, pairs, words;
  Sorted(long long n, int V) {
    met = (V + 15ll) / 16 * 4;
    pairs = (2 * n + 3) / 4 * 4;
    words = n <= FEW ? 0 : met + (n > SORT_PORTABLE * SORT_SHARE ? 2 : 1) * pairs;
  }
};
static cudaLaunchConfig_t sort_config(unsigned ctas, int smem, cudaStream_t s, cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas); cfg.blockDim = dim3(SORT_THREADS); cfg.dynamicSmemBytes = smem; cfg.stream = s;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = max_ctas() == 0 ? 2 : 1;
  return cfg;
}
// CTAs of the cluster on the current device: 16 where it can run as many together (a part of a GPU may not), otherwise 8.  The kernels'
// attributes are set along with it, once per device: 3 us of host time otherwise.  0: an error.
static int sort_ctas() {
  static std::atomic<int> known[64];
  int device;
  if (check_cuda(cudaGetDevice(&device), "cudaGetDevice")) return 0;
  int ctas = known[device & 63].load(std::memory_order_acquire);
  if (ctas) return ctas;
  const auto set = [](auto kernel, int smem) {
    return check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "shared memory of the sorting kernel") ||
           check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), "cluster of the sorting kernel");
  };
  if (set(sort_tokens_kernel<long long, true>, SORT_SMEM_SMALL) || set(sort_tokens_kernel<int, true>, SORT_SMEM_SMALL) ||
      set(sort_tokens_kernel<long long, false>, SORT_SMEM) || set(sort_tokens_kernel<int, false>, SORT_SMEM)) return 0;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = sort_config(SORT_CTAS, SORT_SMEM_SMALL, nullptr, attr);
  cfg.numAttrs = 1;
  int clusters = 0;
  if (cudaOccupancyMaxActiveClusters(&clusters, sort_tokens_kernel<long long, true>, &cfg) != cudaSuccess) {
    cudaGetLastError();
    clusters = 0;
  }
  ctas = clusters > 0 ? SORT_CTAS : SORT_PORTABLE;
  known[device & 63].store(ctas, std::memory_order_release);
  return ctas;
}
// Bits of the passes; V itself is the key of tokens without a gradient.
static Digits digits_of(int V) {
  Digits d = {};
  int bits = 0;
  while (V >> bits) ++bits;
  d.passes = (bits + SORT_DIGIT - 1) / SORT_DIGIT;
  for (int i = 0, left = bits; i < d.passes; ++i) {
    d.bits[i] = (left + d.passes - i - 1) / (d.passes - i);
    left -= d.bits[i];
  }
  return d;
}
static const uint2* sorted_pairs(const void* sorted, long long n, int V, int ctas) {
  const Sorted at(n, V);
  const uint32_t* words = static_cast<const uint32_t*>(sorted);
  return reinterpret_cast<const uint2*>(words + at.met + (n > ctas * SORT_SHARE && digits_of(V).passes % 2 ? at.pairs : 0));
}

template <typename I>
static int sort_tokens(const void* tokens, int n, int V, long long padding, void* sorted, cudaStream_t s) {
  const int most = sort_ctas();
  if (!most) return -1;
  const Sorted at(n, V);
  uint32_t* words = static_cast<uint32_t*>(sorted);
  const bool small = n <= most * SORT_SHARE;
  uint2 *a = reinterpret_cast<uint2*>(words + at.met), *b = small ? nullptr : reinterpret_cast<uint2*>(words + at.met + at.pairs);
  const auto kernel = small ? sort_tokens_kernel<I, true> : sort_tokens_kernel<I, false>;
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = sort_config(n <= SORT_ALONE ? 1 : most, small ? SORT_SMEM_SMALL : SORT_SMEM, s, attr);
  AXB_CUDA(cudaLaunchKernelEx(&cfg, kernel, static_cast<const I*>(tokens), n, V, padding, digits_of(V), a, b, reinterpret_cast<uint8_t*>(words)));
  return 0;
}

// Partial sums of the chunks, and how many chunks the segments take that begin in them.
struct GradWork {
  long long chunks, Hp, pieces, words;
  GradWork(long long n, int H) {
    chunks = (n + CHUNK - 1) / CHUNK;
    Hp = (H + 3) / 4 * 4;
    pieces = (chunks + 3) / 4 * 4;
    words = n <= FEW ? 0 : pieces + chunks * Hp;
  }
};

static int rows_to_zero(int row_bytes) { return row_bytes >= ZERO_BYTES ? 1 : ZERO_BYTES / row_bytes; }

template <typename T, int N>
static int sum_few_rows(const void* tokens, int token_bytes, int n, const void* dy, long long pitch, int V, int H, float scale, long long padding,
                        void* dtable, cudaStream_t s) {
  const int columns = SUM_THREADS * 16 / static_cast<int>(sizeof(T)), slices = (H + columns - 1) / columns;
  const int most = rows_to_zero(H * static_cast<int>(sizeof(T))), zero_rows = most < FEW_ZERO ? most : FEW_ZERO;
  const dim3 grid(static_cast<unsigned>(n * slices + (V + zero_rows - 1) / zero_rows));
  if (token_bytes == 8)
    AXB_CUDA(pdl_launch(sum_few_rows_kernel<T, long long, N>, grid, dim3(SUM_THREADS), 0, s, static_cast<const long long*>(tokens), n,
                        static_cast<const T*>(dy), pitch, V, H, scale, padding, static_cast<T*>(dtable), slices, zero_rows));
  else
    AXB_CUDA(pdl_launch(sum_few_rows_kernel<T, int, N>, grid, dim3(SUM_THREADS), 0, s, static_cast<const int*>(tokens), n, static_cast<const T*>(dy),
                        pitch, V, H, scale, padding, static_cast<T*>(dtable), slices, zero_rows));
  return 0;
}

template <typename T, int N>
static int sum_rows(const void* sorted, int n, const void* dy, long long pitch, int V, int H, float scale, void* dtable, int* words, cudaStream_t s) {
  const GradWork work(n, H);
  const int columns = SUM_THREADS * 16 / static_cast<int>(sizeof(T)), slices = (H + columns - 1) / columns;
  const int zero_rows = rows_to_zero(H * static_cast<int>(sizeof(T)));
  const long long sum_blocks = work.chunks * slices, blocks = sum_blocks + (V + static_cast<long long>(zero_rows) - 1) / zero_rows;
  if (blocks > 0x7fffffffll) { set_error("gradient of an embedding: %d tokens with rows of %d values are too many blocks", n, H); return -1; }
  const int ctas = sort_ctas();
  if (!ctas) return -1;
  const uint2* pairs = sorted_pairs(sorted, n, V, ctas);
  float* partial = reinterpret_cast<float*>(words + work.pieces);
  AXB_CUDA(pdl_launch(sum_rows_kernel<T, N>, dim3(static_cast<unsigned>(blocks)), dim3(SUM_THREADS), 0, s, pairs, n, static_cast<const T*>(dy),
                      pitch, V, H, static_cast<int>(work.Hp), scale, static_cast<const uint8_t*>(sorted), static_cast<T*>(dtable), partial, words,
                      slices, sum_blocks, zero_rows));
  const int full = n / CHUNK;                    // a long segment fills one chunk and begins in another
  AXB_CUDA(pdl_launch(join_rows_kernel<T>, dim3(static_cast<unsigned>((work.Hp + JOIN_COLS - 1) / JOIN_COLS), full / 2 < JOIN_BLOCKS ? full / 2 : JOIN_BLOCKS),
                      dim3(JOIN_THREADS), 0, s, pairs, static_cast<const int*>(words), full, H, static_cast<int>(work.Hp), scale,
                      static_cast<const float*>(partial), static_cast<T*>(dtable)));
  return 0;
}

template <typename T>
static int gradient(const void* tokens, int token_bytes, const void* sorted, int n, const void* dy, long long pitch, int V, int H, float scale,
                    long long padding, void* dtable, int* work, cudaStream_t s) {
  if (n == 0) {
    AXB_CUDA(cudaMemsetAsync(dtable, 0, static_cast<size_t>(V) * H * sizeof(T), s));
    return 0;
  }
  const int size = sizeof(T), bytes = piece_bytes(size, {address(dy), address(dtable), static_cast<unsigned long long>(H) * size,
                                                         static_cast<unsigned long long>(pitch) * size});
  if (n <= FEW) {
    const auto sums = bytes == 16 ? sum_few_rows<T, 16 / sizeof(T)> : bytes == 8 ? sum_few_rows<T, 8 / sizeof(T)>
                    : bytes == 4 ? sum_few_rows<T, 4 / sizeof(T)> : sum_few_rows<T, 1>;
    return sums(tokens, token_bytes, n, dy, pitch, V, H, scale, padding, dtable, s);
  }
  const auto sums = bytes == 16 ? sum_rows<T, 16 / sizeof(T)> : bytes == 8 ? sum_rows<T, 8 / sizeof(T)> : bytes == 4 ? sum_rows<T, 4 / sizeof(T)>
                                                                                                                     : sum_rows<T, 1>;
  return sums(sorted, n, dy, pitch, V, H, scale, dtable, work, s);
}

template <typename T>
static int look_up_by(const void* tokens, int token_bytes, long long n, const void* table, long long pitch, int V, int H, float scale, void* out,
                      bool beside, cudaStream_t s) {
  const int size = sizeof(T), bytes = piece_bytes(size, {address(table), address(out), static_cast<unsigned long long>(H) * size,
                                                         static_cast<unsigned long long>(pitch) * size});
  const auto go = [&](auto index) {
    using I = decltype(index);
    const auto kernel = bytes == 16 ? look_up<T, I, 16 / sizeof(T)> : bytes == 8 ? look_up<T, I, 8 / sizeof(T)>
                      : bytes == 4 ? look_up<T, I, 4 / sizeof(T)> : look_up<T, I, 1>;
    return kernel(tokens, n, table, pitch, V, H, scale, out, beside, s);
  };
  return token_bytes == 8 ? go(0ll) : go(0);
}

}  // namespace axb

using namespace axb;

static int refused(const char* what, long long n, int V, int H, int dtype, int token_bytes) {
  if (n >= 0 && n <= 0x7fffffffll && V >= 1 && V <= (1 << 30) && H >= 1 && H <= (1 << 25) && dtype >= 0 && dtype <= 2 && (token_bytes == 4 || token_bytes == 8)) return 0;
  set_error("%s: %lld tokens of %d bytes, table %d x %d of type %d", what, n, token_bytes, V, H, dtype);
  return -1;
}
static int misaligned(const char* what, const void* p) {
  if (address(p) % 16 == 0) return 0;
  set_error("%s: the workspace must be 16-byte aligned", what);
  return -1;
}

extern "C" long long axb_embedding_sorted_words(long long n, int V) { return Sorted(n, V).words; }

extern "C" int axb_embedding(const void* tokens, int token_bytes, long long n, const void* table, long long pitch, int V, int H, float scale,
                             void* out, long long padding, void* sorted, int dtype, void* stream) {
  if (refused("embedding", n, V, H, dtype, token_bytes) || misaligned("embedding", sorted)) return -1;
  if (n == 0) return 0;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool sort = sorted && n > FEW;
  if (sort && (token_bytes == 8 ? sort_tokens<long long>(tokens, static_cast<int>(n), V, padding, sorted, s)
                                : sort_tokens<int>(tokens, static_cast<int>(n), V, padding, sorted, s))) return -1;
  const auto go = dtype == 0 ? look_up_by<__nv_bfloat16> : dtype == 1 ? look_up_by<__half> : look_up_by<float>;
  return go(tokens, token_bytes, n, table, pitch, V, H, scale, out, sort && max_ctas() == 0, s);
}

extern "C" long long axb_embedding_grad_words(long long n, int H) { return GradWork(n, H).words; }

extern "C" int axb_embedding_grad(const void* tokens, int token_bytes, const void* sorted, long long n, const void* dy, long long pitch, int V, int H,
                                  float scale, long long padding, void* dtable, void* work, int dtype, void* stream) {
  if (refused("gradient of an embedding", n, V, H, dtype, token_bytes) || misaligned("gradient of an embedding", work) ||
      misaligned("gradient of an embedding", sorted)) return -1;
  if (n > FEW && (!sorted || !work)) { set_error("gradient of an embedding: %lld tokens have been sorted, and take a workspace", n); return -1; }
  const auto go = dtype == 0 ? gradient<__nv_bfloat16> : dtype == 1 ? gradient<__half> : gradient<float>;
  return go(tokens, token_bytes, sorted, static_cast<int>(n), dy, pitch, V, H, scale, padding, dtable, static_cast<int*>(work),
            static_cast<cudaStream_t>(stream));
}
