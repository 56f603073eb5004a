// Selection of beam search: of all continuations of the beams of a prompt, value = score + logit - log sum exp(logits of the beam), the
// `beams` best, equal values in the order of (beam, token).
//
// Bound by reading the logits once.  A first launch cuts every beam's row into runs of chunks of 4 KB.  A warp copies the chunks of its run
// into shared memory, one ahead, and goes over each twice: no block ever waits for its warps, and the loops are short (the same code for
// values in registers is five times as long, and was waited for longer than the data).  The K-th largest of the lanes' maxima is reached
// by at least K values of the chunk and, with few beams, by few others; what reaches the largest such bound so far goes into a list, of
// which the K best are kept in the end.  The order within a beam is that of its logits, so that nothing has to be known of the sum.  A
// second launch puts the runs of a beam together and merges the beams.
//
// Where the list overflows, the K best are found one by one, and the run's chunks are read again for each: rows of mostly equal (masked)
// values, and ordinary ones with many beams or many chunks in a run, as a bound is that of one chunk's 32 lanes and nothing is taken out
// of the list.  Normal logits fill it with 32 values of four chunks for 8 beams, 89 for 16, 132 for 20, with 149 of 28 chunks for 8, and of
// a single chunk for 28 beams and more.  The second launch is a block per prompt, whose warps merge a beam's lists in K rounds for every
// 128 entries.  Both suit the beams of most searches, not 32: one prompt over 128,256 values takes 10.6, 34 and 370 us with 8, 16 and
// 32 beams, 64 prompts over 32,000 values with 16 beams 153, 256 with 8 beams 42.
//
// A run's sum is 32-bit: terms of exp2, which a lane adds one after another, within 2^-18 of the sum.  Runs are joined and values formed in
// 64 bits, as the order of two beams' tokens depends on differences of their sums' logarithms that 32-bit values of twenty or so round
// away; candidates of two beams that are closer than their sums are exact may still change places.
//
// 32 prompts, 8 beams (a fifth have ended), 128,256 bf16 values: 21.2 us, 3.1 TB/s of what is read.  Then the schedulers issue in half of
// the cycles and the unit of exp2 is busy for 0.45 of them: five warps per scheduler do not hide the dependent steps of a chunk.  One
// prompt, 4 beams, 32,000 values: 5.8 us for two launches.  Tried beside it, same case: chunks of 2 KB 24.6 us, neighbouring warps on
// different rows 23.3, blocks of one or two such warps 22.0, 22.6.
//
// A value that is not a number counts as -inf, and so do a score of +inf and every value of a beam whose sum is none.  Of a beam that has
// ended only the end token goes on, with the beam's score.
#include <type_traits>

#include "common.cuh"

namespace axb {

constexpr int BEAM_MOST = 32;            // beams
constexpr int BEAM_WARPS = 4;            // of a block of the first launch
constexpr int BEAM_LOADS = 8;            // 16-byte words of a lane, of a chunk
constexpr int BEAM_CHUNK = 32 * BEAM_LOADS * 16;     // bytes
constexpr int BEAM_LIST = 128;           // values of a run that reach the bounds, at most
constexpr int BEAM_AT_ONCE = 32;         // runs per SM: 24 warps fit, beams that have ended leave room; 24, 48, 64: 22.9, 22.5, 21.8 us for 21.2 (the 8 beams above)
constexpr int SELECT_THREADS = 256;
constexpr float BEAM_LOWEST = -3.4028234663852886e38f;
constexpr float BEAM_ORDINARY = 4096.f;  // references whose product with L is rounded by at most 2^-12
constexpr float LOG2E = 1.4426950408889634f;

struct BeamArgs {
  const void* logits;                    // [B, K, V]
  const float* scores;                   // [B, K]
  const unsigned char* done;             // [B, K] or null
  float* out_scores;
  long long* out_tokens;
  int* out_parents;
  unsigned char* out_done;
  // of every row and run: (reference, sum), then K keys and tokens, best first
  float2* sums;
  uint2* lists;
  int K, V, eos, parts, chunks;          // runs of a row, chunks of a run
  long long items;                       // runs of all rows
};

// 32-bit key with the order of the numbers; 0 is below all of them.  -0 counts as 0.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// The best of what the lanes hold (the larger key, then the lower token); key 0: none is left.  It is taken out.
template <int N> __device__ __forceinline__ uint2 take_best(uint32_t (&key)[N], int (&token)[N]) {
  uint32_t k = 0u;
#pragma unroll
  for (int i = 0; i < N; ++i) k = max(k, key[i]);
  k = __reduce_max_sync(0xffffffffu, k);
  int t = 0x7fffffff;
#pragma unroll
  for (int i = 0; i < N; ++i) if (key[i] == k) t = min(t, token[i]);
  t = __reduce_min_sync(0xffffffffu, t);
#pragma unroll
  for (int i = 0; i < N; ++i) if (token[i] == t) key[i] = 0u;
  return make_uint2(k, static_cast<uint32_t>(t));
}

// The `K` best of a list's `count` entries, at most 32 N, in their order.
template <int N> __device__ __forceinline__ void keep_best(const uint2* list, int count, uint2* out, int K) {
  const int lane = threadIdx.x & 31;
  uint32_t key[N];
  int token[N];
  uint2 mine = make_uint2(0u, 0u);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = i * 32 + lane;
    key[i] = 0u; token[i] = 0x7fffffff;
    if (e < count) { key[i] = list[e].x; token[i] = static_cast<int>(list[e].y); }
  }
  for (int e = 0; e < K; ++e) {
    const uint2 best = take_best(key, token);
    if (lane == e) mine = best;
  }
  if (lane < K) out[lane] = mine;
}

// 16 bytes of logits: words of two 16-bit values or one of 32 bits.
template <typename T> struct Values {
  static constexpr int COUNT = 16 / sizeof(T), PER_WORD = 4 / sizeof(T);
  uint32_t word[4];
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (__is_same(T, float)) return __uint_as_float(word[i]);
    else {
      const uint32_t w = word[i / 2];
      if constexpr (__is_same(T, __nv_bfloat16)) return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
      else return __half2float(__ushort_as_half(static_cast<unsigned short>(i & 1 ? w >> 16 : w & 0xffffu)));
    }
  }
  __device__ __forceinline__ uint32_t largest() const { return larger(larger(word[0], word[1]), larger(word[2], word[3])); }
  // the larger ones of two words' values; whether any of a word's values reaches `w`'s; a word of one value, the larger value of a word
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    if constexpr (__is_same(T, float)) return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    else if constexpr (__is_same(T, __nv_bfloat16)) {
      const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
      return *reinterpret_cast<const uint32_t*>(&m);
    } else {
      const __half2 m = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
      return *reinterpret_cast<const uint32_t*>(&m);
    }
  }
  static __device__ __forceinline__ uint32_t reaching(uint32_t a, uint32_t w) {
    if constexpr (__is_same(T, float)) return __uint_as_float(a) >= __uint_as_float(w) ? 0xffffffffu : 0u;
    else if constexpr (__is_same(T, __nv_bfloat16)) return __hge2_mask(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&w));
    else return __hge2_mask(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&w));
  }
  // bit j: value j reaches `w`'s
  __device__ __forceinline__ uint32_t hits(uint32_t w) const {
    if constexpr (PER_WORD == 1) {
      return (reaching(word[0], w) & 1u) | (reaching(word[1], w) & 2u) | (reaching(word[2], w) & 4u) | (reaching(word[3], w) & 8u);
    } else {
      const uint32_t b = (reaching(word[0], w) & 0x00020001u) | (reaching(word[1], w) & 0x00080004u) | (reaching(word[2], w) & 0x00200010u) |
                         (reaching(word[3], w) & 0x00800040u);
      return (b | b >> 16) & 0xffu;
    }
  }
  static __device__ __forceinline__ uint32_t word_of(float x) {      // x is one of the type's numbers
    if constexpr (__is_same(T, float)) return __float_as_uint(x);
    else if constexpr (__is_same(T, __nv_bfloat16)) return (__float_as_uint(x) >> 16) * 0x10001u;
    else return __half_as_ushort(__float2half_rn(x)) * 0x10001u;
  }
  static __device__ __forceinline__ float largest_of(uint32_t w) {
    const Values v = {{w, w, w, w}};
    if constexpr (__is_same(T, float)) return v[0];
    else return fmaxf(v[0], v[1]);
  }
};

// Two 32-bit numbers in a register pair.
__device__ __forceinline__ unsigned long long pair_of(float a, float b) {
  unsigned long long p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
  return p;
}
__device__ __forceinline__ void unpair(unsigned long long p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ unsigned long long fma_pair(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long d;
  asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ unsigned long long add_pair(unsigned long long a, unsigned long long b) {
  unsigned long long d;
  asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// What a sum of exponentials with the reference m has been divided by, as a power of two (L the rounded log2(e)).  An ordinary reference
// is taken off as rn(m L), which one instruction does with x L; where the rounding of m L is no longer small (chunks of masked values,
// logits of any size) exponents are (x - m) L.  The sums of both kinds go together through this number.
__device__ __forceinline__ double reference_log2(float m) {
  return fabsf(m) < BEAM_ORDINARY ? static_cast<double>(m * LOG2E) : static_cast<double>(m) * static_cast<double>(LOG2E);
}

// One chunk into shared memory, of which the row has V values from `from` on; VEC: every row starts on 16 bytes.  Whole words are
// copied, the last ones of a row and rows off 16 bytes value by value; what is not there is -inf.
template <typename T, bool VEC> __device__ __forceinline__ void copy_chunk(uint4* to, const T* from, int V) {
  constexpr int COUNT = 16 / sizeof(T), CHUNK = BEAM_CHUNK / sizeof(T);
  const int lane = threadIdx.x & 31, whole = VEC ? min(V, CHUNK) / COUNT : 0;
#pragma unroll
  for (int i = 0; i < BEAM_LOADS; ++i)
    if (i * 32 + lane < whole)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to + i * 32 + lane)), "l"(from + (i * 32 + lane) * COUNT) : "memory");
  using Bits = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;
  constexpr Bits lowest = static_cast<Bits>(__is_same(T, float) ? 0xff800000u : __is_same(T, __half) ? 0xfc00u : 0xff80u);
#pragma unroll 8
  for (int t = whole * COUNT + lane; t < CHUNK; t += 32) reinterpret_cast<Bits*>(to)[t] = t < V ? reinterpret_cast<const Bits*>(from)[t] : lowest;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * BEAM_WARPS) beam_rows_kernel(const BeamArgs a) {
  using X = Values<T>;
  constexpr int CHUNK = BEAM_CHUNK / sizeof(T);
  __shared__ uint4 s_chunk[BEAM_WARPS][2][BEAM_LOADS * 32];
  __shared__ uint2 s_list[BEAM_WARPS][BEAM_LIST];
  __shared__ unsigned s_count[BEAM_WARPS];
  pdl_launch_next();
  pdl_wait();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, K = a.K;
  const long long run = static_cast<long long>(blockIdx.x) * BEAM_WARPS + w;
  if (run >= a.items) return;
  // rows of several runs are 4 KB and more: their runs are counted in 32 bits
  const int row = static_cast<int>(a.parts == 1 ? run : static_cast<unsigned>(run) / a.parts), first = static_cast<int>(run - static_cast<long long>(row) * a.parts) * a.chunks;
  if (a.done && a.done[row]) return;
  const int last = min(first + a.chunks, (a.V + CHUNK - 1) / CHUNK);
  const T* values = static_cast<const T*>(a.logits) + static_cast<long long>(row) * a.V;
  auto copy = [&](int chunk, int buffer) {
    if (chunk < last) copy_chunk<T, VEC>(s_chunk[w][buffer], values + static_cast<long long>(chunk) * CHUNK, a.V - chunk * CHUNK);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (lane == 0) s_count[w] = 0u;
  copy(first, 0);
  float m = BEAM_LOWEST, sum = 0.f;          // the reference, raised only where a value exceeds it by far: few roundings of the sum
  uint32_t bound = 0u;
  for (int chunk = first, buffer = 0; chunk < last; ++chunk, buffer ^= 1) {
    __syncwarp();                            // the other buffer has been read
    copy(chunk + 1, buffer ^ 1);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
    const uint4* words = s_chunk[w][buffer] + lane;
    auto at = [&](int i) {
      const uint4 u = words[i * 32];
      return X{{u.x, u.y, u.z, u.w}};
    };
    uint32_t most_of[BEAM_LOADS], most;
#pragma unroll
    for (int i = 0; i < BEAM_LOADS; ++i) {
      most_of[i] = at(i).largest();
      most = i ? X::larger(most, most_of[i]) : most_of[i];
    }
    // the K-th largest of the lanes' maxima (equal ones count once: a lower bound does as well)
    uint32_t mine = order_key(X::largest_of(most));
    const uint32_t largest = __reduce_max_sync(0xffffffffu, mine);
    uint32_t kth = largest;
    for (int e = 1; e < K; ++e) {
      if (mine == kth) mine = 0u;
      kth = __reduce_max_sync(0xffffffffu, mine);
    }
    bound = max(bound, kth);
    const float top = fmaxf(key_value(largest), BEAM_LOWEST);
    if (top > m + 8.f || chunk == first) {
      sum *= exp2f(static_cast<float>(reference_log2(m) - reference_log2(top)));
      m = top;
    }
    const bool ordinary = fabsf(m) < BEAM_ORDINARY;
    const unsigned long long scale = pair_of(LOG2E, LOG2E), shift = pair_of(-m * LOG2E, -m * LOG2E);
    const uint32_t reach = X::word_of(bound ? key_value(bound) : -INFINITY);      // as numbers
    if (ordinary) {
      // exp(x - m) as exp2(x L - rn(m L)), two at a time
      unsigned long long sums[2] = {0ull, 0ull};
#pragma unroll 4
      for (int i = 0; i < BEAM_LOADS; ++i) {
        const X x = at(i);
#pragma unroll
        for (int j = 0; j < X::COUNT; j += 2) {
          float u, v;
          unpair(fma_pair(pair_of(x[j], x[j + 1]), scale, shift), u, v);
          sums[j / 2 & 1] = add_pair(sums[j / 2 & 1], pair_of(exp2f(u), exp2f(v)));
        }
      }
      float even, odd;
      unpair(add_pair(sums[0], sums[1]), even, odd);
      sum += even + odd;
    } else {
      for (int i = 0; i < BEAM_LOADS; ++i) {
        const X x = at(i);
#pragma unroll
        for (int j = 0; j < X::COUNT; ++j) sum += exp2f((x[j] - m) * LOG2E);
      }
    }
    // the words that hold values that reach the bound, then those values: few
    uint32_t some = 0u;
#pragma unroll
    for (int i = 0; i < BEAM_LOADS; ++i) some |= X::reaching(most_of[i], reach) ? 1u << i : 0u;
    while (some) {
      const int i = __ffs(some) - 1, base = chunk * CHUNK + (i * 32 + lane) * X::COUNT;
      some &= some - 1;
      for (uint32_t hits = at(i).hits(reach); hits; hits &= hits - 1) {
        const int j = __ffs(hits) - 1, t = base + j;
        const unsigned n = t < a.V ? atomicAdd(&s_count[w], 1u) : BEAM_LIST;
        if (n < BEAM_LIST) s_list[w][n] = make_uint2(order_key(static_cast<float>(reinterpret_cast<const T*>(words + i * 32)[j])), t);
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) a.sums[run] = make_float2(m, sum);
  __syncwarp();
  const int count = static_cast<int>(s_count[w]);
  uint2* out = a.lists + run * K;
  if (count <= 32) keep_best<1>(s_list[w], count, out, K);
  else if (count <= BEAM_LIST) keep_best<BEAM_LIST / 32>(s_list[w], count, out, K);
  else {
    // K times the best behind the one before
    uint2 before = make_uint2(0xffffffffu, 0u);
    for (int e = 0; e < K; ++e) {
      uint32_t key[1] = {0u};
      int token[1] = {0x7fffffff};
      for (int chunk = first; chunk < last; ++chunk) {
        if (last - first > 1) {
          __syncwarp();
          copy(chunk, 0);
          asm volatile("cp.async.wait_group 0;" ::: "memory");
          __syncwarp();
        }
        for (int i = 0; i < BEAM_LOADS; ++i) {
          const uint4 u = s_chunk[w][0][i * 32 + lane];
          const X x = {{u.x, u.y, u.z, u.w}};
#pragma unroll
          for (int j = 0; j < X::COUNT; ++j) {
            const uint32_t k = order_key(x[j]);
            const int t = chunk * CHUNK + (i * 32 + lane) * X::COUNT + j;
            const bool behind = e == 0 || k < before.x || (k == before.x && t > static_cast<int>(before.y));
            if (t < a.V && behind && k > key[0]) { key[0] = k; token[0] = t; }      // t grows: the lowest of equal ones stays
          }
        }
      }
      before = take_best(key, token);
      if (lane == 0) out[e] = before;
    }
  }
}

// 64-bit key with the order of the numbers, 0 below all of them.
__device__ __forceinline__ unsigned long long order_key(double x) {
  const unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(x));
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ double key_value(unsigned long long k) {
  return __longlong_as_double(static_cast<long long>(k >> 63 ? k & 0x7fffffffffffffffull : ~k));
}

// A run's sum for the reference `top` of its row.
__device__ __forceinline__ double run_sum(float2 s, float top) {
  return static_cast<double>(s.y) * exp2(reference_log2(s.x) - static_cast<double>(top) * static_cast<double>(LOG2E));
}

// One block per prompt.  A warp per beam: the beam's sum, its parts' lists; then the beams' lists, K rounds, a lane per beam.
__global__ void __launch_bounds__(SELECT_THREADS) beam_select_kernel(const BeamArgs a) {
  constexpr int AT_ONCE = 4;               // entries of a lane, beside one of the best so far
  __shared__ unsigned long long s_value[BEAM_MOST][BEAM_MOST];      // order keys, 0: none
  __shared__ int s_token[BEAM_MOST][BEAM_MOST];
  pdl_launch_next();
  pdl_wait();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, K = a.K, V = a.V, b = blockIdx.x;
  const double none = -__longlong_as_double(0x7ff0000000000000ll);
  const long long entries = static_cast<long long>(a.parts) * K;
  for (int row = w; row < K; row += SELECT_THREADS / 32) {
    const size_t at = static_cast<size_t>(b) * K + row;
    const bool done = a.done && a.done[at];
    const float given = a.scores[at];
    uint2 first[AT_ONCE];
    float2 s = make_float2(BEAM_LOWEST, 0.f);
    if (!done) {                         // what most calls need, on its way together
      if (lane < a.parts) s = a.sums[at * a.parts + lane];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i)
        first[i] = i * 32 + lane < entries ? a.lists[at * entries + i * 32 + lane] : make_uint2(0u, 0x7fffffffu);
    }
    const double score = given < -none ? given : none;      // no sum of logarithms of probabilities is +inf
    double value = none;
    int token = -1;                      // this lane's entry of the beam's list
    if (done) {
      if (score > none) {                // the end token, then the others in their order
        value = lane == 0 ? score : none;
        token = lane == 0 ? a.eos : lane - (lane <= a.eos);
      }
    } else {
      float top = s.x;
      for (int i = 32 + lane; i < a.parts; i += 32) top = fmaxf(top, a.sums[at * a.parts + i].x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      double sum = run_sum(s, top);
      for (int i = 32 + lane; i < a.parts; i += 32) {
        s = a.sums[at * a.parts + i];
        sum += run_sum(s, top);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const double log_sum = log(sum) + static_cast<double>(top);
      uint2 best = make_uint2(0u, 0x7fffffffu);
      for (long long e0 = 0; e0 < entries; e0 += 32 * AT_ONCE) {
        uint32_t key[AT_ONCE + 1] = {best.x};
        int tokens[AT_ONCE + 1] = {static_cast<int>(best.y)};
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
          const long long e = e0 + i * 32 + lane;
          if (e0) first[i] = e < entries ? a.lists[at * entries + e] : make_uint2(0u, 0x7fffffffu);
          key[i + 1] = first[i].x; tokens[i + 1] = static_cast<int>(first[i].y);
        }
        for (int e = 0; e < K; ++e) {
          const uint2 x = take_best(key, tokens);
          if (lane == e) best = x;
        }
      }
      if (best.x) { value = score + (static_cast<double>(key_value(best.x)) - log_sum); token = static_cast<int>(best.y); }
      if (!(value == value)) value = none;
    }
    if (__shfl_sync(0xffffffffu, value, 0) == none) token = lane;      // nothing of this beam counts: its first tokens
    if (lane < K) { s_value[row][lane] = token >= 0 && token < V ? order_key(value) : 0ull; s_token[row][lane] = token; }
  }
  __syncthreads();
  if (w) return;
  int at = 0;                            // of this lane's beam
  unsigned long long mine = lane < K ? s_value[lane][0] : 0ull;
  for (int i = 0; i < K; ++i) {
    // the best value, then the lowest beam: within a beam the list has the order of the tokens
    const uint32_t hi = static_cast<uint32_t>(mine >> 32), lo = static_cast<uint32_t>(mine);
    const uint32_t top_hi = __reduce_max_sync(0xffffffffu, hi), top_lo = __reduce_max_sync(0xffffffffu, hi == top_hi ? lo : 0u);
    const int row = __ffs(__ballot_sync(0xffffffffu, hi == top_hi && lo == top_lo)) - 1;
    if (lane == row) {
      const size_t o = static_cast<size_t>(b) * K + i;
      const int token = s_token[lane][at];
      a.out_scores[o] = static_cast<float>(key_value(mine));
      a.out_tokens[o] = token;
      a.out_parents[o] = lane;
      if (a.done) a.out_done[o] = a.done[static_cast<size_t>(b) * K + lane] || token == a.eos;
      ++at;
      mine = at < K ? s_value[lane][at] : 0ull;
    }
  }
}

// Chunks of a run: as many warps as there are at once share them all.  Runs of a row.
static int beam_chunks(int B, int K, int V, int size) {
  const long long chunks = (static_cast<long long>(V) * size + BEAM_CHUNK - 1) / BEAM_CHUNK, warps = static_cast<long long>(BEAM_AT_ONCE) * sm_count_current();
  const long long each = (chunks * B * K + warps - 1) / warps;
  return static_cast<int>(each < chunks ? each : chunks);
}
static int beam_runs(int V, int size, int chunks) {
  return static_cast<int>(((static_cast<long long>(V) * size + BEAM_CHUNK - 1) / BEAM_CHUNK + chunks - 1) / chunks);
}

}  // namespace axb

using namespace axb;

// 32-bit words of the workspace: two per row and run, then two per entry of their lists
extern "C" long long axb_beam_select_words(int B, int K, int V, int dtype) {
  const int size = dtype == 2 ? 4 : 2;
  return 2ll * B * K * beam_runs(V, size, beam_chunks(B, K, V, size)) * (1 + K);
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
  const int size = dtype == 2 ? 4 : 2, chunks = beam_chunks(B, K, V, size), parts = beam_runs(V, size, chunks);
  const long long items = static_cast<long long>(B) * K * parts;
  const BeamArgs a{logits, scores, (const unsigned char*)done, out_scores, out_tokens, out_parents, (unsigned char*)out_done,
                   (float2*)work, (uint2*)work + items, K, V, eos, parts, chunks, items};
  const bool vec = (reinterpret_cast<uintptr_t>(logits) & 15) == 0 && static_cast<long long>(V) * size % 16 == 0;
  void (*kern)(BeamArgs) = dtype == 0 ? (vec ? beam_rows_kernel<__nv_bfloat16, true> : beam_rows_kernel<__nv_bfloat16, false>)
                           : dtype == 1 ? (vec ? beam_rows_kernel<__half, true> : beam_rows_kernel<__half, false>)
                                        : (vec ? beam_rows_kernel<float, true> : beam_rows_kernel<float, false>);
  const long long blocks = (items + BEAM_WARPS - 1) / BEAM_WARPS;
  if (blocks > 0x7fffffffll) { set_error("beam_select: too many logits in one call"); return -1; }
  AXB_CUDA(pdl_launch(kern, dim3((unsigned)blocks), dim3(32 * BEAM_WARPS), 0, (cudaStream_t)stream, a));
  AXB_CUDA(pdl_launch(beam_select_kernel, dim3(B), dim3(SELECT_THREADS), 0, (cudaStream_t)stream, a));
  return 0;
}
