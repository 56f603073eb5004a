// Log-probabilities of given tokens, entropy and best alternatives of rows of logits, and their gradient.
//
//   d_j = (z_j - m) scale, m = max z;  s = sum exp(d_j);  w = sum exp(d_j) d_j
//   log-probability of t: d_t - log s;  entropy: log s - w / s;  alternatives: the largest z, equal ones in their order
//   dz_j = scale ( sum_i g_i [j = t_i] - p_j ( sum_i g_i + h (d_j - log s + H) ) ),  p_j = exp(d_j) / s
// with g_i the gradients of the log-probabilities of the token and of the alternatives t_i, h that of the entropy H.
//
// Bound by reading the logits, once forward and once backward (which writes as many).  Forward, a row belongs to a block, or to a cluster
// where there are few rows: its blocks put their statistics together through distributed shared memory, in one launch and without a
// workspace.  A thread keeps its own maximum and rescales its sums when 16-byte words of the next tile raise it.
//
// Alternatives come in the same pass.  The K-th largest of the threads' maxima so far (of 32 of them, the largest of every warp's) is
// reached by K of the values, and by few others: what is above it goes to a list in shared memory.  The bound is taken anew whenever the
// values behind it have doubled.  Values that equal it count in the first tile only: later ones come after K that are no
// smaller.  In the end what is below the last bound is dropped and the rest put in order by counting.  Where the list was too short (rows that
// grow, or of mostly equal values) the row is read again for what is above the last bound, and for the first values that equal it if these
// are fewer than K; so it is for -inf, which no list has.  Rows with NaN are gone through word by word, the list cut down to K after each.
//
// One B200, device time: 4096 rows of 128,256 bf16 values with entropy 161.8 us (their bytes at the copy's rate: 160.7), the gradient 336
// (321); 8 x 2047 rows of 50,304, 15 % of them ignored, 219 (214).  6.4 instructions a value, 8.0 with entropy.  64 rows of 128,256
// with 20 alternatives 16.1 to 16.9 us, without 7: a chain of loads, bounds, lists and the exchange, in which no other block fills in.
// Tried: words with values above the bound one after another by the whole warp (4096 rows of 32,000, 20 alternatives: 106 us for 96), every
// value of a tile by the thread that has it (more instructions still), bounds by 16 counts over the block (64 rows, one alternative: 20.6
// us for 12.4), one list with atomics for the block (no faster), registers for four blocks an SM instead of three (no faster).
#include <type_traits>

#include "common.cuh"

namespace axb {

constexpr int TP_MOST = 32;                // alternatives
// 16-byte words of a thread, of a tile: 4, the next ones loaded before these are used, or 8 without, where a block has that many: 4096 rows of
// 32,000 bf16 values 45.9 us for 48.6, 64 of 128,256 with 20 alternatives (a part of the vocabulary masked) 14.4 for 16.5; a row of 32,000 over 8
// blocks 7.0 for 6.5.
constexpr int TP_FEW_WORDS = 4, TP_MANY_WORDS = 8;
constexpr int TP_KEEP = 64;                // entries that a list is cut down to, at most
constexpr float TP_LOG2E = 1.4426950408889634f;
constexpr double TP_LN2 = 0.6931471805599453;
// Bytes of a row that a warp takes, up to 8 alternatives (4000 rows of 4000 bf16 values: 18.2 us with 8 for 26.7 with blocks of 128 threads,
// 57 with 24 for 28) and 20 of half as many (16384 rows of 2000: 54 us with 20 for 101; 300 of 1500 with 24: 22 for 7, as 32 maxima bound
// the 24th of so few values badly).  Of 4000 rows and more it saves throughout, of 1200 up to 2000 values with 8 (9.7 us for 11.3; 4000 values
// 14.7 for 11.6), of fewer up to 1000 values (300 with 8: 4.9 for 6.5); otherwise few rows wait for one warp's longer chain, by up to 3 us: 64 of
// 4000 with 8 9.0 for 6.5, 300 of 1500 with 20 8.0 for 7.1, one of 2000 with 20 6.9 for 4.6.  TP_MIDDLE: bytes that a block of 128 threads
// takes where there are few rows (one of 32,000 bf16 values, 5 alternatives: 6.9 us with clusters of 256, 7.3 with those of 128).  Many
// rows always take 128: their last tile is emptier with 256 (8 x 2047 rows of 50,304 values 221 us for 251).
constexpr long long TP_NARROW = 8192, TP_MIDDLE = 32768;
// Blocks per SM up to which rows are split over clusters, where alternatives are asked for: 64 rows of 128,256 values with 20 of them 16.1 us,
// with 4 blocks 17.1; 148 of them 24.4 for 27.7, 64 of 32,000 10.7 for 13.8 (100 of 50,304 with 5 13.8 for 13.1).
constexpr long long TP_ROOM = 2;
// Factors 1 / temperature: a flushed one times -inf would be NaN, and so would the maximum's zero times one that overflows.
constexpr float TP_COLDEST = 0x1p-100f;
constexpr float TP_FAR = -8192.f;          // exponents below are this: their powers are zero, and their products with them too

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

// 32-bit key with the order of the numbers, a NaN above all of them; -0 counts as 0.  Every key is above 0 and below 2^32 - 1.
__device__ __forceinline__ uint32_t tp_key(float x) {
  if (x != x) return 0xff800001u;            // +inf has 0xff800000
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t TP_LOWEST = 0x007fffffu, TP_ZERO = 0x80000000u;  // of -inf, of 0
__device__ __forceinline__ float tp_key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

__device__ __forceinline__ float tp_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two 32-bit numbers in a register pair.
struct Two {
  unsigned long long p;
  __device__ __forceinline__ Two() {}
  __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b)); }
  __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
};
__device__ __forceinline__ Two operator+(Two a, Two b) { Two d; asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(d.p) : "l"(a.p), "l"(b.p)); return d; }
__device__ __forceinline__ Two operator*(Two a, Two b) { Two d; asm("mul.rn.ftz.f32x2 %0, %1, %2;" : "=l"(d.p) : "l"(a.p), "l"(b.p)); return d; }
__device__ __forceinline__ Two fma(Two a, Two b, Two c) {
  Two d;
  asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(d.p) : "l"(a.p), "l"(b.p), "l"(c.p));
  return d;
}

// 16 bytes of logits
template <typename T> struct Word {
  static constexpr int COUNT = 16 / sizeof(T);
  uint32_t u[4];
  __device__ __forceinline__ void pair(int i, float& a, float& b) const {       // values 2 i and 2 i + 1
    if constexpr (__is_same(T, float)) { a = __uint_as_float(u[2 * i]); b = __uint_as_float(u[2 * i + 1]); }
    else if constexpr (__is_same(T, __nv_bfloat16)) { a = __uint_as_float(u[i] << 16); b = __uint_as_float(u[i] & 0xffff0000u); }
    else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      a = f.x; b = f.y;
    }
  }
  __device__ __forceinline__ float one(int i) const {                           // value i
    const int k = __is_same(T, float) ? i : i / 2;
    const uint32_t lower = k & 1 ? u[1] : u[0], upper = k & 1 ? u[3] : u[2], x = k & 2 ? upper : lower;
    if constexpr (__is_same(T, float)) return __uint_as_float(x);
    else if constexpr (__is_same(T, __nv_bfloat16)) return __uint_as_float(i & 1 ? x & 0xffff0000u : x << 16);
    else return __half2float(__ushort_as_half(static_cast<unsigned short>(i & 1 ? x >> 16 : x & 0xffffu)));
  }
  // bit i: value i is above x, one of the type's numbers, or is x where that counts
  __device__ __forceinline__ unsigned reaching(float x, bool equal) const {
    if constexpr (__is_same(T, float)) {
      unsigned hits = 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) hits |= (equal ? __uint_as_float(u[i]) >= x : __uint_as_float(u[i]) > x) ? 1u << i : 0u;
      return hits;
    } else {
      using H = std::conditional_t<__is_same(T, __half), __half2, __nv_bfloat162>;
      Word like;
      like.set_pair(0, x, x);
      const H* h = reinterpret_cast<const H*>(u);
      const H bound = *reinterpret_cast<const H*>(like.u);
      unsigned m[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) m[i] = equal ? __hge2_mask(h[i], bound) : __hgt2_mask(h[i], bound);
      const unsigned all = (m[0] & 0x00020001u) | (m[1] & 0x00080004u) | (m[2] & 0x00200010u) | (m[3] & 0x00800040u);
      return (all | all >> 16) & 0xffu;
    }
  }
  __device__ __forceinline__ void set_pair(int i, float a, float b) {
    if constexpr (__is_same(T, float)) { u[2 * i] = __float_as_uint(a); u[2 * i + 1] = __float_as_uint(b); }
    else if constexpr (__is_same(T, __nv_bfloat16)) { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); u[i] = *reinterpret_cast<const uint32_t*>(&h); }
    else { const __half2 h = __floats2half2_rn(a, b); u[i] = *reinterpret_cast<const uint32_t*>(&h); }
  }
  __device__ __forceinline__ float largest() const {                            // NaN left out
    if constexpr (__is_same(T, float))
      return fmaxf(fmaxf(__uint_as_float(u[0]), __uint_as_float(u[1])), fmaxf(__uint_as_float(u[2]), __uint_as_float(u[3])));
    else {
      using H = std::conditional_t<__is_same(T, __half), __half2, __nv_bfloat162>;
      const H* h = reinterpret_cast<const H*>(u);
      const H m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
      Word w;
      w.u[0] = *reinterpret_cast<const uint32_t*>(&m);
      float a, b;
      w.pair(0, a, b);
      return fmaxf(a, b);
    }
  }
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

// A row of V values as 16-byte words on the 16-byte boundaries of `like` (the row itself, or the row that its gradient is written to):
// word i holds values [i COUNT - lead, (i + 1) COUNT - lead), of which the first and the last may have some only.  What is not there is -inf.
template <typename T> struct RowWords {
  static constexpr int COUNT = Word<T>::COUNT;
  const T* z;
  int V, lead, words, shift;                 // shift: bytes from the boundary in front of a word to the word, in the row itself
  __device__ __forceinline__ RowWords(const T* z_, int V_, const T* like) : z(z_), V(V_) {
    lead = static_cast<int>(reinterpret_cast<unsigned long long>(like) % 16 / sizeof(T));
    words = (V + lead + COUNT - 1) / COUNT;
    shift = static_cast<int>((reinterpret_cast<unsigned long long>(z_) - reinterpret_cast<unsigned long long>(like)) & 15u);
  }
  __device__ __forceinline__ bool whole(int i) const { return i * COUNT >= lead && (i + 1) * COUNT - lead <= V; }
  __device__ __forceinline__ Word<T> operator[](int i) const {
    const int j = i * COUNT - lead;
    Word<T> w;
    if (shift == 0 && whole(i)) {
      const uint4 u = __ldcs(reinterpret_cast<const uint4*>(z + j));
      w.u[0] = u.x; w.u[1] = u.y; w.u[2] = u.z; w.u[3] = u.w;
    } else if (shift != 0 && j >= COUNT && j + 2 * COUNT <= V) {
      // the words on both sides of the boundary inside, moved together
      const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(z + j) - shift);
      const uint4 a = __ldg(p), b = __ldg(p + 1);
      uint32_t t[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
      if (shift & 8) {
#pragma unroll
        for (int k = 0; k < 6; ++k) t[k] = t[k + 2];
      }
      if (shift & 4) {
#pragma unroll
        for (int k = 0; k < 5; ++k) t[k] = t[k + 1];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) w.u[k] = __funnelshift_r(t[k], t[k + 1], 8 * (shift & 3));
    } else {
#pragma unroll
      for (int k = 0; k < COUNT; k += 2) {
        const float a = j + k >= 0 && j + k < V ? tp_value(z, j + k) : -INFINITY, b = j + k + 1 >= 0 && j + k + 1 < V ? tp_value(z, j + k + 1) : -INFINITY;
        w.set_pair(k / 2, a, b);
      }
    }
    return w;
  }
};
template <typename T> __device__ __forceinline__ Word<T> tp_nothing() {
  Word<T> w;
  for (int k = 0; k < 4; ++k) w.u[k] = __is_same(T, float) ? 0xff800000u : __is_same(T, __half) ? 0xfc00fc00u : 0xff80ff80u;
  return w;
}

// Sums with the reference m: s of exp2((z - m) c), w of that times its exponent.  m = -inf: nothing so far.
struct Stats {
  float m, s, w;
  __device__ __forceinline__ void rescale(float to, float c) {          // to >= m
    if (to == m) return;
    const float x = fmaxf((m - to) * c, TP_FAR), f = tp_exp2(x);
    w = f * (w + s * x);
    s *= f;
    m = to;
  }
};

// The logarithm of a sum: of 2^e m, m between the roots of 1/2 and 2, e log 2 + 2 atanh((m - 1) / (m + 1)) by the series of atanh, five terms
// of which leave 2^-29.  Within 2^-24 or so of the sum's; that of a 64-bit number took a row's last warp 1.2 us.
__device__ __forceinline__ double tp_log(float s) {
  if (!(s > 0.f && s < INFINITY)) return s == 0.f ? -INFINITY : s;
  int e = static_cast<int>(__float_as_uint(s) >> 23) - 127;
  float m = __uint_as_float((__float_as_uint(s) & 0x007fffffu) | 0x3f800000u);
  if (m > 1.41421356f) { m *= 0.5f; ++e; }
  const float t = __fdiv_rn(m - 1.f, m + 1.f), q = t * t;
  const float series = fmaf(q, fmaf(q, fmaf(q, fmaf(q, 1.f / 9, 1.f / 7), 1.f / 5), 1.f / 3), 1.f);
  return e * TP_LN2 + static_cast<double>(2.f * t * series);
}

using Entry = unsigned long long;            // key << 32 | 2^32 - 1 - place: the largest comes first
__device__ __forceinline__ Entry tp_entry(uint32_t key, int place) { return static_cast<Entry>(key) << 32 | (0xffffffffu - static_cast<uint32_t>(place)); }
__device__ __forceinline__ int tp_place(Entry e) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(e)); }

constexpr Entry TP_NONE = 0;                 // below all others

// Shared memory of a row's list.
template <int THREADS> struct List {
  static constexpr int ROOM = THREADS * 8 + TP_KEEP, SOME = THREADS == 32 ? TP_KEEP : 8 * TP_MOST;
  static constexpr int WARPS = THREADS / 32, SHARE = ROOM / WARPS;    // every warp fills a part of its own
  Entry entry[ROOM], some[SOME], best[TP_MOST];
  alignas(16) uint32_t bound[2][32];
  int filled[WARPS];
  int count, few, n[3];
};
// ... and of what the blocks of a cluster give to the first of them
struct Gathered {
  Entry best[8][TP_MOST];
  Stats stats[8];
};

// Threads of a row wait for one another: a warp alone (blocks of several rows), or the block.
template <int THREADS> __device__ __forceinline__ void tp_sync() {
  if constexpr (THREADS == 32) __syncwarp();
  else __syncthreads();
}

// A key that at least K of the row's threads reach with theirs: the K-th largest of 32 of these, the largest of every warp's.
template <int THREADS> __device__ __forceinline__ uint32_t bound_of(List<THREADS>& l, uint32_t key, int K, int turn) {
  constexpr int EACH = 32 / (THREADS / 32);
  const int lane = threadIdx.x & 31;
  if constexpr (THREADS == 32) {
    l.bound[turn][lane] = key;
  } else {
    uint32_t mine = 0u;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      if (i >= K) break;                     // no warp has more of the K largest
      const uint32_t most = __reduce_max_sync(0xffffffffu, key);
      if (lane == __ffs(__ballot_sync(0xffffffffu, key == most)) - 1) key = 0u;
      if (lane == i) mine = most;
    }
    if (lane < EACH) l.bound[turn][threadIdx.x / 32 * EACH + lane] = mine;
  }
  tp_sync<THREADS>();
  key = l.bound[turn][lane];
  int larger = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint4 k = *reinterpret_cast<const uint4*>(&l.bound[turn][4 * i]);
    larger += (k.x > key) + (k.y > key) + (k.z > key) + (k.w > key);
  }
  return __reduce_min_sync(0xffffffffu, larger < K ? key : 0xffffffffu);
}

// The K largest of some[0, n), n <= SOME, in their order, to best: what an entry's place is, its threads count.
template <int THREADS> __device__ __forceinline__ void put_in_order(List<THREADS>& l, int n, int K) {
  const int tid = threadIdx.x % THREADS;
  int each = 1;                              // threads of an entry
  while (each < 32 && 2 * each * n <= THREADS) each *= 2;
  const int part = tid & (each - 1);
  for (int base = 0; base < n; base += THREADS / each) {
    const int i = base + tid / each;
    const Entry e = i < n ? l.some[i] : TP_NONE;
    int rank = 0;
    for (int k = part; k < n; k += each) rank += l.some[k] > e;
    for (int o = each / 2; o > 0; o >>= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
    if (part == 0 && i < n && rank < K) l.best[rank] = e;
  }
  tp_sync<THREADS>();
}

// The K largest of the first n entries, n >= K, in their order, to best.  All threads of the block.
template <int THREADS> __device__ __noinline__ void take_best(List<THREADS>& l, int n, int K) {
  const int tid = threadIdx.x % THREADS;
  if (tid < 3) l.n[tid] = 0;
  tp_sync<THREADS>();
  Entry least = 0;
  if (n > List<THREADS>::SOME) {
    // the bits of a bound that at least K reach, until few do; entries differ, so that the last bit leaves K
    int reach = n;
    for (int bit = 63, turn = 0; bit >= 0 && reach > List<THREADS>::SOME; --bit, turn = turn == 2 ? 0 : turn + 1) {
      const Entry t = least | 1ull << bit;
      int mine = 0;
      for (int i = tid; i < n; i += THREADS) mine += l.entry[i] >= t;
      mine = __reduce_add_sync(0xffffffffu, mine);
      if ((tid & 31) == 0 && mine) atomicAdd(&l.n[turn], mine);
      tp_sync<THREADS>();
      const int all = l.n[turn];
      if (tid == 0) l.n[turn == 0 ? 2 : turn - 1] = 0;       // all have read that one
      if (all >= K) { least = t; reach = all; }
    }
    tp_sync<THREADS>();
    if (tid == 0) l.n[0] = 0;
    tp_sync<THREADS>();
  }
  for (int i = tid; i < n; i += THREADS) {
    const Entry e = l.entry[i];
    if (e >= least) l.some[atomicAdd(&l.n[0], 1)] = e;
  }
  tp_sync<THREADS>();
  put_in_order(l, l.n[0], K);
}
// ... which the list then consists of.  Returns the key of the last.
template <int THREADS> __device__ __forceinline__ uint32_t keep_best(List<THREADS>& l, int n, int K) {
  const int tid = threadIdx.x % THREADS;
  take_best(l, n, K);
  if (tid < K) l.entry[tid] = l.best[tid];
  if (tid == 0) l.count = K;
  tp_sync<THREADS>();
  return static_cast<uint32_t>(l.best[K - 1] >> 32);
}

// The list of words [from, to) by their keys, a word of every thread at a time: what comes later counts where its key is above the K-th so far.
template <typename T, int THREADS> __device__ __noinline__ void gather_slowly(List<THREADS>& l, const RowWords<T>& row, int from, int to, int K) {
  const int tid = threadIdx.x % THREADS;
  uint32_t over = 0u;
  tp_sync<THREADS>();                        // all have read the count
  if (tid == 0) l.count = 0;
  tp_sync<THREADS>();
  for (int base = from; base < to; base += THREADS) {
    const int i = base + tid, j0 = i * Word<T>::COUNT - row.lead;
    if (i < to) {
      for (int k = 0; k < Word<T>::COUNT; ++k) {
        const int j = j0 + k;
        if (j < 0 || j >= row.V) continue;
        const uint32_t key = tp_key(tp_value(row.z, j));
        if (key > over) l.entry[atomicAdd(&l.count, 1)] = tp_entry(key, j);
      }
    }
    tp_sync<THREADS>();
    const int n = l.count;
    tp_sync<THREADS>();
    if (n > TP_KEEP) over = keep_best(l, n, K);
  }
}

// The list of words [from, to) with the keys above `over`, which K of them reach (TP_LOWEST: or not); with the first ones that equal it, where
// the others are fewer than K.  `listed` >= 0: the others are there already, in `some`.
// A second reading, mostly from the L2: 1000 rows of 128,256 bf16 values that grow, 5 alternatives, 274 us (random ones 56); word by word with
// the list cut down each time 2606.
template <typename T, int THREADS> __device__ __noinline__ void gather_again(List<THREADS>& l, const RowWords<T>& row, int from, int to, uint32_t over, int listed, int K) {
  constexpr int COUNT = Word<T>::COUNT;
  const int tid = threadIdx.x % THREADS;
  const float bound = tp_key_value(over);
  tp_sync<THREADS>();
  if (tid < listed) l.entry[tid] = l.some[tid];
  if (tid == 0) l.count = max(listed, 0);
  tp_sync<THREADS>();
  if (listed < 0) {
    for (int i = from + tid; i < to; i += THREADS) {
      const Word<T> w = row[i];
      for (unsigned hits = w.reaching(bound, false); hits; hits &= hits - 1u) {
        const int k = __ffs(hits) - 1;
        const uint32_t key = tp_key(w.one(k));
        if (key <= over) continue;           // a value that counts as zero
        const int at = atomicAdd(&l.count, 1);
        if (at < List<THREADS>::ROOM) l.entry[at] = tp_entry(key, i * COUNT - row.lead + k);
      }
    }
    tp_sync<THREADS>();
  }
  int n = l.count;
  tp_sync<THREADS>();                        // all have read the count
  if (n > List<THREADS>::ROOM) {
    gather_slowly<T, THREADS>(l, row, from, to, K);
    return;
  }
  for (int base = from; base < to && n < K; base += THREADS) {
    const int i = base + tid;
    if (i < to) {
      const Word<T> w = row[i];
#pragma unroll
      for (int k = 0; k < COUNT; ++k) {
        const int j = i * COUNT - row.lead + k;
        if (tp_key(w.one(k)) == over && j >= 0 && j < row.V) l.entry[atomicAdd(&l.count, 1)] = tp_entry(over, j);
      }
    }
    tp_sync<THREADS>();
    n = l.count;
    tp_sync<THREADS>();
  }
}

__device__ __forceinline__ uint32_t tp_ctas() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
// Into the shared memory of the cluster's first block, where the variable is at the same address.
__device__ __forceinline__ uint32_t tp_of_first(const void* p) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(0));
  return a;
}
__device__ __forceinline__ void tp_give(float* to, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(tp_of_first(to)), "f"(v) : "memory");
}
__device__ __forceinline__ void tp_give(Entry* to, Entry v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(tp_of_first(to)), "l"(v) : "memory");
}
template <int LANES> __device__ __forceinline__ Stats tp_join_lanes(Stats t, float c) {
  float m = t.m;
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  t.rescale(m, c);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    t.s += __shfl_xor_sync(0xffffffffu, t.s, o);
    t.w += __shfl_xor_sync(0xffffffffu, t.w, o);
  }
  return t;
}

// Threads of a block: four rows of a warp each, or one row.
template <int THREADS> constexpr int TP_BLOCK = THREADS == 32 ? 128 : THREADS;

template <typename T, bool ENTROPY, bool TOP, int THREADS, int WORDS>
__global__ void __launch_bounds__(TP_BLOCK<THREADS>)
token_probs_kernel(const TokenProbsArgs a, int rows, float* log_probs, float* entropy, float* top_log_probs, long long* top_tokens, float4* stats) {
  constexpr int COUNT = Word<T>::COUNT, TILE = THREADS * WORDS, WARPS = THREADS / 32;
  constexpr int ROWS = TP_BLOCK<THREADS> / THREADS;
  __shared__ Stats s_stats[WARPS];
  __shared__ std::conditional_t<(ROWS > 1), int, Gathered> s_gathered;
  __shared__ std::conditional_t<TOP, List<THREADS>, int> s_lists[ROWS];
  pdl_launch_next();
  pdl_wait();
  const int tid = threadIdx.x % THREADS, lane = tid & 31, K = a.top;
  const int ctas = ROWS > 1 ? 1 : static_cast<int>(tp_ctas()), cta = ROWS > 1 ? 0 : static_cast<int>(cluster_cta_rank());
  if (ROWS > 1 && blockIdx.x * ROWS + threadIdx.x / THREADS >= static_cast<unsigned>(rows)) return;
  const int line = ROWS > 1 ? static_cast<int>(blockIdx.x * ROWS + threadIdx.x / THREADS) : blockIdx.x / ctas;
  const int b = line / a.per_batch, r = line - b * a.per_batch;
  auto& s_list = s_lists[ROWS > 1 ? threadIdx.x / THREADS : 0];
  const T* z = static_cast<const T*>(a.logits) + b * a.batch_stride + r * a.row_stride;
  const long long token = a.tokens ? a.tokens[b * a.token_batch_stride + r * a.token_stride] : 0;
  const RowWords<T> row(z, a.V, z);
  const int share = (row.words + ctas - 1) / ctas, from = min(cta * share, row.words), to = min(from + share, row.words);
  // whole words are [lo, hi); the values in front of and behind them, of the row's first and last word, are taken one by one
  const int lo = from + (from == 0 && row.lead > 0), hi = to - (to == row.words && to > lo && !row.whole(to - 1));
  const int head = from == 0 && to > 0 && row.lead > 0 ? min(COUNT - row.lead, a.V) : 0;
  const int behind = to == row.words && to > 0 ? max(hi * COUNT - row.lead, head) : a.V;
  const uint4* words = reinterpret_cast<const uint4*>(z - row.lead);
  const float c = a.scale * TP_LOG2E;
  const Word<T> nothing = tp_nothing<T>();
  Word<T> next[WORDS];
  const auto load = [&](Word<T>& w, int i) {
    const uint4 u = __ldcs(words + i);
    w.u[0] = u.x; w.u[1] = u.y; w.u[2] = u.z; w.u[3] = u.w;
  };
  const auto fetch = [&](int base) {
    if (base + TILE <= hi) {
#pragma unroll
      for (int k = 0; k < WORDS; ++k) load(next[k], base + tid + k * THREADS);
    } else {
#pragma unroll
      for (int k = 0; k < WORDS; ++k) {
        next[k] = nothing;
        if (base + tid + k * THREADS < hi) load(next[k], base + tid + k * THREADS);
      }
    }
  };
  const auto single = [&](float x) {         // statistics of one value: exp(x - x) is 1, or NaN
    const float y = x == -INFINITY ? 0.f : x;
    return Stats{fmaxf(x, -INFINITY), tp_exp2(x - y), 0.f};
  };
  // a warp's part of the list
  int filled = 0;
  const auto push = [&](bool hit, float x, int j) {
    if constexpr (TOP) {
      const unsigned hits = __ballot_sync(0xffffffffu, hit);
      const int at = filled + __popc(hits & ((1u << lane) - 1u));
      if (hit && at < List<THREADS>::SHARE) s_list.entry[(tid >> 5) * List<THREADS>::SHARE + at] = tp_entry(tp_key(x), j);
      filled += __popc(hits);
    }
  };
  // where few blocks run, the token is not waited for: an ignored row then costs the reading of a tile
  const bool early = ROWS > 1 || ctas > 1;
  if (early) fetch(lo);
  if (a.tokens && token == a.ignored) {     // for all blocks of a cluster
    if (cta != 0) return;
    if (tid == 0) {
      if (log_probs) log_probs[line] = 0.f;
      if (entropy) entropy[line] = 0.f;
      stats[line] = make_float4(0.f, 1.f, 0.f, 0.f);
    }
    if (TOP && tid < K) {
      top_log_probs[static_cast<long long>(line) * K + tid] = 0.f;
      top_tokens[static_cast<long long>(line) * K + tid] = -1;
    }
    return;
  }
  const long long t = token - a.start;
  float zt = 0.f;
  if (tid == 0 && a.tokens) zt = token < 0 || token >= a.total ? __int_as_float(0x7fffffff) : t >= 0 && t < a.V ? tp_value(z, static_cast<int>(t)) : 0.f;
  if constexpr (TOP) {
    if (tid == 0) s_list.count = s_list.few = 0;
    if (tid < TP_MOST) s_list.best[tid] = TP_NONE;
    tp_sync<THREADS>();
  }
  if (ROWS == 1 && ctas > 1) {
    __syncwarp();
    cluster_arrive();
  }
  if (!early) fetch(lo);
  const float x_head = tid < head ? tp_value(z, tid) : -INFINITY;
  Stats st = single(x_head);
  uint32_t over = 0u;                        // a bound that K values reach which come before the next tile
  int tiles = 0, turn = 0;
  int base = lo;
  do {
    Word<T> now[WORDS];
    float most[WORDS];
#pragma unroll
    for (int k = 0; k < WORDS; ++k) now[k] = next[k];
    if (WORDS == TP_FEW_WORDS && base + TILE < hi) fetch(base + TILE);
#pragma unroll
    for (int k = 0; k < WORDS; ++k) most[k] = now[k].largest();
    float top = most[0];
#pragma unroll
    for (int k = 1; k < WORDS; ++k) top = fmaxf(top, most[k]);
    st.rescale(fmaxf(st.m, top), c);
    const float ref = st.m == -INFINITY ? 0.f : st.m;
    const Two minus(-ref, -ref), by(c, c);
    Two s2(0.f, 0.f), w2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < WORDS; ++k) {
#pragma unroll
      for (int i = 0; i < COUNT / 2; ++i) {
        float u, v;
        now[k].pair(i, u, v);
        ((Two(u, v) + minus) * by).get(u, v);
        const Two e(tp_exp2(u), tp_exp2(v));
        s2 = s2 + e;
        if constexpr (ENTROPY) w2 = fma(e, Two(fmaxf(u, TP_FAR), fmaxf(v, TP_FAR)), w2);
      }
    }
    float u, v;
    s2.get(u, v);
    st.s += u + v;
    if constexpr (ENTROPY) {
      w2.get(u, v);
      st.w += u + v;
    }
    if constexpr (TOP) {
      const bool first = base == lo;
      if (first) {
        over = bound_of(s_list, tp_key(st.m), K, 0);
        if (head) push(tid < head && tp_key(x_head) >= over && x_head > -INFINITY, x_head, tid);
      }
      const bool equal = first && over > TP_LOWEST;
      // what counts as zero may be a little less
      const float bound = over <= TP_LOWEST ? -INFINITY : equal && over == TP_ZERO ? -1.17549435e-38f : tp_key_value(over);
      if (filled <= List<THREADS>::SHARE && __any_sync(0xffffffffu, equal ? top >= bound : top > bound)) {
        // every lane takes the next of its words that have such values, and the next of these: one of each for nearly all
        const int j0 = (base + tid) * COUNT - row.lead;
        unsigned some = 0u;
#pragma unroll
        for (int k = 0; k < WORDS; ++k) some |= (equal ? most[k] >= bound : most[k] > bound) && base + tid + k * THREADS < hi ? 1u << k : 0u;
        while (__any_sync(0xffffffffu, some != 0u)) {
          const int k = some ? __ffs(some) - 1 : 0;
          Word<T> w = now[0];
#pragma unroll
          for (int i = 1; i < WORDS; ++i)
#pragma unroll
            for (int h = 0; h < 4; ++h) w.u[h] = k == i ? now[i].u[h] : w.u[h];
          unsigned hits = some ? w.reaching(bound, equal) : 0u;
          some &= some - 1u;
          while (__any_sync(0xffffffffu, hits != 0u)) {
            const int i = hits ? __ffs(hits) - 1 : 0;
            push(hits != 0u, w.one(i), j0 + k * THREADS * COUNT + i);
            hits &= hits - 1u;
          }
        }
      }
      // anew after 2, 4, 8 ... tiles, where it saves more than it takes: 110 instructions of every warp, against some 100 of one for a tile
      // with values above the old bound, of which it has K / tiles (4096 rows of 32,000 values, 5 alternatives: 69.8 us, with half the factor 71.8)
      if (++tiles >= 2 && (tiles & (tiles - 1)) == 0 && K * ((hi - base) / TILE) > 2 * WARPS * tiles)
        over = bound_of(s_list, tp_key(st.m), K, turn ^= 1);
    }
    base += TILE;
    if (WORDS != TP_FEW_WORDS && base < hi) fetch(base);
  } while (base < hi);
  if (to == row.words && behind < a.V && tid < 32) {
    const bool there = lane < COUNT && behind + lane < a.V;
    const float x = there ? tp_value(z, behind + lane) : -INFINITY;
    Stats o = single(x);
    const float m = fmaxf(st.m, o.m);
    st.rescale(m, c);
    o.rescale(m, c);
    st.s += o.s; st.w += o.w;
    push(there && tp_key(x) >= over && x > -INFINITY, x, behind + lane);
  }
  const float most_of_thread = st.m;
  st = tp_join_lanes<32>(st, c);
  if (lane == 0) {
    if (WARPS > 1) s_stats[tid >> 5] = st;
    if constexpr (TOP) s_list.filled[tid >> 5] = filled;
  }
  tp_sync<THREADS>();
  if constexpr (WARPS > 1) {
    st = s_stats[lane & (WARPS - 1)];
    st = tp_join_lanes<WARPS>(st, c);
  }
  if constexpr (TOP) {
    int few = 0, before = 0, listed = -1;
    bool again = false;                      // there was no room for all
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      const int n = s_list.filled[i];
      again |= n > List<THREADS>::SHARE;
      if (i < (tid >> 5)) before += n;
      few += n;
    }
    const Entry* mine = s_list.entry + (tid >> 5) * List<THREADS>::SHARE;
    if (!again && few <= TP_KEEP) {
      for (int i = lane; i < filled; i += 32) s_list.some[before + i] = mine[i];
      tp_sync<THREADS>();
      if (few < K) {                         // values of -inf among the best, or no others in this block
        again = true;
        listed = few;
        over = TP_LOWEST;
      }
    } else {
      // those that reach a last bound: K at least
      over = bound_of(s_list, tp_key(most_of_thread), K, turn ^ 1);
      for (int i = 0; i < filled && !again; i += 32) {
        const Entry e = i + lane < filled ? mine[i + lane] : TP_NONE;
        const bool good = e != TP_NONE && static_cast<uint32_t>(e >> 32) >= over;
        const unsigned those = __ballot_sync(0xffffffffu, good);
        int at = 0;
        if (lane == 0 && those) at = atomicAdd(&s_list.few, __popc(those));
        at = __shfl_sync(0xffffffffu, at, 0) + __popc(those & ((1u << lane) - 1u));
        if (good && at < List<THREADS>::SOME) s_list.some[at] = e;
      }
      tp_sync<THREADS>();
      few = s_list.few;
      again |= few > List<THREADS>::SOME;
    }
    const bool nan = st.s != st.s;
    if (nan || again) {
      if (nan) gather_slowly<T, THREADS>(s_list, row, from, to, K);
      else gather_again<T, THREADS>(s_list, row, from, to, max(over, TP_LOWEST), listed, K);
      const int n = s_list.count;
      if (n > 0) take_best(s_list, n, min(n, K));
    } else {
      put_in_order(s_list, few, K);
    }
  }
  if constexpr (ROWS == 1) {
    if (ctas > 1) {
      __syncwarp();
      cluster_wait();                        // the first block runs
      if (tid < 32) {
        if constexpr (TOP) {
          if (lane < K) tp_give(&s_gathered.best[cta][lane], s_list.best[lane]);
        }
        if (lane == 0) {
          tp_give(&s_gathered.stats[cta].m, st.m);
          tp_give(&s_gathered.stats[cta].s, st.s);
          tp_give(&s_gathered.stats[cta].w, st.w);
        }
      }
      if constexpr (TOP) {
        if (tid == 0) s_list.few = 0;
      }
      __syncthreads();
      cluster_sync_all();
      if (cta != 0) return;
      st = (lane & 7) < ctas ? s_gathered.stats[lane & 7] : Stats{-INFINITY, 0.f, 0.f};
      st = tp_join_lanes<8>(st, c);          // 8 blocks at most
      if constexpr (TOP) {
        // what reaches the largest of the blocks' K-th
        over = __reduce_max_sync(0xffffffffu, lane < ctas ? static_cast<uint32_t>(s_gathered.best[lane][K - 1] >> 32) : 0u);
        for (int i = tid; i < ctas * TP_MOST; i += THREADS) {
          if (i % TP_MOST >= K) continue;
          const Entry e = s_gathered.best[i / TP_MOST][i % TP_MOST];
          if (e != TP_NONE && static_cast<uint32_t>(e >> 32) >= over) s_list.some[atomicAdd(&s_list.few, 1)] = e;
        }
        __syncthreads();
        put_in_order(s_list, s_list.few, K);
      }
    }
  }
  if (tid >= 32) return;
  const double log_s = tp_log(st.s);
  if (tid == 0) {
    const float H = ENTROPY ? static_cast<float>(log_s - __fdiv_rn(st.w, st.s) * TP_LN2) : 0.f;
    if (a.whole) {
      if (log_probs) log_probs[line] = static_cast<float>((static_cast<double>(zt) - st.m) * a.scale - log_s);
      if (entropy) entropy[line] = H;
    }
    stats[line] = a.whole ? make_float4(st.m, st.s, H, static_cast<float>(log_s)) : make_float4(st.m, st.s, static_cast<float>(st.w * TP_LN2), zt);
  }
  if constexpr (TOP) {
    if (tid < K) {
      const Entry e = s_list.best[tid];
      const float x = tp_key_value(static_cast<uint32_t>(e >> 32));
      const long long i = static_cast<long long>(line) * K + tid;
      top_log_probs[i] = a.whole ? static_cast<float>((static_cast<double>(x) - st.m) * a.scale - log_s) : x;
      top_tokens[i] = a.start + tp_place(e);
    }
  }
}

// The adjoint, one pass: (sub, mul, exp2, fma, mul) a value.  Words are loaded and stored past the L1, which takes 336 us for 351 with
// ordinary stores (4096 x 128,256 bf16); rows that lie differently to 16 bytes than their gradients' are put together from two words.
// out [rows, V] dense; stats (m, s, H, log s) of the whole vocabulary; null gradients are zeros.  A block has `span` words of a row.
constexpr int TP_BWD_THREADS = 256, TP_BWD_WORDS = 4;
template <typename T, bool ENTROPY>
__global__ void __launch_bounds__(TP_BWD_THREADS)
token_probs_bwd_kernel(const TokenProbsArgs a, const float4* stats, const float* d_log_probs, const float* d_entropy, const float* d_top,
                       const long long* top_tokens, T* out, int spans, int span) {
  constexpr int COUNT = Word<T>::COUNT, TILE = TP_BWD_THREADS * TP_BWD_WORDS;
  __shared__ float s_g[TP_MOST + 1];
  __shared__ long long s_t[TP_MOST + 1];
  pdl_launch_next();
  pdl_wait();
  const int tid = threadIdx.x, line = blockIdx.x / spans, part = blockIdx.x - line * spans, b = line / a.per_batch, r = line - b * a.per_batch;
  const T* z = static_cast<const T*>(a.logits) + b * a.batch_stride + r * a.row_stride;
  T* dz = out + static_cast<long long>(line) * a.V;
  const RowWords<T> row(z, a.V, dz);
  const int from = part * span, to = min(from + span, row.words);
  const auto put = [&](int i, const Word<T>& w) {
    const int j = i * COUNT - row.lead;
    if (row.whole(i)) __stcs(reinterpret_cast<uint4*>(dz + j), make_uint4(w.u[0], w.u[1], w.u[2], w.u[3]));
    else {
#pragma unroll
      for (int k = 0; k < COUNT; k += 2) {
        float x, y;
        w.pair(k / 2, x, y);
        if (j + k >= 0 && j + k < a.V) dz[j + k] = tp_store<T>(x);
        if (j + k + 1 >= 0 && j + k + 1 < a.V) dz[j + k + 1] = tp_store<T>(y);
      }
    }
  };
  const long long token = a.tokens ? a.tokens[b * a.token_batch_stride + r * a.token_stride] : 0;
  if (a.tokens && token == a.ignored) {
    Word<T> zero;
    zero.u[0] = zero.u[1] = zero.u[2] = zero.u[3] = 0u;
    for (int i = from + tid; i < to; i += TP_BWD_THREADS) put(i, zero);
    return;
  }
  const int n = 1 + (d_top ? a.top : 0);
  if (tid < n) {
    const long long i = static_cast<long long>(line) * a.top + tid - 1;
    float g = tid ? d_top[i] : d_log_probs ? d_log_probs[line] : 0.f;
    if (tid == 0 && d_log_probs && (token < 0 || token >= a.total)) g = __int_as_float(0x7fffffff);
    s_g[tid] = g;
    s_t[tid] = tid ? top_tokens[i] - a.start : a.tokens ? token - a.start : -1;
  }
  __syncthreads();
  const float4 st = stats[line];
  const float log_s = st.w, h = ENTROPY ? d_entropy[line] : 0.f, c = a.scale * TP_LOG2E;
  float all = 0.f;
  for (int i = 0; i < n; ++i) all += s_g[i];
  // exp2(x) (A + B x), x = (z - m) c
  const float by_s = -a.scale / st.y, A = by_s * (all + h * (st.z - log_s)), B = by_s * h * static_cast<float>(TP_LN2);
  const Two minus(-st.x, -st.x), by(c, c), A2(A, A), B2(B, B);
  for (int base = from; base < to; base += TILE) {
    Word<T> now[TP_BWD_WORDS];
#pragma unroll
    for (int k = 0; k < TP_BWD_WORDS; ++k)
      if (base + tid + k * TP_BWD_THREADS < to) now[k] = row[base + tid + k * TP_BWD_THREADS];
#pragma unroll
    for (int k = 0; k < TP_BWD_WORDS; ++k) {
      if (base + tid + k * TP_BWD_THREADS >= to) break;
#pragma unroll
      for (int i = 0; i < COUNT / 2; ++i) {
        float u, v;
        now[k].pair(i, u, v);
        ((Two(u, v) + minus) * by).get(u, v);
        Two e(tp_exp2(u), tp_exp2(v));
        if constexpr (ENTROPY) e = e * fma(B2, Two(fmaxf(u, TP_FAR), fmaxf(v, TP_FAR)), A2);
        else e = e * A2;
        e.get(u, v);
        now[k].set_pair(i, u, v);
      }
      put(base + tid + k * TP_BWD_THREADS, now[k]);
    }
  }
  // the tokens that have a gradient of their own, of this block's words
  __syncthreads();
  if (tid < n && s_t[tid] >= 0 && s_t[tid] < a.V) {
    const int j = static_cast<int>(s_t[tid]), i = (j + row.lead) / COUNT;
    if (i >= from && i < to) {
      const float x = (tp_value(z, j) - st.x) * c;
      float g = 0.f;
      for (int k = 0; k < n; ++k) if (s_t[k] == j) g += s_g[k];
      dz[j] = tp_store<T>(tp_exp2(x) * (A + (ENTROPY ? B * fmaxf(x, TP_FAR) : 0.f)) + g * a.scale);
    }
  }
}

static int fill(TokenProbsArgs& a, const char* what, const void* logits, long long batch_stride, long long row_stride, const long long* tokens,
                long long token_batch_stride, long long token_stride, int batches, int per_batch, int V, long long start, long long total, int top,
                float scale, long long ignored, int whole, int dtype, const float* stats, bool best) {
  if (reinterpret_cast<unsigned long long>(stats) % 16 || !stats || (top > 0 && !best)) {
    set_error("%s: statistics must be there, on 16 bytes, and the alternatives' tensors where some are asked for", what);
    return -1;
  }
  if (batches < 1 || per_batch < 1 || static_cast<long long>(batches) * per_batch > 0x7fffffffll || V < 1 || V > (1 << 30) || top < 0 ||
      top > TP_MOST || top > V || !(scale >= TP_COLDEST && scale <= 1.f / TP_COLDEST) || dtype < 0 || dtype > 2) {
    set_error("%s: %d x %d rows of %d values, %d alternatives, scale %g, type %d", what, batches, per_batch, V, top, scale, dtype);
    return -1;
  }
  a = {logits, batch_stride, row_stride, tokens, token_batch_stride, token_stride, start, total, per_batch, V, top, whole, scale, ignored};
  return 0;
}

template <typename T, bool ENTROPY, bool TOP, int THREADS>
static int tell(const TokenProbsArgs& a, long long rows, float* log_probs, float* entropy, float* top_log_probs, long long* top_tokens, float4* stats,
                cudaStream_t s) {
  // blocks of a row: as many as there is room for with four on every SM (TP_ROOM, where alternatives are asked for), each with a word at least for all of its threads
  const long long words = (a.V + Word<T>::COUNT - 1) / Word<T>::COUNT, room = (TOP ? TP_ROOM : 4ll) * sm_count_current();
  unsigned ctas = 1;
  while (THREADS > 32 && ctas < 8 && rows * ctas * 2 * THREADS <= room * 256 && words / (2 * ctas) >= THREADS) ctas *= 2;
  cudaLaunchConfig_t cfg = {};
  constexpr int ROWS = TP_BLOCK<THREADS> / THREADS;
  cfg.gridDim = dim3(static_cast<unsigned>((rows + ROWS - 1) / ROWS * ctas)); cfg.blockDim = dim3(TP_BLOCK<THREADS>); cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = max_ctas() == 0 ? 2 : 1;
  auto kernel = token_probs_kernel<T, ENTROPY, TOP, THREADS, TP_FEW_WORDS>;
  if constexpr (THREADS > 32)
    if (words / ctas >= TP_MANY_WORDS * THREADS) kernel = token_probs_kernel<T, ENTROPY, TOP, THREADS, TP_MANY_WORDS>;
  AXB_CUDA(cudaLaunchKernelEx(&cfg, kernel, a, static_cast<int>(rows), log_probs, entropy, top_log_probs, top_tokens, stats));
  return 0;
}

template <typename T>
static int tell_of(const TokenProbsArgs& a, long long rows, float* log_probs, float* entropy, float* top_log_probs, long long* top_tokens,
                   float4* stats, cudaStream_t s) {
  const bool H = entropy || !a.whole;
  const long long bytes = static_cast<long long>(a.V) * sizeof(T);
  const auto with = [&](auto threads) {
    constexpr int N = decltype(threads)::value;
    return H ? (a.top ? tell<T, true, true, N> : tell<T, true, false, N>) : (a.top ? tell<T, false, true, N> : tell<T, false, false, N>);
  };
  const bool many = rows >= 4ll * sm_count_current();
  const auto go = bytes <= TP_NARROW && a.top <= (2 * bytes <= TP_NARROW ? 20 : 8) ? with(std::integral_constant<int, 32>())
                : many || bytes <= TP_MIDDLE ? with(std::integral_constant<int, 128>()) : with(std::integral_constant<int, 256>());
  return go(a, rows, log_probs, entropy, top_log_probs, top_tokens, stats, s);
}

template <typename T>
static int untell(const TokenProbsArgs& a, long long rows, const float4* stats, const float* d_log_probs, const float* d_entropy, const float* d_top,
                  const long long* top_tokens, void* out, cudaStream_t s) {
  const long long words = a.V / Word<T>::COUNT + 2, tile = TP_BWD_THREADS * TP_BWD_WORDS, tiles = (words + tile - 1) / tile;
  long long spans = 16ll * sm_count_current() / rows;
  spans = spans < 1 ? 1 : spans > tiles ? tiles : spans;
  const long long span = (tiles + spans - 1) / spans * tile;
  spans = (words + span - 1) / span;
  AXB_CUDA(pdl_launch(d_entropy ? token_probs_bwd_kernel<T, true> : token_probs_bwd_kernel<T, false>, dim3(static_cast<unsigned>(rows * spans)),
                      dim3(TP_BWD_THREADS), 0, s, a, stats, d_log_probs, d_entropy, d_top, top_tokens, static_cast<T*>(out), static_cast<int>(spans),
                      static_cast<int>(span)));
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
           start, total, top, scale, ignored, whole, dtype, stats, top_log_probs && top_tokens)) return -1;
  const auto go = dtype == 0 ? tell_of<__nv_bfloat16> : dtype == 1 ? tell_of<__half> : tell_of<float>;
  return go(a, static_cast<long long>(batches) * per_batch, log_probs, entropy, top_log_probs, top_tokens, reinterpret_cast<float4*>(stats),
            static_cast<cudaStream_t>(stream));
}

extern "C" int axb_token_log_probs_bwd(const void* logits, long long batch_stride, long long row_stride, const long long* tokens,
                                       long long token_batch_stride, long long token_stride, const float* stats, const float* d_log_probs,
                                       const float* d_entropy, const float* d_top, const long long* top_tokens, void* out, int batches,
                                       int per_batch, int V, long long start, long long total, int top, float scale, long long ignored, int dtype,
                                       void* stream) {
  TokenProbsArgs a;
  if (fill(a, "gradient of token log-probabilities", logits, batch_stride, row_stride, tokens, token_batch_stride, token_stride, batches,
           per_batch, V, start, total, top, scale, ignored, 1, dtype, stats, !d_top || top_tokens)) return -1;
  const auto go = dtype == 0 ? untell<__nv_bfloat16> : dtype == 1 ? untell<__half> : untell<float>;
  return go(a, static_cast<long long>(batches) * per_batch, reinterpret_cast<const float4*>(stats), d_log_probs, d_entropy, d_top, top_tokens, out,
            static_cast<cudaStream_t>(stream));
}
