// Attention of new tokens over a key/value cache in blocks of 8-bit codes (see kv_cache.cu for the layout).
//
//   s = scale * ks * (q . k)      o = sum_t p_t vs v_t / sum_t p_t,   p = softmax of s over the tokens that a query sees
//
// What bounds it is reading 2 D bytes per token and KV head once.  A sequence here is the tokens of one request, KV head and group of up
// to 8 or 16 query columns (query heads of the KV head x new tokens; 128 where there are more than 48, see below); its unit of work is a
// tile of 32 tokens, after a start that counts as two.  One block per SM takes a run of units as long as every other block's, whatever the lengths of the requests, and its eight
// warps equal parts of that: a run ends inside one sequence and goes on in the next.  A sequence that one warp has seen whole is written
// at once; those that warps of a block share are put together in shared memory, those that blocks share by a second launch, always in
// the order of the tokens: the same call gives the same bits.
//
// Measured on one B200, D 128, device time: 64 requests of 17 to 8,192 tokens, 8 KV heads of 4 query heads: 90.0 us, 6.0 TB/s; 3 of 60,001
// to 131,072: 96.6 us, 6.08 TB/s; 24 of 700 to 2,048, 16 KV heads, 8 new tokens, int8: 33.3 us, 4.1 TB/s, of which the ends of the runs
// and the second launch are about 10; one request of 900 tokens 10.0 us, two launches' latency (blocks of a
// cluster that join few sequences in their shared memory, in one launch, have not been tried).  The loop alone issues in half of the
// cycles.  Tried for the long case when it took 100 us: 6, 7, 9, 12 warps per SM 113, 102, 126, 122; three tiles of a warp's ring instead
// of two 109; more than 128 KB of an SM's copies on their way at once makes all of them slower.  Starts that count as 0, 2, 4 tiles:
// ragged batch 102, 91, 91 us.
//
// A warp keeps everything in registers.  Scores are S^T = K Q^T (m16n8k16, rows = tokens), so that the few query columns fill the narrow
// side of the instruction; O^T = V^T P^T (rows = values of the head).  Which value of a head is which row or k index is free as long as
// both operands agree, and is chosen such that every thread reads 16 consecutive bytes: of K 16 values of its token, of V 16 values of
// each of its four tokens, whose bytes are then interleaved pairwise.  Codes become fp16, which holds them exactly; queries are scaled
// by a power of two into fp16 (exact but for values below 2^-28 of a row's largest at 16-bit inputs).  Scores, sums, denominators and
// outputs are 32-bit.
//
// The scale of a block of values moves into the exponent: a tile weighs exp2(s + log2 vs - m'), with m' following the maximum of that sum,
// beside exp2(s - m) for the denominator, so that neither overflows nor vanishes whatever the scales of the blocks are.  These weights are
// rounded to fp16, the type that holds the codes exactly: 2^-11 of each weight from 2^-26 (e^-18) of the largest one seen so far up, at most
// 2^-37 of that largest below, where the rest of many tokens may still count beside one whose values are next to nothing (the denominator
// has them whole).  That range is what m' is placed for (CA_RISE, CA_ROOM).
#include <cuda_fp8.h>

#include "common.cuh"

namespace axb {

constexpr int CA_TILE = 32;              // tokens of a tile: two halves of 16, the rows of an instruction
constexpr int CA_WARPS = 8;               // 6, 7, 9 or 12 are slower (above)
constexpr int CA_STAGES = 2;             // tiles of a warp's ring; three are slower
constexpr int CA_MAX_ROWS = 1024;        // requests of one launch: their tiles are counted in shared memory
constexpr int CA_LEAST_TILES = 8;        // of a block's run: shorter ones are not worth their partial sums
constexpr int CA_START = 2;              // what the start of a sequence costs a warp, in tiles
constexpr float CA_LOWEST = -3.0e38f;
// References are raised when a score exceeds the one that they were raised for by CA_RISE octaves; that of the weights stands CA_ROOM below
// it.  Weights stay below 2^(CA_ROOM + CA_RISE + 1) = 2^15, and fp16 has normal numbers down to 2^-14: 2^-(14 + CA_ROOM) = 2^-26 of a
// weight at the reference.  References raised by 8, 4, 2, 1 octaves (room for 6, 10, 12, 13): ragged batch 90.1, 90.1, 90.0, 90.0 us; 16
// columns 50.0, 50.5, 50.8, 51.0; 128 columns 139.6, 140.0, 140.1, 140.2.
constexpr float CA_RISE = 2.f, CA_ROOM = 12.f;

struct AttendArgs {
  const void* q;
  long long q_row, q_token, q_group;     // strides in elements; heads of a group are dense
  void* out;                             // [R, S, G * P, D]
  const uint8_t *k, *v;
  const float *ks, *vs;
  const int *tables, *lengths, *fresh;
  int R, S, G, P, W, N, shift;
  int groups;                            // of query columns
  float scale_log2;
  int workers;                           // blocks of the grid
  int* before;                           // [R + 1] units of the requests before each, per KV head and group
  int2* ends;                            // of every sequence: the slot of its first partial result (-1: finished), the block of its last
  float* part;                           // [2 * workers][columns][D + 4]: sums, then m, m', l
  unsigned int* status;                  // for the waits of the wide kernel
  unsigned long long timeout_ns;
};

// The units of a sequence are its tiles, after START that stand for its start.  `active` blocks share all units; block w starts at
// units * w / active.
template <int TILE, int START> __device__ __forceinline__ int sequence_units(int length) { return length ? (length - 1) / TILE + 1 + START : 0; }
__device__ __forceinline__ int active_blocks(long long units, int workers, int least) {
  const long long want = (units + least - 1) / least;
  return static_cast<int>(want < workers ? (want < 1 ? 1 : want) : workers);
}
__device__ __forceinline__ long long first_unit(long long units, int w, int active) { return units * w / active; }

// Units of the requests before each, [R + 1], and lengths, in shared memory: one scan per block of the grid.
template <int TILE, int START, int WARPS>
__device__ __forceinline__ void scan_units(const AttendArgs& a, int* before, int* lengths) {
  __shared__ int sums[WARPS];
  const int tid = threadIdx.x, lane = tid & 31, most = min(static_cast<long long>(a.W) << a.shift, 0x7fffff00ll);
  const int per = (a.R + 32 * WARPS - 1) / (32 * WARPS), r0 = tid * per;
  int mine = 0;
  for (int r = r0; r < min(r0 + per, a.R); ++r) {
    lengths[r] = min(max(a.lengths[r], 0), most);
    mine += sequence_units<TILE, START>(lengths[r]);
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const int u = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += u; }
  if (lane == 31) sums[tid >> 5] = incl;
  __syncthreads();
  int at = incl - mine;
  for (int i = 0; i < tid >> 5; ++i) at += sums[i];
  for (int r = r0; r < min(r0 + per, a.R); ++r) {
    before[r] = at;
    if (blockIdx.x == 0) a.before[r] = at;
    at += sequence_units<TILE, START>(lengths[r]);
  }
  if (r0 < a.R && r0 + per >= a.R) { before[a.R] = at; if (blockIdx.x == 0) a.before[a.R] = at; }
  __syncthreads();
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Four codes as fp16: bytes 0 and 1, bytes 2 and 3.
template <bool INT8> __device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (INT8) {      // 1024 + (x + 128) is the half with x + 128 in its low byte
    const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    w ^= 0x80808080u;
    const uint32_t l = __byte_perm(w, 0x64646464u, 0x4140), h = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&l), off), b = __hsub2(*reinterpret_cast<const __half2*>(&h), off);
    lo = *reinterpret_cast<const uint32_t*>(&a);
    hi = *reinterpret_cast<const uint32_t*>(&b);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(w));
  }
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "l"(policy) : "memory");
}
__device__ __forceinline__ uint64_t evict_first() {
  uint64_t p;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }
// Queries times 2^-e lie below 2^15, an octave under fp16's largest number, so that small values of a row keep what they can; sums of 128
// products with codes stay far inside 32 bits.  Zero and what is not finite stay as they are; for queries below 2^-103 the range is not
// used up, so that the powers of two, and their products with the softmax scale, stay normal numbers.
__device__ __forceinline__ int query_exponent(float largest) {
  const int e = static_cast<int>(__float_as_uint(largest) >> 23) - 127;
  return e > 127 || e < -126 ? 0 : max(e, -103) - 14;
}
template <int WORDS> __device__ __forceinline__ void shared_words(const uint8_t* p, uint32_t* w) {
  if constexpr (WORDS == 4) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    w[0] = u.x; w[1] = u.y;
  }
}

// A tile in shared memory: 32 rows of keys, 32 of values, then for each half ks, vs and whether the block exists.  The 16-byte words of
// a 128-byte line are exchanged such that neither the reads of K (two rows, four words each at a time) nor those of V (four rows, two
// words) meet.
template <int D> struct Stage {
  static constexpr int BYTES = CA_TILE * D, SIZE = 2 * BYTES + 32;
  static __device__ __forceinline__ int key_word(int row, int c) {
    return D == 128 ? row * 8 + (c ^ ((row & 1) << 2)) : row * 4 + c;
  }
  static __device__ __forceinline__ int value_word(int row, int c) {
    return D == 128 ? row * 8 + (c ^ (row & 6)) : (row >> 1) * 8 + ((((row & 1) << 2) + c) ^ (row & 6));
  }
};

// Shared memory of a warp: its ring, which the partial sums of its last sequence take the place of, and those of its first one where
// others follow.
template <int D, int NT> __host__ __device__ constexpr int part_bytes() { return 8 * NT * (D + 4) * 4; }
template <int D, int NT> __host__ __device__ constexpr int ring_bytes() {
  const int ring = CA_STAGES * Stage<D>::SIZE;
  return ring > part_bytes<D, NT>() ? ring : part_bytes<D, NT>();
}
template <int D, int NT> __host__ __device__ constexpr int warp_bytes() { return ring_bytes<D, NT>() + part_bytes<D, NT>(); }

// The sum of partial results of a column: references, denominator, sums; lane i has values N i .. of the D = 32 N.
template <int N> struct Partial {
  float m1 = CA_LOWEST, m2 = CA_LOWEST, l = 0.f, o[N] = {};
  // n more, in their order: row(x) are the sums of the x-th with what belongs to them behind, there(x) whether it exists.  Four at a
  // time, so that their loads wait for nothing.
  template <typename There, typename Row> __device__ __forceinline__ void add(int n, const There& there, const Row& row) {
    const int lane = threadIdx.x & 31;
    for (int x0 = 0; x0 < n; x0 += 4) {
      float f[4][N];
      float4 stat[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        stat[y] = make_float4(CA_LOWEST, CA_LOWEST, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < N; ++i) f[y][i] = 0.f;
        if (x0 + y >= n || !there(x0 + y)) continue;
        const float* z = row(x0 + y);
        stat[y] = *reinterpret_cast<const float4*>(z + 32 * N);
        if constexpr (N == 4) { const float4 u = *reinterpret_cast<const float4*>(z + lane * N); f[y][0] = u.x; f[y][1] = u.y; f[y][2] = u.z; f[y][3] = u.w; }
        else { const float2 u = *reinterpret_cast<const float2*>(z + lane * N); f[y][0] = u.x; f[y][1] = u.y; }
      }
      const float n1 = fmaxf(fmaxf(m1, fmaxf(stat[0].x, stat[1].x)), fmaxf(stat[2].x, stat[3].x));
      const float n2 = fmaxf(fmaxf(m2, fmaxf(stat[0].y, stat[1].y)), fmaxf(stat[2].y, stat[3].y));
      const float old = exp2_fast(m2 - n2);
      l *= exp2_fast(m1 - n1);
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] *= old;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const float w = exp2_fast(stat[y].y - n2);
        l += stat[y].z * exp2_fast(stat[y].x - n1);
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] += w * f[y][i];
      }
      m1 = n1; m2 = n2;
    }
  }
  __device__ __forceinline__ void store(float* z) const {
    const int lane = threadIdx.x & 31;
    if constexpr (N == 4) *reinterpret_cast<float4*>(z + lane * N) = make_float4(o[0], o[1], o[2], o[3]);
    else *reinterpret_cast<float2*>(z + lane * N) = make_float2(o[0], o[1]);
    if (lane == 0) *reinterpret_cast<float4*>(z + 32 * N) = make_float4(m1, m2, l, 0.f);
  }
};
template <typename T> __device__ __forceinline__ uint32_t pack_row(float lo, float hi) {
  if constexpr (__is_same(T, __half)) return pack_f16(lo, hi);
  else { const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi); return *reinterpret_cast<const uint32_t*>(&b); }
}
template <typename T> __device__ __forceinline__ T* output_row(const AttendArgs& a, int r, int g, int c, int D) {
  return static_cast<T*>(a.out) + ((static_cast<size_t>(r) * a.S + c / a.P) * a.G * a.P + g * a.P + c % a.P) * D;
}
// A denominator of 0: nothing of what the column sees is there.
template <typename T, int N> __device__ __forceinline__ void write_row(T* out, const Partial<N>& p) {
  const float f = p.l != 0.f ? exp2_fast(p.m2 - p.m1) / p.l : 0.f;
  float x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = p.l != 0.f ? p.o[i] * f : 0.f;
  uint32_t* to = reinterpret_cast<uint32_t*>(out) + (threadIdx.x & 31) * (N / 2);
  if constexpr (N == 4) *reinterpret_cast<uint2*>(to) = make_uint2(pack_row<T>(x[0], x[1]), pack_row<T>(x[2], x[3]));
  else *to = pack_row<T>(x[0], x[1]);
}

// A sequence that a warp has not seen whole: its request, KV head and group of columns, and what of it was seen; ends < 0: none.
struct Open { int r, g, group, ends; };      // ends: 1 the first tile, 2 the last one

template <typename T, int D, bool INT8, int NT>
__global__ void __launch_bounds__(32 * CA_WARPS, 1) attend_kernel(const AttendArgs a) {
  constexpr int KC = D / 64, MT = D / 16, VW = D / 32, COLS = 8 * NT;
  extern __shared__ __align__(16) uint8_t ring[];      // of every warp; then the units of the requests before each, [R + 1], and lengths
  int* before = reinterpret_cast<int*>(ring + CA_WARPS * warp_bytes<D, NT>());
  int* lengths = before + a.R + 1;
  __shared__ Open open[CA_WARPS][2];         // the sequences that a warp has not seen whole: its first and its last
  pdl_launch_next();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, g8 = lane >> 2, j4 = lane & 3, BT = 1 << a.shift;
  scan_units<CA_TILE, CA_START, CA_WARPS>(a, before, lengths);
  const uint64_t policy = evict_first();     // read once: what else is in the L2, the code of the ends among it, stays there
  const int per_tile = a.G * a.groups;
  const long long units = static_cast<long long>(before[a.R]) * per_tile;
  const int active = active_blocks(units, a.workers, CA_LEAST_TILES);
  if (blockIdx.x >= active || units == 0) return;
  const long long first = first_unit(units, blockIdx.x, active), many = first_unit(units, blockIdx.x + 1, active) - first;
  const long long begin = first + many * wid / CA_WARPS, end = first + many * (wid + 1) / CA_WARPS;
  if (lane < 2) open[wid][lane].ends = -1;
  __syncwarp();

  int r = 0;
  for (int hi = a.R; hi - r > 1;) { const int mid = (r + hi) / 2; if (before[mid] <= begin / per_tile) r = mid; else hi = mid; }
  for (long long u = begin; u < end;) {
    while (before[r + 1] <= u / per_tile) ++r;
    const int per_sequence = before[r + 1] - before[r], tiles = per_sequence - CA_START;
    const long long within = u - static_cast<long long>(before[r]) * per_tile;
    const int item = static_cast<int>(within / per_sequence), g = a.groups == 1 ? item : item / a.groups, group = item - g * a.groups;
    const int x0 = static_cast<int>(within - static_cast<long long>(item) * per_sequence);
    const int x1 = static_cast<int>(min(static_cast<long long>(per_sequence), x0 + (end - u)));
    u += x1 - x0;
    const int t0 = max(x0 - CA_START, 0), t1 = x1 - CA_START;
    if (t1 <= t0) continue;
    const int length = lengths[r], fresh = a.fresh ? min(max(a.fresh[r], 0), a.S) : a.S;
    const int col0 = group * COLS, cols = min(a.S * a.P - col0, COLS);

    // the ids of 32 blocks, one per lane, ahead of their use
    const int* table = a.tables + static_cast<size_t>(r) * a.W;
    const int halves = (length + 15) / 16, down_shift = a.shift - 4;      // halves of tiles to blocks
    int id_base = 2 * t0 >> down_shift;
    int ids = id_base + lane < a.W ? table[id_base + lane] : -1;
    uint8_t* mine = ring + wid * warp_bytes<D, NT>();
    auto fetch = [&](int t, int stage) {
      if (t < t1) {
        const uint32_t to = smem_u32(mine) + stage * Stage<D>::SIZE;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int half = 2 * t + h, b = half >> down_shift;
          if (b - id_base == 32) { id_base = b; ids = b + lane < a.W ? table[b + lane] : -1; }
          const int id = __shfl_sync(0xffffffffu, ids, b - id_base);
          const bool there = half < halves && id >= 0 && id < a.N;
          if (lane == 0) asm volatile("st.shared.b32 [%0], %1;" ::"r"(to + 2 * Stage<D>::BYTES + 16 * h + 8), "r"(static_cast<int>(there)) : "memory");
          if (!there) continue;
          const size_t head = static_cast<size_t>(id) * a.G + g;
          if (lane < 2) copy4(to + 2 * Stage<D>::BYTES + 16 * h + 4 * lane, (lane ? a.vs : a.ks) + head);
          const size_t from = ((head << a.shift) + ((half * 16) & (BT - 1))) * D;
#pragma unroll
          for (int x = 0; x < D / 32; ++x) {
            const int i = x * 32 + lane, row = 16 * h + i / (D / 16), c = i % (D / 16);
            copy16(to + Stage<D>::key_word(row, c) * 16, a.k + from + i * 16, policy);
            copy16(to + Stage<D>::BYTES + Stage<D>::value_word(row, c) * 16, a.v + from + i * 16, policy);
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };

    __syncwarp();                            // the ring's last tile of the sequence before has been read
    for (int i = 0; i < CA_STAGES - 1; ++i) fetch(t0 + i, i);
    // queries as the B operand of the scores, scaled into fp16; what their columns see
    uint32_t qf[NT][D / 16][2];
    float cscale[NT][2];
    int seen[NT][2], all = 0x7fffffff;         // tokens that columns 2 j, 2 j + 1 see; those that every column sees
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int c = col0 + n * 8 + g8;
      float f[KC][16], largest = 0.f;
      if (n * 8 + g8 < cols) {
        const T* p = static_cast<const T*>(a.q) + r * a.q_row + (c / a.P) * a.q_token + g * a.q_group + (c % a.P) * D + j4 * 16;
#pragma unroll
        for (int h = 0; h < KC; ++h)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint4 w4 = __ldg(reinterpret_cast<const uint4*>(p + h * 64 + x * 8));
            const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              float2 t;
              if constexpr (__is_same(T, __half)) t = __half22float2(*reinterpret_cast<const __half2*>(&w[y]));
              else t = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[y]));
              f[h][x * 8 + 2 * y] = t.x; f[h][x * 8 + 2 * y + 1] = t.y;
              largest = fmaxf(largest, fmaxf(fabsf(t.x), fabsf(t.y)));
            }
          }
      } else {
#pragma unroll
        for (int h = 0; h < KC; ++h)
#pragma unroll
          for (int x = 0; x < 16; ++x) f[h][x] = 0.f;
      }
      largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
      largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
      const int e = query_exponent(largest);
      const float up = power_of_two(-e), down = power_of_two(e) * a.scale_log2;
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
        const float* x = &f[s / 4][(s % 4) * 4];
        qf[n][s][0] = pack_f16(x[0] * up, x[1] * up);
        qf[n][s][1] = pack_f16(x[2] * up, x[3] * up);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        cscale[n][h] = __shfl_sync(0xffffffffu, down, (2 * j4 + h) * 4);
        const int cc = n * 8 + 2 * j4 + h, i = (col0 + cc) / a.P;
        seen[n][h] = cc < cols && i < fresh ? min(max(length - fresh + i + 1, 0), length) : 0;
        if (seen[n][h] > 0) all = min(all, seen[n][h]);
      }
    }
    all = __reduce_min_sync(0xffffffffu, all);

    float acc[NT][MT][4], m1[NT][2], m2[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[n][i][0] = acc[n][i][1] = acc[n][i][2] = acc[n][i][3] = 0.f;
      m1[n][0] = m1[n][1] = m2[n][0] = m2[n][1] = CA_LOWEST;
      l[n][0] = l[n][1] = 0.f;
    }

    int stage = 0;
    for (int t = t0; t < t1; ++t) {
      asm volatile("cp.async.wait_group %0;" ::"n"(CA_STAGES - 2) : "memory");
      __syncwarp();                          // everyone's part of this tile is there, and the tile before has been read
      fetch(t + CA_STAGES - 1, stage == 0 ? CA_STAGES - 1 : stage - 1);
      const uint8_t* at = mine + stage * Stage<D>::SIZE;
      stage = stage == CA_STAGES - 1 ? 0 : stage + 1;
      float ks[2], vs[2];
      bool there[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t w[4];
        shared_words<4>(at + 2 * Stage<D>::BYTES + 16 * h, w);
        there[h] = w[2] != 0u;
        ks[h] = there[h] ? __uint_as_float(w[0]) : 1.f;
        vs[h] = there[h] ? __uint_as_float(w[1]) : 1.f;
      }
      if (!there[0] && !there[1]) continue;

      float s[2][NT][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t k[2][D / 16];
#pragma unroll
        for (int x = 0; x < KC; ++x) {
          shared_words<4>(at + Stage<D>::key_word(16 * h + g8, 4 * x + j4) * 16, k[0] + 4 * x);
          shared_words<4>(at + Stage<D>::key_word(16 * h + g8 + 8, 4 * x + j4) * 16, k[1] + 4 * x);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) s[h][n][0] = s[h][n][1] = s[h][n][2] = s[h][n][3] = 0.f;
        float odd[NT][4] = {};             // two chains of dependent products
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          uint32_t a0, a1, a2, a3;
          widen<INT8>(k[0][i], a0, a2);
          widen<INT8>(k[1][i], a1, a3);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(i & 1 ? odd[n] : s[h][n], a0, a1, a2, a3, qf[n][i][0], qf[n][i][1]);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[h][n][i] += odd[n][i];
      }
      // vs = 2^ev fv, 1 <= fv < 2
      float ev[2], fv[2];
      bool above = false;
      const bool ragged = t * CA_TILE + CA_TILE > all || !there[0] || !there[1];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ev[h] = static_cast<float>(static_cast<int>(__float_as_uint(vs[h]) >> 23) - 127);
        fv[h] = __uint_as_float((__float_as_uint(vs[h]) & 0x7fffffu) | 0x3f800000u);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float& x = s[h][n][i];
            x *= cscale[n][i & 1] * ks[h];
            if (ragged && (!there[h] || t * CA_TILE + 16 * h + g8 + (i >> 1) * 8 >= seen[n][i & 1])) x = -INFINITY;
            above |= x > m1[n][i & 1] + CA_RISE || x + ev[h] > m2[n][i & 1] + (CA_ROOM + CA_RISE);
          }
      }
      if (__any_sync(0xffffffffu, above)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float n1 = fmaxf(fmaxf(s[0][n][i], s[0][n][i + 2]), fmaxf(s[1][n][i], s[1][n][i + 2]));
            float n2 = fmaxf(fmaxf(s[0][n][i], s[0][n][i + 2]) + ev[0], fmaxf(s[1][n][i], s[1][n][i + 2]) + ev[1]);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
              n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, o));
              n2 = fmaxf(n2, __shfl_xor_sync(0xffffffffu, n2, o));
            }
            n1 = fmaxf(m1[n][i], n1); n2 = fmaxf(m2[n][i], n2 - CA_ROOM);
            l[n][i] *= exp2_fast(m1[n][i] - n1);
            const float f = exp2_fast(m2[n][i] - n2);
            m1[n][i] = n1; m2[n][i] = n2;
#pragma unroll
            for (int y = 0; y < MT; ++y) { acc[n][y][i] *= f; acc[n][y][i + 2] *= f; }
          }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t p[NT][2], v[4][VW];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = 16 * h + 2 * j4 + (i & 1) + (i >> 1) * 8;
          // D / 8 bytes of the row: a word of 16, or half of one
          shared_words<VW>(at + Stage<D>::BYTES + (D == 128 ? Stage<D>::value_word(row, g8) * 16 : Stage<D>::value_word(row, g8 >> 1) * 16 + (g8 & 1) * 8), v[i]);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            l[n][i & 1] += exp2_fast(s[h][n][i] - m1[n][i & 1]);
            w[i] = exp2_fast(s[h][n][i] + ev[h] - m2[n][i & 1]) * fv[h];
          }
          p[n][0] = transpose8x8(pack_f16(w[0], w[1]));
          p[n][1] = transpose8x8(pack_f16(w[2], w[3]));
        }
        if (ragged) {
          // rows behind the sequence hold anything; a NaN that some columns see and others do not is kept from the others below
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!there[h] || t * CA_TILE + 16 * h + 2 * j4 + (i & 1) + (i >> 1) * 8 >= length)
#pragma unroll
              for (int w = 0; w < VW; ++w) v[i][w] = 0u;
          if constexpr (!INT8) {
            bool bad = false;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int w = 0; w < VW; ++w) bad |= __vcmpeq4(v[i][w] & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0u;
            if (__any_sync(0xffffffffu, bad)) {
              // 1 where a value is NaN, times 1 where a column sees its token: a count above zero makes the sum NaN
              uint32_t see[NT][2];
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int token = t * CA_TILE + 16 * h + g8 + 8 * e;
                  see[n][e] = transpose8x8(pack_f16(token < seen[n][0] ? 1.f : 0.f, token < seen[n][1] ? 1.f : 0.f));
                }
#pragma unroll
              for (int w = 0; w < VW; ++w) {
                uint32_t one[4];                 // 1 in e4m3
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const uint32_t nan = __vcmpeq4(v[i][w] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                  v[i][w] &= ~nan;
                  one[i] = nan & 0x38383838u;
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                  uint32_t a0, a1, a2, a3;
                  widen<false>(__byte_perm(one[0], one[1], x ? 0x7362 : 0x5140), a0, a1);
                  widen<false>(__byte_perm(one[2], one[3], x ? 0x7362 : 0x5140), a2, a3);
#pragma unroll
                  for (int n = 0; n < NT; ++n) {
                    float count[4] = {0.f, 0.f, 0.f, 0.f};
                    mma_f16(count, a0, a1, a2, a3, see[n][0], see[n][1]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) if (count[i] > 0.f) acc[n][2 * w + x][i] = __uint_as_float(0x7fffffffu);
                  }
                }
              }
            }
          }
        }
#pragma unroll
        for (int w = 0; w < VW; ++w)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            uint32_t a0, a1, a2, a3;
            widen<INT8>(__byte_perm(v[0][w], v[1][w], x ? 0x7362 : 0x5140), a0, a1);
            widen<INT8>(__byte_perm(v[2][w], v[3][w], x ? 0x7362 : 0x5140), a2, a3);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16(acc[n][2 * w + x], a0, a1, a2, a3, p[n][0], p[n][1]);
          }
      }
    }

    // thread (g8, j4) has values g8 * D / 8 .. of columns 2 j4 and 2 j4 + 1
    const bool whole = t0 == 0 && t1 == tiles;
    const int slot = u < end ? 0 : 1;        // the last of this warp's, or its first of several
    if (whole && lane == 0) a.ends[static_cast<size_t>(r) * per_tile + item] = make_int2(-1, 0);
    if (!whole) {
      __syncwarp();                          // the ring has been read: the sums take its place
      if (lane == 0) open[wid][slot] = Open{r, g, group, (t0 == 0) + 2 * (t1 == tiles)};
    }
    float* parts = reinterpret_cast<float*>(mine + (slot == 0 ? ring_bytes<D, NT>() : 0));
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float total = l[n][h];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        if (seen[n][h] <= 0) total = 0.f;
        const int cc = n * 8 + 2 * j4 + h;
        if (cc >= cols) continue;
        if (whole) {
          const float f = total != 0.f ? exp2_fast(m2[n][h] - m1[n][h]) / total : 0.f;      // 0: nothing of what the column sees is there
          T* o = output_row<T>(a, r, g, col0 + cc, D) + g8 * (D / 8);
#pragma unroll
          for (int x = 0; x < D / 64; ++x) {
            uint32_t w[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const float* z = acc[n][x * 4 + y];
              const float lo = total != 0.f ? z[h] * f : 0.f, hi = total != 0.f ? z[h + 2] * f : 0.f;
              w[y] = pack_row<T>(lo, hi);
            }
            *reinterpret_cast<uint4*>(o + x * 8) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else {
          float* o = parts + cc * (D + 4);
#pragma unroll
          for (int i = 0; i < MT; i += 2)
            *reinterpret_cast<float4*>(o + g8 * (D / 8) + 2 * i) =
                make_float4(acc[n][i][h], acc[n][i][h + 2], acc[n][i + 1][h], acc[n][i + 1][h + 2]);
          if (g8 == 0) *reinterpret_cast<float4*>(o + D) = make_float4(m1[n][h], m2[n][h], total, 0.f);
        }
      }
  }

  // Sequences that several warps of the block share: put together here, finished where the block has seen them whole.
  __syncthreads();
  // lane x looks at the x-th; a sequence starts where it is not that of the one before
  Open mine_open = {0, 0, 0, -1};
  if (lane < 2 * CA_WARPS) mine_open = (&open[0][0])[lane];
  const unsigned some = __ballot_sync(0xffffffffu, mine_open.ends >= 0), earlier = some & ((1u << lane) - 1u);
  const int prior = earlier ? 31 - __clz(earlier) : 0;
  const int prior_r = __shfl_sync(0xffffffffu, mine_open.r, prior), prior_g = __shfl_sync(0xffffffffu, mine_open.g, prior);
  const int prior_group = __shfl_sync(0xffffffffu, mine_open.group, prior);
  const bool same = earlier && prior_r == mine_open.r && prior_g == mine_open.g && prior_group == mine_open.group;
  unsigned starts = __ballot_sync(0xffffffffu, mine_open.ends >= 0 && !same);
  int turn = 0;                              // columns of all those sequences, a warp for each in turn
  while (starts) {
    const int i = __ffs(starts) - 1;
    starts &= starts - 1;
    const unsigned here = some & (starts ? (1u << (__ffs(starts) - 1)) - 1u : 0xffffffffu) & ~((1u << i) - 1u);
    const int last = 31 - __clz(here), first_r = __shfl_sync(0xffffffffu, mine_open.r, i), g = __shfl_sync(0xffffffffu, mine_open.g, i);
    const int group = __shfl_sync(0xffffffffu, mine_open.group, i);
    const int first_ends = __shfl_sync(0xffffffffu, mine_open.ends, i), last_ends = __shfl_sync(0xffffffffu, mine_open.ends, last);
    const bool whole = (first_ends & 1) && (last_ends & 2);
    const int col0 = group * COLS, cols = min(a.S * a.P - col0, COLS);
    const int skip = (wid - turn % CA_WARPS + CA_WARPS) % CA_WARPS;
    // a sequence that began in another block is this block's first
    const size_t slot = 2 * static_cast<size_t>(blockIdx.x) + (first_ends & 1);
    if (threadIdx.x == 0) {
      int2* ends = a.ends + static_cast<size_t>(first_r) * per_tile + g * a.groups + group;
      if (first_ends & 1) ends->x = whole ? -1 : static_cast<int>(slot);
      if (last_ends & 2) ends->y = blockIdx.x;
    }
    turn += cols;
    for (int cc = skip; cc < cols; cc += CA_WARPS) {
      Partial<D / 32> p;
      auto row = [&](int x) {
        x += i;
        return reinterpret_cast<const float*>(ring + x / 2 * warp_bytes<D, NT>() + (x & 1 ? 0 : ring_bytes<D, NT>())) + cc * (D + 4);
      };
      p.add(last - i + 1, [&](int x) { return (here >> (i + x) & 1u) != 0u; }, row);
      if (whole) { write_row(output_row<T>(a, first_r, g, col0 + cc, D), p); continue; }
      p.store(a.part + (slot * COLS + cc) * (D + 4));
    }
  }
}

// ----------------------------------------------------------------------------- more than 48 query columns

// The same sums on tcgen05, for groups of up to 128 columns (rows of the products: S = Q K^T, O = P V with M = 128): the codes of a tile of
// 128 tokens are widened once for all of them.  24 requests of 4,096 tokens, 8 KV heads, 128 columns: 140 us (int8 136), 52 GFLOP of
// products; about 4,000 cycles a tile, of which the exp2 unit needs 1,000.  A warp's steps wait for one another (a load of 32 scores 300
// cycles, their maximum 350, their weights 500; scores are loaded twice, once for each), and two warps per scheduler do not hide that.  All
// 17 warps have 96 registers; sharing those out by role has not been tried.  With both threads of a column on one tile, which have to
// meet in each, 17 us more.  One block per SM, with roles:
//
//   warps 0-7   softmax, two threads per column (lane of tensor memory), for every other tile each, with sums of their own: the queries
//               into shared memory, then per tile the largest score and the weights as fp16 in the place of the scores; at the end of a
//               sequence both put its sums together
//   warps 8-15  codes, of keys (8-11) and values: 16 bytes of a lane, a tile ahead in registers, widened to fp16 into shared memory
//               (128-byte rows, swizzled)
//   warp 16     the products: O += P(t) V(t), then S(t + 2) into the same buffer; two buffers of scores, sums, keys and values each
//
// Every wait is bounded.  What a column sees of a tile where it ends differs from column to column, and values that are NaN there must
// not reach those that do not see them: they become zeros, and the sums of the columns that see them NaN, afterwards.
constexpr int CW_TILE = 128;
constexpr int CW_START = 1;              // what the start of a sequence costs a block, in tiles
constexpr int CW_LEAST_TILES = 2;
constexpr int CW_COLUMNS = 128;
constexpr int CW_WARPS = 17, CW_CODE_WARPS = 4;      // all; that widen keys, and values

template <int D> struct Wide {
  static constexpr int CHUNK = 128 * 128;              // 128 rows of 64 fp16 values
  static constexpr int MATRIX = D / 64 * CHUNK;
  static constexpr int K = MATRIX, V = 3 * MATRIX, BARS = 5 * MATRIX, FIXED = BARS + 256 + 1024;
  static constexpr int ROWS = 512 / D, PASSES = D / 16;      // token rows of a warp at a time, 16 bytes per lane; times per tile
  static __device__ __forceinline__ int at(int row, int unit) { return (unit >> 3) * CHUNK + row * 128 + (((unit ^ row) & 7) << 4); }      // 16-byte unit of a row
};

__device__ __forceinline__ uint4 load_once(const void* p) {
  uint4 u;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(p));
  return u;
}
// 16 columns of tensor memory of a warp's 32 lanes.
__device__ __forceinline__ void tmem_st_32x16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      : : "r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}

// The pieces of sequences of a block's run, in their order; every role walks through them by itself.
struct WideWalk {
  long long u, end;
  int r, g, group, item, t0, t1, tiles;
  __device__ __forceinline__ WideWalk(const AttendArgs& a, const int* before) {
    const int per_tile = a.G * a.groups;
    const long long units = static_cast<long long>(before[a.R]) * per_tile;
    const int active = active_blocks(units, a.workers, CW_LEAST_TILES);
    u = end = 0;
    r = 0;
    if (blockIdx.x >= active || units == 0) return;
    u = first_unit(units, blockIdx.x, active);
    end = first_unit(units, blockIdx.x + 1, active);
    for (int hi = a.R; hi - r > 1;) { const int mid = (r + hi) / 2; if (before[mid] <= u / per_tile) r = mid; else hi = mid; }
  }
  __device__ __forceinline__ bool next(const AttendArgs& a, const int* before) {
    const int per_tile = a.G * a.groups;
    while (u < end) {
      while (before[r + 1] <= u / per_tile) ++r;
      const int per_sequence = before[r + 1] - before[r];
      const long long within = u - static_cast<long long>(before[r]) * per_tile;
      item = static_cast<int>(within / per_sequence);
      g = item / a.groups;
      group = item - g * a.groups;
      const int x0 = static_cast<int>(within - static_cast<long long>(item) * per_sequence);
      const int x1 = static_cast<int>(min(static_cast<long long>(per_sequence), x0 + (end - u)));
      u += x1 - x0;
      tiles = per_sequence - CW_START;
      t0 = max(x0 - CW_START, 0);
      t1 = x1 - CW_START;
      if (t1 > t0) return true;
    }
    return false;
  }
};

// What the columns of a group see: all that see anything the tokens below lo, none those from hi on.
struct WideSeen { int lo, hi; };
__device__ __forceinline__ WideSeen wide_seen(const AttendArgs& a, int r, int length, int group) {
  const int fresh = a.fresh ? min(max(a.fresh[r], 0), a.S) : a.S, col0 = group * CW_COLUMNS;
  const int first = col0 / a.P, last = min((min(col0 + CW_COLUMNS, a.S * a.P) - 1) / a.P, fresh - 1);
  return {min(max(length - fresh + min(first, fresh) + 1, 1), length), last < first ? 0 : min(max(length - fresh + last + 1, 0), length)};
}

template <typename T, int D, bool INT8>
__global__ void __launch_bounds__(32 * CW_WARPS, 1) attend_wide_kernel(const AttendArgs a) {
  using W = Wide<D>;
  constexpr int CODE_PASSES = W::PASSES, PASS_ROWS = W::ROWS * CW_CODE_WARPS;
  extern __shared__ uint8_t raw_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + W::BARS);
  uint64_t *k_full = bars, *k_empty = bars + 2, *v_full = bars + 4, *v_empty = bars + 6, *s_full = bars + 8, *p_full = bars + 10;
  uint64_t *meta_full = bars + 12, *q_full = bars + 16, *pv_done = bars + 17, *pair = bars + 19;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(bars + 23);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_at + 1);
  int* before = reinterpret_cast<int*>(smem + W::BARS + 256);
  int* lengths = before + a.R + 1;
  // of the last four tiles: scales, whether a block exists, tokens whose values were NaN (32 of each warp that widens them)
  __shared__ __align__(16) float4 s_scale[4][8];      // of keys; exponent and fraction of that of values
  __shared__ uint32_t s_there[4];
  __shared__ __align__(16) uint32_t s_nan[4][CW_CODE_WARPS];
  __shared__ __align__(16) float4 s_state[2][CW_COLUMNS];      // of a column's two threads at the end of a sequence
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, BT = 1 << a.shift;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], CW_CODE_WARPS); mbar_init(&v_full[i], CW_CODE_WARPS); mbar_init(&k_empty[i], 1); mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 4); mbar_init(&pv_done[i], 1);
    }
    for (int i = 0; i < 4; ++i) { mbar_init(&meta_full[i], 1); mbar_init(&pair[i], 2); }
    mbar_init(q_full, 8);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 16) { tmem_alloc(tmem_at, 512); tmem_relinquish(); }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  pdl_launch_next();                       // the tensor memory is this block's
  pdl_wait();
  scan_units<CW_TILE, CW_START, CW_WARPS>(a, before, lengths);      // ends in a barrier
  const uint32_t tmem = *tmem_at;          // scores, then weights: columns 0 .. 127 and 128 .. 255; sums: 256 .. 383 and 384 .. 511
  const uint64_t timeout = a.timeout_ns;
  bool ok = true;
  WideWalk walk(a, before);
  uint32_t cnt = 0;                        // tiles so far: buffers and phases

  if (warp < 8) {                          // ------------------------------------------------ softmax
    const int quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    uint32_t meets = 0;
    auto meet = [&] {                      // the two warps of 32 columns
      __syncwarp();
      if (lane == 0) mbar_arrive(&pair[quarter]);
      const bool met = mbar_wait(&pair[quarter], meets++ & 1, abort_flag, timeout);
      __syncwarp();
      return met;
    };
    while (ok && walk.next(a, before)) {
      const int length = lengths[walk.r], col0 = walk.group * CW_COLUMNS, cols = min(a.S * a.P - col0, CW_COLUMNS), c = col0 + row;
      const int fresh = a.fresh ? min(max(a.fresh[walk.r], 0), a.S) : a.S;
      const WideSeen see = wide_seen(a, walk.r, length, walk.group);
      const int seen = row < cols && c / a.P < fresh ? min(max(length - fresh + c / a.P + 1, 0), length) : 0;
      const bool mine = quarter * 32 < cols;      // of the warp
      // queries: the products that read the ones before are done, their scores have been seen
      float cscale = 0.f;
      {
        const T* q = static_cast<const T*>(a.q) + walk.r * a.q_row + (c / a.P) * a.q_token + walk.g * a.q_group + (c % a.P) * D;
        float largest = 0.f;
        auto value = [&](uint32_t w) {
          if constexpr (__is_same(T, __half)) return __half22float2(*reinterpret_cast<const __half2*>(&w));
          else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
        };
        if (row < cols)
#pragma unroll 4
          for (int i = 0; i < D / 8; ++i) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(q) + i);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) { const float2 f = value(w[j]); largest = fmaxf(largest, fmaxf(fabsf(f.x), fabsf(f.y))); }
          }
        const int e = query_exponent(largest);
        const float up = copysignf(power_of_two(-e), a.scale_log2);      // so that the largest score is that of the largest product
        cscale = power_of_two(e) * fabsf(a.scale_log2);
#pragma unroll 4
        for (int i = half * (D / 16); i < half * (D / 16) + D / 16; ++i) {
          uint4 u = make_uint4(0u, 0u, 0u, 0u);
          if (row < cols) {
            u = __ldg(reinterpret_cast<const uint4*>(q) + i);
            uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) { const float2 f = value(w[j]); w[j] = pack_f16(f.x * up, f.y * up); }
            u = make_uint4(w[0], w[1], w[2], w[3]);
          }
          *reinterpret_cast<uint4*>(smem + W::at(row, i)) = u;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
      }
      float m1 = CA_LOWEST, m2 = CA_LOWEST, l = 0.f;
      const uint32_t s_at = tmem + lanes + half * 128, o_at = tmem + lanes + 256 + half * 128;
      // the sums of columns that see a token whose values were NaN in tile t, the x-th so far
      auto mend = [&](int t, uint32_t x) {
        const uint4 some = *reinterpret_cast<const uint4*>(s_nan[x & 3]);
        if ((some.x | some.y | some.z | some.w) == 0u) return;
        for (int w = 0; w < CW_CODE_WARPS; ++w) {
          uint32_t bad = s_nan[x & 3][w];
          while (bad) {
            const int bit = __ffs(bad) - 1, within = bit / W::ROWS * PASS_ROWS + w * W::ROWS + bit % W::ROWS, token = t * CW_TILE + within;
            bad &= bad - 1;
            const int id = a.tables[static_cast<size_t>(walk.r) * a.W + (token >> a.shift)];
            const uint8_t* v = a.v + (((static_cast<size_t>(id) * a.G + walk.g) << a.shift) + (token & (BT - 1))) * D;
            for (int b = 0; b < D / 32; ++b) {
              uint32_t o[32];
              tmem_ld_32x32(o_at + b * 32, o);
              tmem_ld_wait(o);
#pragma unroll
              for (int i = 0; i < 32; ++i) if (token < seen && (v[b * 32 + i] & 0x7f) == 0x7f) o[i] = 0x7fffffffu;
              tmem_st_32x32(o_at + b * 32, o);
            }
            tmem_st_wait();
          }
        }
      };
      int done = -1;                       // this warp's last tile
      for (int t = walk.t0; t < walk.t1; ++t, ++cnt) {
        if ((cnt & 1) != half) continue;
        if (!mbar_wait(&meta_full[cnt & 3], (cnt >> 2) & 1, abort_flag, timeout) ||
            !mbar_wait(&s_full[half], (cnt >> 1) & 1, abort_flag, timeout)) { ok = false; break; }
        __syncwarp();
        tcgen05_fence_after();
        const uint32_t there = s_there[cnt & 3];
        const bool ragged = t * CW_TILE + CW_TILE > see.lo || there != 0xffu;
        // 32 scores, masked where the column does not see their tokens, and the scales of their two blocks
        auto scores = [&](int b0, uint32_t (&x)[32], float4 (&scale)[2]) {
          tmem_ld_32x32(s_at + b0 * 16, x);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            scale[h] = s_scale[cnt & 3][b0 + h];
            const float f = cscale * scale[h].x;
            scale[h].x = f < 1.17549435e-38f ? 1.17549435e-38f : f;      // above 0: -inf stays what it is
          }
          tmem_ld_wait(x);
          if (ragged)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int end = there >> (b0 + h) & 1u ? seen - (t * CW_TILE + 16 * (b0 + h)) : 0;
#pragma unroll
              for (int i = 0; i < 16; ++i) if (i >= end) x[h * 16 + i] = 0xff800000u;
            }
        };
        float g1 = -INFINITY, g2 = -INFINITY;
        if (mine)
#pragma unroll 1
          for (int b0 = 0; b0 < 8; b0 += 2) {
            uint32_t x[32];
            float4 scale[2];
            scores(b0, x, scale);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float top[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t* z = x + h * 16 + 4 * i;
                top[i] = fmaxf(fmaxf(__uint_as_float(z[0]), __uint_as_float(z[1])), fmaxf(__uint_as_float(z[2]), __uint_as_float(z[3])));
              }
              const float y = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale[h].x;
              g1 = fmaxf(g1, y);
              g2 = fmaxf(g2, y + scale[h].y);
            }
          }
        if (done >= 0) {                   // the sums so far: every phase of the barrier is seen, in order
          if (!mbar_wait(&pv_done[half], ((cnt >> 1) & 1) ^ 1, abort_flag, timeout)) { ok = false; break; }
          __syncwarp();
          tcgen05_fence_after();
          if (!INT8 && mine) mend(done, cnt - 2);
        }
        if (mine) {
          if (__any_sync(0xffffffffu, g1 > m1 + CA_RISE || g2 > m2 + (CA_ROOM + CA_RISE))) {
            const float n1 = fmaxf(m1, g1), n2 = fmaxf(m2, g2 - CA_ROOM), f = exp2_fast(m2 - n2);
            l *= exp2_fast(m1 - n1);
            m1 = n1; m2 = n2;
            if (done >= 0)
#pragma unroll 1
              for (int b = 0; b < D / 32; ++b) {
                uint32_t o[32];
                tmem_ld_32x32(o_at + b * 32, o);
                tmem_ld_wait(o);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                tmem_st_32x32(o_at + b * 32, o);
              }
          }
          float2 sum0 = make_float2(0.f, 0.f), sum1 = sum0;
#pragma unroll 1
          for (int b0 = 0; b0 < 8; b0 += 2) {      // the weights of 32 scores take the place of the first 16 of them, or of earlier ones
            uint32_t x[32], p[16];
            float4 scale[2];
            scores(b0, x, scale);
            // exp2(s + ev - m2) is exp2(s - m1) exp2(ev + m1 - m2), but where the latter would bring back what the former has lost
            const float shift[2] = {scale[0].y + m1 - m2, scale[1].y + m1 - m2};
            const bool apart = __any_sync(0xffffffffu, shift[0] > 60.f || shift[1] > 60.f);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float2 f2 = make_float2(scale[h].x, scale[h].x), low = make_float2(-m1, -m1);
              const float weight = exp2_fast(shift[h]) * scale[h].z;
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                float2 e = __ffma2_rn(make_float2(__uint_as_float(x[h * 16 + 2 * i]), __uint_as_float(x[h * 16 + 2 * i + 1])), f2, low);
                e.x = exp2_fast(e.x); e.y = exp2_fast(e.y);
                if (i & 1) sum1 = __fadd2_rn(sum1, e); else sum0 = __fadd2_rn(sum0, e);
                e = __fmul2_rn(e, make_float2(weight, weight));
                p[h * 8 + i] = pack_f16(e.x, e.y);
              }
            }
            if (apart)
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                  p[h * 8 + i] = pack_f16(exp2_fast(__uint_as_float(x[h * 16 + 2 * i]) * scale[h].x + scale[h].y - m2) * scale[h].z,
                                          exp2_fast(__uint_as_float(x[h * 16 + 2 * i + 1]) * scale[h].x + scale[h].y - m2) * scale[h].z);
            tmem_st_32x16(s_at + b0 * 8, p);
          }
          l += (sum0.x + sum0.y) + (sum1.x + sum1.y);
          tmem_st_wait();
        }
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[half]);
        done = t;
      }
      if (!ok) break;
      if (done >= 0) {                     // the warp's last tile was the piece's last or the one before
        const uint32_t x = cnt - (walk.t1 - done);
        if (!mbar_wait(&pv_done[half], (x >> 1) & 1, abort_flag, timeout)) { ok = false; break; }
        __syncwarp();
        tcgen05_fence_after();
        if (!INT8 && mine) mend(done, x);
      }
      // both halves of the tiles: each thread puts half of the values together
      s_state[half][row] = make_float4(m1, m2, l, done >= 0 ? 1.f : 0.f);
      tcgen05_fence_before();
      if (!meet()) { ok = false; break; }
      tcgen05_fence_after();
      const float4 other = s_state[half ^ 1][row];
      const bool starts = walk.t0 == 0, ends = walk.t1 == walk.tiles, whole = starts && ends;
      const size_t slot = 2 * static_cast<size_t>(blockIdx.x) + starts;
      if (tid == 0) {
        int2* at = a.ends + static_cast<size_t>(walk.r) * a.G * a.groups + walk.item;
        if (starts) at->x = whole ? -1 : static_cast<int>(slot);
        if (ends) at->y = blockIdx.x;
      }
      if (mine) {
        const float n1 = fmaxf(m1, other.x), n2 = fmaxf(m2, other.y);
        const float w0 = exp2_fast((half ? other.y : m2) - n2), w1 = exp2_fast((half ? m2 : other.y) - n2);
        const bool first = half ? other.w != 0.f : done >= 0, second = half ? done >= 0 : other.w != 0.f;
        // the first half's sum first, whichever thread adds
        const float l0 = (half ? other.z : l) * exp2_fast((half ? other.x : m1) - n1), l1 = (half ? l : other.z) * exp2_fast((half ? m1 : other.x) - n1);
        const float total = seen > 0 ? l0 + l1 : 0.f, f = total != 0.f ? exp2_fast(n2 - n1) / total : 0.f;
        float* part = a.part + (slot * CW_COLUMNS + row) * (D + 4);
        T* out = output_row<T>(a, walk.r, walk.g, c, D);
#pragma unroll 1
        for (int b = half * (D / 64); b < half * (D / 64) + D / 64; ++b) {
          float o[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.f;
#pragma unroll 1
          for (int k = 0; k < 2; ++k) {
            if (!(k ? second : first)) continue;
            uint32_t x[32];
            tmem_ld_32x32(tmem + lanes + 256 + k * 128 + b * 32, x);
            tmem_ld_wait(x);
            const float w = k ? w1 : w0;
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] += w * __uint_as_float(x[i]);
          }
          if (row >= cols) continue;
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            if (whole) {
              uint32_t w[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) w[j] = pack_row<T>(total != 0.f ? o[i + 2 * j] * f : 0.f, total != 0.f ? o[i + 2 * j + 1] * f : 0.f);
              *reinterpret_cast<uint4*>(out + b * 32 + i) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
              *reinterpret_cast<float4*>(part + b * 32 + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
              *reinterpret_cast<float4*>(part + b * 32 + i + 4) = make_float4(o[i + 4], o[i + 5], o[i + 6], o[i + 7]);
            }
          }
        }
        if (!whole && row < cols && half == 0) *reinterpret_cast<float4*>(part + D) = make_float4(n1, n2, total, 0.f);
      }
      tcgen05_fence_before();              // the next sequence's first products follow both warps' reads
      if (!meet()) { ok = false; break; }
    }
    if (!ok && lane == 0) report_status(a.status, 0x443u);
  } else if (warp < 16) {                  // ------------------------------------------------ codes: warps 8-11 keys, 12-15 values
    const int w4 = warp & 3;
    const bool keys = warp < 12;
    uint64_t *full = keys ? k_full : v_full, *empty = keys ? k_empty : v_empty;
    uint8_t* matrix = smem + (keys ? W::K : W::V);
    const uint8_t* codes = keys ? a.k : a.v;
    const int within = D == 128 ? ((lane >> 2) & 1) + 2 * (lane >> 4) : lane >> 2;      // row of the warp's; 16 bytes of it: pairs of rows
    const int c16 = D == 128 ? (lane & 3) + 4 * ((lane >> 3) & 1) : lane & 3;           // share a store's banks
    const int row0 = w4 * W::ROWS + within;
    // what is on its way of a tile
    struct Coming { uint4 x[CODE_PASSES]; float ks, vs; int lo; bool valid, there; };      // scales: of warp 8's lanes 0 .. 7
    WideSeen see = {0, 0};
    int length = 0, limit = 0, t = 0, ids = -1;      // lane i: block of tokens 16 i ..
    const int* table = nullptr;
    auto start = [&](bool fresh_piece) {
      if (fresh_piece) {
        length = lengths[walk.r];
        see = wide_seen(a, walk.r, length, walk.group);
        limit = keys ? length : see.hi;
        table = a.tables + static_cast<size_t>(walk.r) * a.W;
        t = walk.t0;
      }
      const int token = t * CW_TILE + 16 * lane;
      ids = lane < 8 && token < length ? table[token >> a.shift] : -1;
    };
    bool have = walk.next(a, before);
    if (have) start(true);
    auto fetch = [&](Coming& s) {
      s.valid = have;
      if (!have) return;
      const int id = ids >= 0 && ids < a.N ? ids : -1;
      s.lo = see.lo - t * CW_TILE;
#pragma unroll
      for (int p = 0; p < CODE_PASSES; ++p) {
        const int token = t * CW_TILE + p * PASS_ROWS + row0, block = __shfl_sync(0xffffffffu, id, (p * PASS_ROWS + w4 * W::ROWS) / 16);
        s.x[p] = make_uint4(0u, 0u, 0u, 0u);
        if (block >= 0 && token < limit)
          s.x[p] = load_once(codes + ((((static_cast<size_t>(block) * a.G + walk.g) << a.shift) + (token & (BT - 1))) * D) + c16 * 16);
      }
      if (warp == 8) {
        s.there = id >= 0;
        const size_t head = static_cast<size_t>(max(id, 0)) * a.G + walk.g;
        s.ks = id >= 0 ? a.ks[head] : 1.f;
        s.vs = id >= 0 ? a.vs[head] : 1.f;
      }
      const bool fresh_piece = t + 1 == walk.t1;
      if (fresh_piece) have = walk.next(a, before); else ++t;
      if (have) start(fresh_piece);
    };
    auto widen_tile = [&](Coming& s) {
      if (!mbar_wait(&empty[cnt & 1], ((cnt >> 1) & 1) ^ 1, abort_flag, timeout)) return false;
      __syncwarp();
      if (warp == 8) {
        const uint32_t there = __ballot_sync(0xffffffffu, s.there);
        const uint32_t vs = __float_as_uint(s.vs);       // 2^y z, 1 <= z < 2
        if (lane < 8)
          s_scale[cnt & 3][lane] = make_float4(s.ks, static_cast<float>(static_cast<int>(vs >> 23) - 127), __uint_as_float((vs & 0x7fffffu) | 0x3f800000u), 0.f);
        if (lane == 0) s_there[cnt & 3] = there;
        __syncwarp();
        if (lane == 0) mbar_arrive(&meta_full[cnt & 3]);
      }
      if (!INT8 && !keys) {
        uint32_t bad_rows = 0u;
        if (s.lo < CW_TILE) {
#pragma unroll
          for (int p = 0; p < CODE_PASSES; ++p) {
            uint32_t w[4] = {s.x[p].x, s.x[p].y, s.x[p].z, s.x[p].w}, nan[4], any = 0u;
#pragma unroll
            for (int j = 0; j < 4; ++j) { nan[j] = __vcmpeq4(w[j] & 0x7f7f7f7fu, 0x7f7f7f7fu); any |= nan[j]; }
            const bool some = any != 0u && p * PASS_ROWS + row0 >= s.lo;
            if (some) s.x[p] = make_uint4(w[0] & ~nan[0], w[1] & ~nan[1], w[2] & ~nan[2], w[3] & ~nan[3]);
            const uint32_t lanes = __ballot_sync(0xffffffffu, some);
#pragma unroll
            for (int y = 0; y < W::ROWS; ++y) {
              const uint32_t of_row = D == 128 ? (y & 1 ? 0xf0f0u : 0x0f0fu) << (y >> 1) * 16 : 0xfu << 4 * y;
              if (lanes & of_row) bad_rows |= 1u << (p * W::ROWS + y);
            }
          }
        }
        if (lane == 0) s_nan[cnt & 3][w4] = bad_rows;
      }
#pragma unroll
      for (int p = 0; p < CODE_PASSES; ++p) {
        const uint32_t w[4] = {s.x[p].x, s.x[p].y, s.x[p].z, s.x[p].w};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint4 f;
          widen<INT8>(w[2 * h], f.x, f.y);
          widen<INT8>(w[2 * h + 1], f.z, f.w);
          *reinterpret_cast<uint4*>(matrix + (cnt & 1) * W::MATRIX + W::at(p * PASS_ROWS + row0, 2 * c16 + h)) = f;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[cnt & 1]);
      ++cnt;
      return true;
    };
    Coming next;
    for (fetch(next); next.valid; fetch(next))
      if (!widen_tile(next)) { ok = false; break; }
    if (!ok && lane == 0) report_status(a.status, 0x441u);
  } else if (elect_one()) {                // ------------------------------------------------ products
    const uint32_t idesc_s = umma_idesc(0, 0, 0, 128, 128), idesc_o = umma_idesc(0, 0, 1, 128, D);
    const uint64_t q = umma_smem_desc(smem_u32(smem), 16, 1024);
    auto scores = [&](uint32_t x) {        // of the x-th tile
      if (!mbar_wait(&k_full[x & 1], (x >> 1) & 1, abort_flag, timeout)) return false;
      tcgen05_fence_after();
      const uint64_t kd = umma_smem_desc(smem_u32(smem + W::K + (x & 1) * W::MATRIX), 16, 1024);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const uint64_t off = ((i >> 2) * W::CHUNK + (i & 3) * 32) >> 4;
        umma_f16(tmem + (x & 1) * 128, q + off, kd + off, idesc_s, i != 0 ? 1u : 0u);
      }
      umma_commit(&s_full[x & 1]);
      umma_commit(&k_empty[x & 1]);
      return true;
    };
    for (uint32_t piece = 0; ok && walk.next(a, before); ++piece) {
      if (!mbar_wait(q_full, piece & 1, abort_flag, timeout) || !scores(cnt) || (walk.t0 + 1 < walk.t1 && !scores(cnt + 1))) { ok = false; break; }
      for (int t = walk.t0; t < walk.t1; ++t, ++cnt) {
        if (!mbar_wait(&p_full[cnt & 1], (cnt >> 1) & 1, abort_flag, timeout) ||
            !mbar_wait(&v_full[cnt & 1], (cnt >> 1) & 1, abort_flag, timeout)) { ok = false; break; }
        tcgen05_fence_after();
        const uint64_t vd = umma_smem_desc(smem_u32(smem + W::V + (cnt & 1) * W::MATRIX), W::CHUNK, 1024);
#pragma unroll
        for (int i = 0; i < 8; ++i)        // 16 tokens each
          umma_f16_ts(tmem + 256 + (cnt & 1) * 128, tmem + (cnt & 1) * 128 + i * 8, vd + ((i * 2048) >> 4), idesc_o, t > walk.t0 + 1 || i > 0 ? 1u : 0u);
        umma_commit(&v_empty[cnt & 1]);
        umma_commit(&pv_done[cnt & 1]);
        if (t + 2 < walk.t1 && !scores(cnt + 2)) { ok = false; break; }
      }
    }
    if (!ok) report_status(a.status, 0x442u);
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 16) { __syncwarp(); tcgen05_fence_after(); tmem_dealloc(tmem, 512); }
}

// ----------------------------------------------------------------------------- sequences that several blocks share

constexpr int MERGE_WARPS = 8;

// Adds up the partial sums of the sequences that several blocks share, in the order of their tokens, and writes zeros for requests
// without tokens.  A block per eight columns of a sequence (request, KV head, group of columns); its warps share columns and parts.  Latency: 3 to 4 us
// behind the first launch, at 4 MB of partial sums at most.
template <typename T, int D>
__global__ void __launch_bounds__(32 * MERGE_WARPS) attend_merge_kernel(const AttendArgs a, int columns) {
  __shared__ __align__(16) float sums[MERGE_WARPS][D + 4];
  pdl_launch_next();
  pdl_wait();
  const int w = threadIdx.x >> 5, per_tile = a.G * a.groups;
  const int r = blockIdx.x / per_tile, item = blockIdx.x - r * per_tile, g = a.groups == 1 ? item : item / a.groups;
  const int2 ends = a.ends[blockIdx.x];
  const bool any = a.before[r + 1] != a.before[r];
  if (any && ends.x < 0) return;
  const int col0 = (item - g * a.groups) * columns, cols = min(a.S * a.P - col0, columns);
  const int parts = any ? ends.y - ends.x / 2 + 1 : 0;
  // `share` warps per column, each with a run of the parts
  int share = 1;
  while (2 * share * cols <= MERGE_WARPS && 4 * share < parts) share *= 2;
  const int per = (parts + share - 1) / share;
  for (int c0 = blockIdx.y * (MERGE_WARPS / share); c0 < cols; c0 += gridDim.y * (MERGE_WARPS / share)) {
    const int cc = c0 + w / share, mine = w % share, end = min(parts, mine * per + per);
    Partial<D / 32> p;
    const int x0 = mine * per;
    if (cc < cols)
      p.add(end - x0, [](int) { return true; }, [&](int x) {
        return a.part + (static_cast<size_t>(x0 + x == 0 ? ends.x : (ends.x & ~1) + 2 * (x0 + x)) * columns + cc) * (D + 4);
      });
    if (share > 1) {
      __syncthreads();
      p.store(sums[w]);
      __syncthreads();
      if (mine == 0 && cc < cols) {
        p = Partial<D / 32>();
        p.add(share, [](int) { return true; }, [&](int x) { return sums[w + x]; });
      }
    }
    if (mine == 0 && cc < cols) write_row(output_row<T>(a, r, g, col0 + cc, D), p);
  }
}

// Columns of a group.  24 requests of 4,096 tokens, 8 KV heads of 128 values, us with groups of 8, 16, 128 columns: 8 queries 40, 48, -;
// 9 to 16 64, 51, -; 24 90, 84, 124; 48 -, 122, 127; 56 -, 155, 128; 64 240, 156, 129; 128 -, 295, 140; 512 -, 1178, 481.  1,000 tokens, 64
// values, int8: 48 queries -, 36, 39.5; 56 -, 43, 40.
static int attend_columns(int queries) { return queries <= 8 ? 8 : queries <= 48 ? 16 : CW_COLUMNS; }
static long long before_words(int rows) { return (rows + 1 + 3) / 4 * 4; }
static long long ends_words(int rows, int G, int queries) {
  return (2ll * rows * G * ((queries + attend_columns(queries) - 1) / attend_columns(queries)) + 3) / 4 * 4;
}

template <typename T, int D, bool INT8, int NT>
static int launch_attend(const AttendArgs& a, cudaStream_t stream) {
  constexpr size_t ring = CA_WARPS * warp_bytes<D, NT>(), most = ring + (2 * CA_MAX_ROWS + 1) * sizeof(int);
  static bool configured[64] = {false};
  auto kern = attend_kernel<T, D, INT8, NT>;
  int device = 0;
  AXB_CUDA(cudaGetDevice(&device));
  if (!configured[device & 63]) {
    AXB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most)));
    configured[device & 63] = true;
  }
  AXB_CUDA(pdl_launch(kern, dim3(a.workers), dim3(32 * CA_WARPS), ring + (2 * a.R + 1) * sizeof(int), stream, a));
  AXB_CUDA(pdl_launch(attend_merge_kernel<T, D>, dim3(a.R * a.G * a.groups, NT), dim3(32 * MERGE_WARPS), 0, stream, a, 8 * NT));
  return 0;
}
template <typename T, int D, bool INT8>
static int launch_wide(const AttendArgs& a, cudaStream_t stream) {
  constexpr size_t most = Wide<D>::FIXED + (2 * CA_MAX_ROWS + 1) * sizeof(int);
  static bool configured[64] = {false};
  auto kern = attend_wide_kernel<T, D, INT8>;
  int device = 0;
  AXB_CUDA(cudaGetDevice(&device));
  if (!configured[device & 63]) {
    AXB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most)));
    configured[device & 63] = true;
  }
  AXB_CUDA(pdl_launch(kern, dim3(a.workers), dim3(32 * CW_WARPS), Wide<D>::FIXED + (2 * a.R + 1) * sizeof(int), stream, a));
  AXB_CUDA(pdl_launch(attend_merge_kernel<T, D>, dim3(a.R * a.G * a.groups, CW_COLUMNS / 8), dim3(32 * MERGE_WARPS), 0, stream, a, CW_COLUMNS));
  return 0;
}
template <typename T> static int launch_attend(const AttendArgs& a, int D, bool int8, int columns, cudaStream_t stream) {
  if (columns == CW_COLUMNS)
    return D == 64 ? (int8 ? launch_wide<T, 64, true>(a, stream) : launch_wide<T, 64, false>(a, stream))
                   : (int8 ? launch_wide<T, 128, true>(a, stream) : launch_wide<T, 128, false>(a, stream));
  if (columns == 8)
    return D == 64 ? (int8 ? launch_attend<T, 64, true, 1>(a, stream) : launch_attend<T, 64, false, 1>(a, stream))
                   : (int8 ? launch_attend<T, 128, true, 1>(a, stream) : launch_attend<T, 128, false, 1>(a, stream));
  return D == 64 ? (int8 ? launch_attend<T, 64, true, 2>(a, stream) : launch_attend<T, 64, false, 2>(a, stream))
                 : (int8 ? launch_attend<T, 128, true, 2>(a, stream) : launch_attend<T, 128, false, 2>(a, stream));
}

}  // namespace axb

using namespace axb;

// 32-bit words of the workspace: the counts of units, the sequences' ends, two partial results per block
extern "C" long long axb_cached_attention_words(int R, int S, int G, int P, int D) {
  const int columns = attend_columns(S * P), rows = R < CA_MAX_ROWS ? R : CA_MAX_ROWS;
  return before_words(rows) + ends_words(rows, G, S * P) + 2ll * sm_count_current() * columns * (D + 4);
}

extern "C" int axb_cached_attention(const void* q, long long q_row, long long q_token, long long q_group, const void* k, const void* v,
                                    const float* ks, const float* vs, const int* tables, const int* lengths, const int* fresh, void* out,
                                    void* work, int R, int S, int G, int P, int D, int W, int N, int block_tokens, float scale, int dtype,
                                    int int8, void* stream) {
  int shift = 4;
  while (shift < 7 && block_tokens != 1 << shift) ++shift;
  if (block_tokens != 1 << shift) { set_error("cached_attention: blocks hold 16, 32, 64 or 128 tokens, not %d", block_tokens); return -1; }
  if (D != 64 && D != 128) { set_error("cached_attention: heads of 64 or 128 values, not %d", D); return -1; }
  if (dtype != 0 && dtype != 1) { set_error("cached_attention: bf16 or fp16"); return -1; }
  if (R <= 0 || S <= 0 || G <= 0 || P <= 0 || W <= 0 || N <= 0) { set_error("cached_attention: empty sizes"); return -1; }
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(out) |
        reinterpret_cast<uintptr_t>(work)) & 15) || (q_row | q_token | q_group) % 8) {
    set_error("cached_attention: operands must be 16-byte aligned, strides multiples of 8 elements");
    return -1;
  }
  const int columns = attend_columns(S * P), groups = (S * P + columns - 1) / columns, blocks = sm_count_current();
  AttendArgs a{q, q_row, q_token, q_group, out, (const uint8_t*)k, (const uint8_t*)v, ks, vs, tables, lengths, fresh, R, S, G, P, W, N, shift,
               groups, scale * 1.4426950408889634f, blocks, (int*)work, nullptr, nullptr, nullptr, wait_timeout_ns()};
  if (columns == CW_COLUMNS) {
    int device = 0;
    AXB_CUDA(cudaGetDevice(&device));
    if (!device_status_word(device, &a.status)) { set_error("cached_attention: no status word"); return -1; }
  }
  // of the rows of a launch: their units, of very long tables, are counted in 31 bits
  const long long most = (static_cast<long long>(W) << shift < 0x7fffffffll ? static_cast<long long>(W) << shift : 0x7fffffffll) / CA_TILE + 1 + CA_START;
  const int rows = static_cast<int>(0x7fffffffll / most < CA_MAX_ROWS ? 0x7fffffffll / most : CA_MAX_ROWS);
  for (int r0 = 0; r0 < R; r0 += rows) {
    a.R = R - r0 < rows ? R - r0 : rows;
    a.q = static_cast<const char*>(q) + r0 * q_row * 2;
    a.out = static_cast<char*>(out) + static_cast<size_t>(r0) * S * G * P * D * 2;
    a.tables = tables + static_cast<size_t>(r0) * W;
    a.lengths = lengths + r0;
    a.fresh = fresh ? fresh + r0 : nullptr;
    a.ends = reinterpret_cast<int2*>(a.before + before_words(a.R));
    a.part = reinterpret_cast<float*>(a.before + before_words(a.R) + ends_words(a.R, G, S * P));
    const int st = dtype == 0 ? launch_attend<__nv_bfloat16>(a, D, int8 != 0, columns, (cudaStream_t)stream)
                              : launch_attend<__half>(a, D, int8 != 0, columns, (cudaStream_t)stream);
    if (st) return st;
  }
  return 0;
}
