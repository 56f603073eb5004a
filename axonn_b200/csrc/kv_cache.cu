// Bookkeeping and contents of a key/value cache in blocks: where new tokens go, their keys and values in 8 bits, and rows that go on
// from other rows.
//
//   plan      blocks for the new tokens of every request, from a list of free ones, and the slot of every token
//   store     rotary embedding, the largest magnitude of a block and head, codes x 2^-e, scale 2^e; a block that holds tokens already
//             keeps the larger of its scale and the new one, and its codes are rounded again where it grows
//   reorder   rows of a group take over each other's tables; the unfinished block of a row that changes is copied into its spare block
//
// Layout of one layer: codes [blocks, kv_heads, block_tokens, D] (one head of a block is contiguous), scales [blocks, kv_heads].
#include <cuda_fp8.h>

#include "common.cuh"

namespace axb {

// ----------------------------------------------------------------------------- plan

constexpr int PLAN_THREADS = 256;
constexpr int PLAN_TOKENS = 1024;      // tokens that a block of the grid writes, about

struct PlanArgs {
  const int *lengths, *fresh, *free, *taken;
  int* tables;
  long long* slots;
  int *positions, *lengths_out, *taken_out;
  int R, S, W, N, shift, rows, tokens;      // rows and tokens of a row per block of the grid
};

struct PlanRow { long long length, add; int held, need; };

__device__ __forceinline__ PlanRow plan_row(const PlanArgs& a, int r) {
  PlanRow p;
  p.length = max(a.lengths[r], 0);
  p.add = min(max(a.fresh[r], 0), a.S);
  const long long bt1 = (1ll << a.shift) - 1;
  p.held = static_cast<int>(min((p.length + bt1) >> a.shift, static_cast<long long>(a.W)));
  p.need = static_cast<int>(min((p.length + p.add + bt1) >> a.shift, static_cast<long long>(a.W))) - p.held;
  return p;
}

__device__ __forceinline__ int warp_inclusive(int v) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const int u = __shfl_up_sync(0xffffffffu, v, o); if ((threadIdx.x & 31) >= o) v += u; }
  return v;
}

// Every block adds up what the rows before its own need (their lengths stay in the L2), so that one launch does.  Writes 12 bytes per
// token; 256 requests of one token 4.1 us, 96 prompts of up to 2,048 tokens 3.9 us: a launch's latency.
__global__ void __launch_bounds__(PLAN_THREADS) plan_kernel(const PlanArgs a) {
  __shared__ int warp_sum[PLAN_THREADS / 32], before[PLAN_THREADS / 32];
  __shared__ int s_base[PLAN_THREADS], s_held[PLAN_THREADS], s_got[PLAN_THREADS], s_length[PLAN_THREADS], s_add[PLAN_THREADS];
  pdl_launch_next();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int r0 = blockIdx.x * a.rows, n = min(a.rows, a.R - r0);
  int earlier = 0;
  for (int r = tid; r < r0; r += PLAN_THREADS) earlier += plan_row(a, r).need;
  const int earlier_in_warp = warp_inclusive(earlier);
  PlanRow p = {0, 0, 0, 0};
  if (tid < n) p = plan_row(a, r0 + tid);
  const int incl = warp_inclusive(p.need);
  if (lane == 31) { warp_sum[w] = incl; before[w] = earlier_in_warp; }
  __syncthreads();
  const int used = min(max(a.taken[0], 0), a.N);      // whatever stands there, nothing outside the list is read
  long long base = static_cast<long long>(used) + incl - p.need;
  for (int i = 0; i < PLAN_THREADS / 32; ++i) base += before[i] + (i < w ? warp_sum[i] : 0);
  if (tid < n) {
    const int got = static_cast<int>(min(max(a.N - base, 0ll), static_cast<long long>(p.need)));
    const long long room = (static_cast<long long>(p.held + got) << a.shift) - p.length;
    const int add = static_cast<int>(max(0ll, min(p.add, room)));
    s_base[tid] = static_cast<int>(min(base, static_cast<long long>(a.N))); s_held[tid] = p.held; s_got[tid] = got; s_length[tid] = static_cast<int>(p.length); s_add[tid] = add;
    if (blockIdx.y == 0) {
      a.lengths_out[r0 + tid] = static_cast<int>(p.length) + add;
      if (r0 + tid == a.R - 1) a.taken_out[0] = static_cast<int>(min(base + p.need, static_cast<long long>(a.N)));
    }
  }
  __syncthreads();
  if (blockIdx.y == 0)
    for (int i = w; i < n; i += PLAN_THREADS / 32)
      for (int k = lane; k < s_got[i]; k += 32)
        a.tables[static_cast<size_t>(r0 + i) * a.W + s_held[i] + k] = a.free[s_base[i] + k];
  const int t0 = blockIdx.y * a.tokens, per_row = min(a.tokens, a.S - t0);
  for (int x = tid; x < n * per_row; x += PLAN_THREADS) {
    const int i = x / per_row, t = t0 + x % per_row;
    long long slot = -1;
    int at = -1;
    if (t < s_add[i]) {
      at = s_length[i] + t;
      const int k = at >> a.shift;
      const int block = k < s_held[i] ? a.tables[static_cast<size_t>(r0 + i) * a.W + k] : a.free[s_base[i] + k - s_held[i]];
      slot = block < 0 ? -1 : (static_cast<long long>(block) << a.shift) + (at & ((1 << a.shift) - 1));
      if (block < 0) at = -1;
    }
    const size_t o = static_cast<size_t>(r0 + i) * a.S + t;
    a.slots[o] = slot;
    a.positions[o] = at;
  }
}

// ----------------------------------------------------------------------------- store

constexpr int STORE_UNITS = 4;            // units (eight pairs of one token) that a thread holds
constexpr int LOWEST_EXPONENT = -100;     // of a scale: codes x 2^e and x 2^-e stay normal 32-bit numbers

struct StoreArgs {
  const void* qkv;
  long long row_stride, token_stride, group_stride;      // elements
  const long long* slots;
  const int* positions;
  const float* cs;                   // [angles, D / 2, 2] cosine and sine, or null
  void* q;                           // [R, S, G * P, D], with cs
  uint8_t *k, *v;
  float *ks, *vs;
  int R, S, G, P, N, shift, angles;
  int runs;                          // blocks that a row's new tokens touch, at most
  int job_threads;                   // threads that share a job (one head of one block): a warp or the whole block
  unsigned jobs, job_blocks;
};

template <typename T> __device__ __forceinline__ void widen8(const uint4& u, float* f) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 t;
    if constexpr (__is_same(T, __half)) t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    else t = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
    f[2 * i] = t.x; f[2 * i + 1] = t.y;
  }
}
template <typename T> __device__ __forceinline__ void load8(const T* p, float* f) { widen8<T>(*reinterpret_cast<const uint4*>(p), f); }
template <typename T> __device__ __forceinline__ void store8(T* p, const float* f) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (__is_same(T, __half)) { const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]); w[i] = *reinterpret_cast<const uint32_t*>(&h); }
    else { const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]); w[i] = *reinterpret_cast<const uint32_t*>(&h); }
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Eight pairs (f[i], f[8 + i]) turned by their angles.  Every product is rounded by itself, so that the result is the same to the bit
// wherever it is computed: a contracted product would move codes at rounding borders.
__device__ __forceinline__ void rotate8(float* f, const float* cs) {
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    const float4 t = *reinterpret_cast<const float4*>(cs + 4 * h);
    const float co[2] = {t.x, t.z}, si[2] = {t.y, t.w};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float a = f[2 * h + j], b = f[8 + 2 * h + j];
      f[2 * h + j] = __fsub_rn(__fmul_rn(a, co[j]), __fmul_rn(b, si[j]));
      f[8 + 2 * h + j] = __fadd_rn(__fmul_rn(b, co[j]), __fmul_rn(a, si[j]));
    }
  }
}

// The least e with `largest` <= M 2^e, M the largest code (e4m3: 1.75 x 2^8, int8: 1.984375 x 2^6), from the bits.
template <bool INT8> __device__ __forceinline__ int scale_exponent(float largest) {
  const uint32_t b = __float_as_uint(largest);
  const int e = static_cast<int>(b >> 23) - 127 - (INT8 ? 6 : 8) + ((b & 0x7fffffu) > (INT8 ? 0x7e0000u : 0x600000u));
  return max(e, LOWEST_EXPONENT);
}
// Four values times `scale` as codes.  Values past the largest code (infinities) become it; NaN stays NaN in e4m3 and is 0 in int8.
// FINITE: there are none of those; adding 1.5 x 2^23 leaves the rounded number in the low bits, with one rounding of the product.
template <bool INT8, bool FINITE> __device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float scale) {
  if constexpr (INT8 && FINITE) {
    constexpr float magic = 12582912.f;
    const uint32_t lo = __byte_perm(__float_as_uint(__fmaf_rn(a, scale, magic)), __float_as_uint(__fmaf_rn(b, scale, magic)), 0x0040);
    const uint32_t hi = __byte_perm(__float_as_uint(__fmaf_rn(c, scale, magic)), __float_as_uint(__fmaf_rn(d, scale, magic)), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
  }
  a *= scale; b *= scale; c *= scale; d *= scale;
  if constexpr (INT8) {
    const float f[4] = {a, b, c, d};
    uint32_t o = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int v = f[i] == f[i] ? __float2int_rn(fminf(fmaxf(f[i], -127.f), 127.f)) : 0;
      o |= (static_cast<uint32_t>(v) & 0xffu) << (8 * i);
    }
    return o;
  } else {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  }
}
// |a| and |b|, the larger one; NaN if one is
__device__ __forceinline__ float largest_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(fabsf(b)));
  return m;
}
template <typename T> __device__ __forceinline__ uint32_t largest_nan_16(uint32_t a, uint32_t b) {
  b &= 0x7fff7fffu;
  if constexpr (__is_same(T, __half)) { const __half2 m = __hmax2_nan(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b)); return *reinterpret_cast<const uint32_t*>(&m); }
  else { const __nv_bfloat162 m = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b)); return *reinterpret_cast<const uint32_t*>(&m); }
}
template <bool INT8> __device__ __forceinline__ float code_value(uint32_t byte) {
  if constexpr (INT8) return static_cast<float>(static_cast<int8_t>(byte));
  else return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
}

// Bound by reading the projection once and writing a byte per value: a thread keeps its values in registers between the search for the
// largest and the codes (as they came in where nothing is rotated: more blocks fit an SM, and more loads are on their way).  A job is one
// head of one block, keys or values: a warp where few tokens arrive (a decoding step), a block of threads with up to 64 values each where
// whole blocks are filled.  Nothing is waited for before the loads but the row's first slot; a token's own slot and position are looked at
// when its values are there.  The queries' rotation is further blocks of the same launch.
//
// 16 prompts of up to 2,048 tokens, 16 KV heads of 128 values, bf16 to int8 (309 MB): 59.1 us, 5.2 TB/s, 0.8 of a copy's rate; it issues in
// two thirds of the cycles with half of the warps that fit an SM, four blocks of 256 by their 64 registers.  Two units per thread 69.6 us
// (more of it is bookkeeping), three blocks 65.0, five or 56 registers 77, 63 (spills); slots by one lane per token 60.4.  A token each for
// 128 requests, 8 KV heads of 4 query heads, rotated: 3.9 us, latency.  16 prompts of up to 2,048 tokens of those, rotated, e4m3 (629 MB):
// 232 us, 2.7 TB/s, 0.41 of a copy's rate: values are held as 32-bit numbers, 114 registers leave two blocks of 256 per SM (0.22 of the
// warps), and it issues in 0.31 of the cycles, waiting for its loads.
template <typename T, int D, bool INT8, bool ROPE>
__global__ void __launch_bounds__(256, ROPE ? 2 : 4) store_kernel(const StoreArgs a) {
  constexpr int UNITS = D / 16;            // units of a token: eight pairs (i, i + D / 2) each
  __shared__ float part[8];
  pdl_launch_next();
  pdl_wait();
  const T* qkv = static_cast<const T*>(a.qkv);
  if (ROPE && blockIdx.x >= a.job_blocks) {        // queries
    const long long unit = (blockIdx.x - a.job_blocks) * static_cast<long long>(blockDim.x) + threadIdx.x;
    const int c = static_cast<int>(unit % UNITS) * 8, H = a.G * a.P;
    if (unit / UNITS >= static_cast<long long>(a.R) * a.S * H) return;
    const unsigned row = static_cast<unsigned>(unit / UNITS), token = row / H;      // 31 bits: the host sees to that
    const int h = static_cast<int>(row - token * H);
    float f[16];
    const int at = a.positions[token];
    const long long slot = a.slots[token];
    if (slot >= 0 && (slot >> a.shift) < a.N && at >= 0 && at < a.angles) {
      const unsigned r = token / a.S, g = h / a.P;
      const T* p = qkv + r * a.row_stride + (token - r * a.S) * a.token_stride + g * a.group_stride + (h - g * a.P) * D + c;
      load8(p, f);
      load8(p + D / 2, f + 8);
      rotate8(f, a.cs + (static_cast<size_t>(at) * (D / 2) + c) * 2);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) f[i] = 0.f;
    }
    T* o = static_cast<T*>(a.q) + static_cast<size_t>(row) * D + c;
    store8(o, f);
    store8(o + D / 2, f + 8);
    return;
  }
  const int threads = a.job_threads, tid = threads == 32 ? threadIdx.x & 31 : threadIdx.x;
  const unsigned job = threads == 32 ? blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5) : blockIdx.x;
  if (job >= a.jobs) return;               // whole warps: jobs of more than a warp are whole blocks
  // values next to keys, then heads, so that the rows that neighbouring blocks read lie together
  const bool values = job & 1;
  const unsigned rest = job >> 1, block = rest / a.G;
  const int g = static_cast<int>(rest - block * a.G), r = static_cast<int>(block / a.runs), run = static_cast<int>(block - r * a.runs);
  const int BT = 1 << a.shift;
  const long long* slots = a.slots + static_cast<size_t>(r) * a.S;
  const long long slot0 = slots[0];
  int within = static_cast<int>(slot0 & (BT - 1));
  if (slot0 < 0) {                         // none of the row's, or none in the block that its table lacks: later ones start a block
    unsigned some = 0u;
    int at = 1;
    for (; at < BT && at < a.S; at += 32) {
      some = __ballot_sync(0xffffffffu, at + (tid & 31) < a.S && slots[at + (tid & 31)] >= 0);
      if (some) break;
    }
    if (!some || run == 0) return;
    within = BT - (at + __ffs(some) - 1);
    if (within <= 0) return;
  }
  const int i0 = run == 0 ? 0 : run * BT - within, held = run == 0 ? within : 0;
  if (i0 >= a.S) return;
  const int n = min(BT - held, a.S - i0);
  const long long first = slots[i0];
  const T* x = qkv + r * a.row_stride + static_cast<long long>(i0) * a.token_stride + g * a.group_stride + (a.P + (values ? 1 : 0)) * D;
  uint4 raw[STORE_UNITS][2];
  long long slot[STORE_UNITS];
  int position[STORE_UNITS];
#pragma unroll
  for (int u = 0; u < STORE_UNITS; ++u) {
    const int unit = tid + u * threads, i = unit / UNITS, c = (unit % UNITS) * 8;
    slot[u] = -1;
    if (i >= n) continue;
    const T* p = x + static_cast<long long>(i) * a.token_stride + c;
    raw[u][0] = *reinterpret_cast<const uint4*>(p);
    raw[u][1] = *reinterpret_cast<const uint4*>(p + D / 2);
    slot[u] = slots[i0 + i];
    if (ROPE) position[u] = a.positions[static_cast<size_t>(r) * a.S + i0 + i];
  }
  if (first < 0 || (first >> a.shift) >= a.N || (first & (BT - 1)) != held) return;
  const size_t head = static_cast<size_t>(first >> a.shift) * a.G + g;
  uint8_t* codes = (values ? a.v : a.k) + head * BT * D;
  float* scale_at = (values ? a.vs : a.ks) + head;
  const float old = held ? *scale_at : 0.f;
  float f[ROPE ? STORE_UNITS : 1][16], largest = 0.f;
  uint32_t mine = 0, pairs = 0u;
#pragma unroll
  for (int u = 0; u < STORE_UNITS; ++u) {
    const int unit = tid + u * threads, i = unit / UNITS, c = (unit % UNITS) * 8;
    if (i >= n || slot[u] != first + i || (ROPE && (position[u] < 0 || position[u] >= a.angles))) continue;
    mine |= 1u << u;
    if (!ROPE) {
#pragma unroll
      for (int half = 0; half < 2; ++half)
        pairs = largest_nan_16<T>(largest_nan_16<T>(largest_nan_16<T>(largest_nan_16<T>(pairs, raw[u][half].x), raw[u][half].y), raw[u][half].z), raw[u][half].w);
      continue;
    }
    float* y = f[u];
    widen8<T>(raw[u][0], y);
    widen8<T>(raw[u][1], y + 8);
    if (!values) rotate8(y, a.cs + (static_cast<size_t>(position[u]) * (D / 2) + c) * 2);
#pragma unroll
    for (int j = 0; j < 16; ++j) largest = largest_nan(largest, y[j]);
  }
  if (!ROPE) {
    float y[8];
    widen8<T>(make_uint4(pairs, 0u, 0u, 0u), y);
    largest = largest_nan(y[0], y[1]);
  }
  const bool finite = largest <= 3.4028234663852886e38f;
  if (!finite) {                           // the largest of what is finite
    largest = 0.f;
#pragma unroll
    for (int u = 0; u < STORE_UNITS; ++u) {
      if (!(mine >> u & 1)) continue;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float* y = f[ROPE ? u : 0] + 8 * half;
        if (!ROPE) widen8<T>(raw[u][half], y);
#pragma unroll
        for (int j = 0; j < 8; ++j) { const float m = fabsf(y[j]); if (m <= 3.4028234663852886e38f) largest = fmaxf(largest, m); }
      }
    }
  }
  bool some = __any_sync(0xffffffffu, mine != 0);
  largest = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(largest)));      // not negative: the order of the bits
  if (threads > 32) {
    if ((tid & 31) == 0) part[tid >> 5] = some ? largest : -1.f;
    __syncthreads();
    largest = -1.f;
    for (int i = 0; i < threads / 32; ++i) largest = fmaxf(largest, part[i]);
    some = largest >= 0.f;
  }
  if (!some) return;                       // every token of the run was left out
  const float grown = __uint_as_float(static_cast<uint32_t>(scale_exponent<INT8>(largest) + 127) << 23);
  const float scale = fmaxf(grown, old);
  if (held && old < scale) {               // the tokens that are there already, at the new scale
    const float shrink = old * __frcp_rn(scale);
    for (int i = tid; i < held * (D / 16); i += threads) {
      uint4* at = reinterpret_cast<uint4*>(codes) + i;
      const uint4 u = *at;
      uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = codes4<INT8, false>(code_value<INT8>(w[j] & 0xff), code_value<INT8>((w[j] >> 8) & 0xff), code_value<INT8>((w[j] >> 16) & 0xff),
                                   code_value<INT8>(w[j] >> 24), shrink);
      *at = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  const float inverse = __frcp_rn(scale);
#pragma unroll
  for (int u = 0; u < STORE_UNITS; ++u) {
    if (!(mine >> u & 1)) continue;
    const int unit = tid + u * threads, i = unit / UNITS, c = (unit % UNITS) * 8;
    uint8_t* p = codes + static_cast<size_t>(held + i) * D + c;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float* s = f[ROPE ? u : 0] + 8 * half;
      if (!ROPE) widen8<T>(raw[u][half], s);
      *reinterpret_cast<uint2*>(p + half * (D / 2)) =
          finite ? make_uint2(codes4<INT8, true>(s[0], s[1], s[2], s[3], inverse), codes4<INT8, true>(s[4], s[5], s[6], s[7], inverse))
                 : make_uint2(codes4<INT8, false>(s[0], s[1], s[2], s[3], inverse), codes4<INT8, false>(s[4], s[5], s[6], s[7], inverse));
    }
  }
  if (threads > 32) __syncthreads(); else __syncwarp();      // everyone has read the old scale
  if (tid == 0) *scale_at = scale;
}

// ----------------------------------------------------------------------------- reorder

constexpr int REORDER_THREADS = 128;
constexpr int REORDER_BLOCKS = 32;       // blocks of the grid per SM, before a block takes several heads

struct ReorderArgs {
  uint8_t *k, *v;                    // [layers, N, G, BT, D]
  float *ks, *vs;
  const int *tables, *lengths, *spare, *parents;
  int *tables_out, *lengths_out, *spare_out;
  int R, K, W, N, G, shift, row_bytes, heads;      // row_bytes: of a token and head; heads: per block of the grid
};

// Bound by reading and writing the unfinished blocks of the rows that change, of all layers.  Sources are blocks that rows write into,
// targets are spare ones, so that nothing is read after it was written and the order of the copies does not matter.  Unfinished blocks
// hold 1 to block_tokens - 1 tokens: small blocks of the grid, many to an SM, even that out.  64 rows, 32 layers, 8 heads of 128 values,
// blocks of 64 tokens (201 MB): 32.6 us, 6.2 TB/s (35.5 with a division for every 16 bytes, and then 46.2, 37.6, 37.0 at 8, 16 or 64
// blocks per SM, 39.1 and 38.1 with 256 threads and 8 or 32 blocks, 36.7 with eight loads ahead instead of four).  4 rows, 24 layers, 16
// heads: 3.6 us, a launch's latency.
__global__ void __launch_bounds__(REORDER_THREADS) reorder_kernel(const ReorderArgs a) {
  pdl_launch_next();
  pdl_wait();
  const int r = blockIdx.x, group = r / a.K * a.K, tid = threadIdx.x;
  int parent = a.parents[r];
  parent = group + (parent >= 0 && parent < a.K ? parent : r - group);
  const int length = a.lengths[parent], part = length & ((1 << a.shift) - 1), full = length >> a.shift;
  const bool moved = parent != r && length > 0 && part > 0 && full < a.W;
  if (blockIdx.y == 0 && blockIdx.z == 0) {
    for (int c = tid; c < a.W; c += REORDER_THREADS)
      a.tables_out[static_cast<size_t>(r) * a.W + c] = moved && c == full ? a.spare[r] : a.tables[static_cast<size_t>(parent) * a.W + c];
    if (tid == 0) {
      a.lengths_out[r] = length;
      a.spare_out[r] = moved ? a.tables[static_cast<size_t>(r) * a.W + full] : a.spare[r];
    }
  }
  if (!moved) return;
  const int from = a.tables[static_cast<size_t>(parent) * a.W + full], to = a.spare[r];
  if (from < 0 || from >= a.N || to < 0 || to >= a.N) return;
  const size_t layer = static_cast<size_t>(blockIdx.y) * a.N;
  const int g0 = blockIdx.z * a.heads, heads = min(a.heads, a.G - g0);
  const size_t source = (layer + from) * a.G + g0, target = (layer + to) * a.G + g0;
  if (tid < heads) a.ks[target + tid] = a.ks[source + tid];
  else if (tid >= 32 && tid < 32 + heads) a.vs[target + tid - 32] = a.vs[source + tid - 32];
  const int per_head = part * a.row_bytes / 16, total = 2 * heads * per_head;
  const size_t head_bytes = static_cast<size_t>(a.row_bytes) << a.shift;
  // word `at` of head h, keys then values; REORDER_THREADS words further: heads and words to go, without a division
  const int step_heads = REORDER_THREADS / per_head, step = REORDER_THREADS - step_heads * per_head;
  int h = tid / per_head, at = tid - h * per_head;
  for (int i0 = tid; i0 < total; i0 += 4 * REORDER_THREADS) {
    uint4 u[4];
    size_t to[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const size_t word = (h < heads ? h : h - heads) * head_bytes + at * static_cast<size_t>(16);
      to[j] = word;
      if (i0 + j * REORDER_THREADS < total) u[j] = *reinterpret_cast<const uint4*>((h < heads ? a.k : a.v) + source * head_bytes + word);
      h += step_heads; at += step;
      if (at >= per_head) { at -= per_head; ++h; }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i0 + j * REORDER_THREADS < total) *reinterpret_cast<uint4*>((i0 + j * REORDER_THREADS < total / 2 ? a.k : a.v) + target * head_bytes + to[j]) = u[j];
  }
}

template <typename T, int D> static void (*store_variant(bool int8, bool rope))(StoreArgs) {
  return int8 ? (rope ? store_kernel<T, D, true, true> : store_kernel<T, D, true, false>)
              : (rope ? store_kernel<T, D, false, true> : store_kernel<T, D, false, false>);
}
template <typename T> static void (*store_variant(int D, bool int8, bool rope))(StoreArgs) {
  return D == 64 ? store_variant<T, 64>(int8, rope) : store_variant<T, 128>(int8, rope);
}

// log2 of the tokens of a block, or -1
static int block_shift(int block_tokens) {
  for (int s = 4; s <= 7; ++s) if (block_tokens == 1 << s) return s;
  set_error("block cache: blocks hold 16, 32, 64 or 128 tokens, not %d", block_tokens);
  return -1;
}

}  // namespace axb

using namespace axb;

extern "C" int axb_plan_blocks(const int* lengths, const int* fresh, int* tables, const int* free_blocks, const int* taken, long long* slots,
                               int* positions, int* lengths_out, int* taken_out, int R, int S, int W, int N, int block_tokens, void* stream) {
  const int shift = block_shift(block_tokens);
  if (shift < 0) return -1;
  if (R <= 0 || S <= 0 || W <= 0 || N <= 0) { set_error("plan_blocks: empty sizes"); return -1; }
  if (static_cast<long long>(W) << shift > 0x7fffffffll) { set_error("plan_blocks: tables of more than 2^31 - 1 tokens"); return -1; }
  const int tokens = S < PLAN_TOKENS ? S : PLAN_TOKENS;
  int rows = PLAN_TOKENS / tokens;
  if (rows > PLAN_THREADS) rows = PLAN_THREADS;
  const int chunks = (S + tokens - 1) / tokens;
  if (chunks > 65535) { set_error("plan_blocks: more than %d tokens per row", 65535 * PLAN_TOKENS); return -1; }
  const PlanArgs a{lengths, fresh, free_blocks, taken, tables, slots, positions, lengths_out, taken_out, R, S, W, N, shift, rows, tokens};
  AXB_CUDA(pdl_launch(plan_kernel, dim3((R + rows - 1) / rows, chunks), dim3(PLAN_THREADS), 0, (cudaStream_t)stream, a));
  return 0;
}

extern "C" int axb_store_blocks(const void* qkv, long long row_stride, long long token_stride, long long group_stride, const long long* slots,
                                const int* positions, const float* cs, void* q, void* k, void* v, float* ks, float* vs, int R, int S, int G,
                                int P, int D, int N, int block_tokens, int angles, int dtype, int int8, void* stream) {
  const int shift = block_shift(block_tokens);
  if (shift < 0) return -1;
  if (D != 64 && D != 128) { set_error("store_blocks: heads of 64 or 128 values, not %d", D); return -1; }
  if (dtype != 0 && dtype != 1) { set_error("store_blocks: bf16 or fp16"); return -1; }
  if (R <= 0 || S <= 0 || G <= 0 || P < 0 || N <= 0) { set_error("store_blocks: empty sizes"); return -1; }
  if (((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
        reinterpret_cast<uintptr_t>(cs)) & 15) || (row_stride | token_stride | group_stride) % 8) {
    set_error("store_blocks: operands must be 16-byte aligned, strides multiples of 8 elements");
    return -1;
  }
  StoreArgs a{qkv, row_stride, token_stride, group_stride, slots, positions, cs, q, (uint8_t*)k, (uint8_t*)v, ks, vs, R, S, G, P, N, shift,
              angles};
  a.runs = (S + block_tokens - 2) / block_tokens + 1;
  // a warp holds 32 x STORE_UNITS units: a job of that size or less needs no more
  const int units = (S < block_tokens ? S : block_tokens) * (D / 16);
  a.job_threads = units <= 32 * STORE_UNITS ? 32 : block_tokens * (D / 16) / STORE_UNITS;
  const int threads = a.job_threads == 32 ? 128 : a.job_threads, per_block = threads / a.job_threads;
  const long long jobs = 2ll * R * a.runs * G, job_blocks = (jobs + per_block - 1) / per_block;
  const long long q_rows = cs ? static_cast<long long>(R) * S * G * P : 0, grid = job_blocks + (q_rows * (D / 16) + threads - 1) / threads;
  a.jobs = static_cast<unsigned>(jobs);
  a.job_blocks = static_cast<unsigned>(job_blocks);
  if (grid > 0x7fffffffll || jobs > 0x7fffffffll || q_rows > 0x7fffffffll) { set_error("store_blocks: too many tokens in one call"); return -1; }
  void (*kern)(StoreArgs) = dtype == 0 ? store_variant<__nv_bfloat16>(D, int8 != 0, cs != nullptr) : store_variant<__half>(D, int8 != 0, cs != nullptr);
  AXB_CUDA(pdl_launch(kern, dim3((unsigned)grid), dim3(threads), 0, (cudaStream_t)stream, a));
  return 0;
}

extern "C" int axb_reorder_blocks(void* k, void* v, float* ks, float* vs, const int* tables, const int* lengths, const int* spare,
                                  const int* parents, int* tables_out, int* lengths_out, int* spare_out, int layers, int R, int K, int W,
                                  int N, int G, int block_tokens, int row_bytes, void* stream) {
  const int shift = block_shift(block_tokens);
  if (shift < 0) return -1;
  if (layers <= 0 || R <= 0 || K <= 0 || R % K || W <= 0 || N <= 0 || G <= 0) { set_error("reorder_blocks: empty sizes"); return -1; }
  if (row_bytes % 16 || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15)) {
    set_error("reorder_blocks: operands must be 16-byte aligned, heads of a multiple of 16 values");
    return -1;
  }
  if (layers > 65535) { set_error("reorder_blocks: more than 65535 layers"); return -1; }
  int heads = G < 32 ? G : 32;
  while (heads > 1 && static_cast<long long>(R) * layers * ((G + heads - 1) / heads) < static_cast<long long>(REORDER_BLOCKS) * sm_count_current()) heads = (heads + 1) / 2;
  const ReorderArgs a{(uint8_t*)k, (uint8_t*)v, ks, vs, tables, lengths, spare, parents, tables_out, lengths_out, spare_out,
                      R, K, W, N, G, shift, row_bytes, heads};
  AXB_CUDA(pdl_launch(reorder_kernel, dim3(R, layers, (G + heads - 1) / heads), dim3(REORDER_THREADS), 0, (cudaStream_t)stream, a));
  return 0;
}
