// Low-rank adapters of many requests at once beside a shared projection (LoRA-style fine-tuning and serving of ONE decoder
// for many species / cultivars; the projection is one Linear of deepsdf/networks/deep_sdf_decoder.py:29-62):
//
//   y[m]  = x[m] W^T + b + t[m] B_a^T            t[m] = s_a drop(x[m]) A_a^T      a = adapter of the request that row m is in
//   dx[m] = dy[m] W + drop'(u[m] A_a)            u[m] = s_a dy[m] B_a
//   dA_a  = sum_m u[m]^T drop(x[m])              dB_a = sum_m dy[m]^T t[m]        (the projection is frozen)
//
// x (M, K), W (N, K), A (adapters, r, K), B (adapters, N, r).  Request q has the rows row_start[q] .. row_start[q + 1] - 1 and
// the adapter adapter[q]; a value outside 0 .. adapters - 1, or no request at all, leaves the bare projection.
//
// Arithmetic: every sum is held in 32 bits.  t and u stay in 32 bits in memory; where they meet 16-bit operands on the matrix
// cores they are split into a high and a low bf16 part (off by 2^-17 of themselves; fp32's range, so nothing overflows or goes
// under), and an fp16 operand there into two bf16 parts, which is exact (11 = 8 + 3 bits).  A value kept by the dropout is NOT
// multiplied by 1 / (1 - p) before the product (that would round it): the factor joins s_a.
//
// A row's result depends on its own row and its own adapter alone: a lane of a matrix product holds one row (rows are the
// columns of the MFMA), and what another request's adapter adds is selected away, not multiplied by 0 -- an infinity or NaN in
// one request or one adapter does not reach another request.  Sums over rows (dA, dB) run in a fixed order: no atomics.
#include "hm_internal.h"
#include "hm_keep.h"
#include "../../include/hortimapping_amd.h"
#include "../../include/hortimapping_amd_debug.h"

using namespace hm;

namespace {

typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct Segs {
  const int* row_start;   // [S + 1]
  const int* adapter;     // [S]
  const float* scale;     // [adapters] or nullptr
  int S, n_adapters, M;
};

// last request that starts at or before `row` (-1: none), found by the whole wave: 64 probes a step.  Whatever row_start
// holds, the result is in -1 .. S - 1.
__device__ __forceinline__ int seg_find(const Segs& sg, int row) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = sg.S;
  while (n > 0) {
    const int step = (n + 63) >> 6, at = lo + lane * step;
    const bool le = lane * step < n && sg.row_start[at] <= row;
    const int c = __popcll(__ballot(le));
    if (c == 0) return lo - 1;
    lo += (c - 1) * step;
    if (step == 1) return lo;
    const int left = n - (c - 1) * step;
    n = left < step ? left : step;
  }
  return -1;
}

// the rows of request q inside [r0, r1), and its adapter (-1: none of them)
struct Span { int lo, hi, a; };
__device__ __forceinline__ Span seg_span(const Segs& sg, int q, int r0, int r1) {
  const int s0 = sg.row_start[q], s1 = sg.row_start[q + 1], a = sg.adapter[q];
  Span s = {s0 > r0 ? s0 : r0, s1 < r1 ? s1 : r1, a};
  if (a < 0 || a >= sg.n_adapters || s.lo >= s.hi) s.a = -1;
  return s;
}

// ---- fragments of eight consecutive values along the reduction, and 16 x 16 products over 32 of it
template <typename T> struct Frag8;
template <> struct Frag8<float> { float v[8]; };
template <> struct Frag8<f16> { f16x8 v; };
template <> struct Frag8<bf16> { bf16x8 v; };

__device__ __forceinline__ f32x4 mma16(const Frag8<f16>& a, const Frag8<f16>& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v, b.v, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(const Frag8<bf16>& a, const Frag8<bf16>& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(const Frag8<float>& a, const Frag8<float>& b, f32x4 c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b.v[j], c, 0, 0, 0);
  return c;
}

// keeps the scheduler from spreading a group of loads between the products that wait for them, which it does to save registers:
// these kernels live from the loads in flight
__device__ __forceinline__ void all_loads_first() { __builtin_amdgcn_sched_barrier(0); }

// what a lane of this wave wrote to the LDS is there for its other lanes: LDS accesses of a wave keep their order, so only the
// compiler has to be held
__device__ __forceinline__ void wave_sees_lds() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// p[0 .. 7], of which the first n exist (n <= 0: none): zero where nothing is
template <typename T> __device__ __forceinline__ Frag8<T> frag_load(const T* p, int n) {
  Frag8<T> f;
  if (n >= 8) {
    const Pack8<T> u = *reinterpret_cast<const Pack8<T>*>(p);
#pragma unroll
    for (int j = 0; j < 8; ++j) f.v[j] = u.v[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f.v[j] = j < n ? p[j] : (T)0.f;
  }
  return f;
}
template <typename T> __device__ __forceinline__ Frag8<T> frag_load(const T* p) {
  Frag8<T> f;
  const Pack8<T> u = *reinterpret_cast<const Pack8<T>*>(p);
#pragma unroll
  for (int j = 0; j < 8; ++j) f.v[j] = u.v[j];
  return f;
}
template <typename T> __device__ __forceinline__ void frag_keep(Frag8<T>& f, uint32_t keep) {
#pragma unroll
  for (int j = 0; j < 8; ++j) f.v[j] = (keep >> j) & 1 ? f.v[j] : (T)0.f;
}

// ---- lines of 128 bytes along the reduction: what a row of an LDS tile holds
template <typename T> struct Lines { static constexpr int V = 16 / sizeof(T), KB = 128 / sizeof(T); };
template <typename T> struct alignas(16) Line { T v[16 / sizeof(T)]; };
template <typename T> struct alignas(sizeof(T)) LooseLine { T v[16 / sizeof(T)]; };     // the same at the alignment of one value

template <typename T> __device__ __forceinline__ uint4 line_load(const T* p) {
  return __builtin_bit_cast(uint4, *reinterpret_cast<const LooseLine<T>*>(p));
}
// the first n values of a line (n <= 0: none), zero behind them
template <typename T> __device__ __forceinline__ uint4 line_load(const T* p, int n) {
  constexpr int V = Lines<T>::V;
  if (n >= V) return line_load(p);
  Line<T> o;
#pragma unroll
  for (int j = 0; j < V; ++j) o.v[j] = j < n ? p[j] : (T)0.f;
  return __builtin_bit_cast(uint4, o);
}

// ---- thin products: a wave's share of A (up to 64 rows) times B^T (up to 64 rows), lines w, w + NW, .. of the reduction.  Every
// wave stages its own lines in its own part of the LDS -- global memory sees whole lines (64-byte pieces of rows that lie a power
// of two apart come from few channels and take four times as long), no wave waits for another -- and has the next line's loads
// in flight while it multiplies.
template <int AT, int BT> constexpr int strip_units() { return (AT + BT) * 128; }       // 16-byte units of LDS a wave

template <typename T, int AT, int BT, int NW, bool DROP>
__device__ __forceinline__ void strip_sum(f32x4 (&acc)[BT][AT], const T* A, long long lda, int na, const T* B, long long ldb, int nb, int K,
                                          uint4* own, int w, int lane, const KeepArgs& ka, KeepKey key, int row0) {
  constexpr int V = Lines<T>::V, KB = Lines<T>::KB;
  const int l16 = lane & 15, g = lane >> 4, c = lane & 7, r8 = lane >> 3;
  const char *ba = reinterpret_cast<const char*>(A), *bb = reinterpret_cast<const char*>(B);
  // rows past the end are read as the last one: a row of A or B touches its own results alone
  uint32_t oa[2 * AT], ob[2 * BT];
#pragma unroll
  for (int i = 0; i < 2 * AT; ++i) { const int r = 8 * i + r8; oa[i] = ((uint32_t)(r < na ? r : na - 1) * (uint32_t)lda + c * V) * sizeof(T); }
#pragma unroll
  for (int i = 0; i < 2 * BT; ++i) { const int r = 8 * i + r8; ob[i] = ((uint32_t)(r < nb ? r : nb - 1) * (uint32_t)ldb + c * V) * sizeof(T); }
  const int full = K / KB, lines = (K + KB - 1) / KB;
  uint4 ga[2 * AT], gb[2 * BT];
  auto fetch = [&](int s) {
    const size_t k = (size_t)s * 128;
    if (s < full) {
#pragma unroll
      for (int i = 0; i < 2 * BT; ++i) gb[i] = line_load(reinterpret_cast<const T*>(bb + k + ob[i]));
#pragma unroll
      for (int i = 0; i < 2 * AT; ++i) ga[i] = line_load(reinterpret_cast<const T*>(ba + k + oa[i]));
    } else {
      const int n = K - s * KB - c * V;
#pragma unroll
      for (int i = 0; i < 2 * BT; ++i) gb[i] = line_load(reinterpret_cast<const T*>(bb + k + ob[i]), n);
#pragma unroll
      for (int i = 0; i < 2 * AT; ++i) ga[i] = line_load(reinterpret_cast<const T*>(ba + k + oa[i]), n);
    }
  };
  auto frag = [&](int row, int kk) {
    Frag8<T> f;
    if constexpr (sizeof(T) == 2) {
      f.v = __builtin_bit_cast(decltype(f.v), own[row * 8 + ((4 * kk + g) ^ (row & 7))]);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4 v = __builtin_bit_cast(f32x4, own[row * 8 + ((2 * g + h) ^ (row & 7))]);
#pragma unroll
        for (int j = 0; j < 4; ++j) f.v[4 * h + j] = v[j];
      }
    }
    return f;
  };
  if (w < lines) fetch(w);
  for (int s = w; s < lines; s += NW) {
#pragma unroll
    for (int i = 0; i < 2 * AT; ++i) { const int r = 8 * i + r8; own[r * 8 + (c ^ (r & 7))] = ga[i]; }
#pragma unroll
    for (int i = 0; i < 2 * BT; ++i) { const int r = 16 * AT + 8 * i + r8; own[r * 8 + (c ^ (r & 7))] = gb[i]; }
    if (s + NW < lines) fetch(s + NW);
    wave_sees_lds();
#pragma unroll
    for (int kk = 0; kk < KB / 32; ++kk) {
      Frag8<T> a[AT];
#pragma unroll
      for (int i = 0; i < AT; ++i) a[i] = frag(16 * i + l16, kk);
#pragma unroll
      for (int m = 0; m < BT; ++m) {
        Frag8<T> x = frag(16 * AT + 16 * m + l16, kk);
        if (DROP) frag_keep(x, keep8(ka, key, (uint64_t)(row0 + 16 * m + l16), (uint32_t)((s * KB + 32 * kk + 8 * g) >> 3)));
#pragma unroll
        for (int i = 0; i < AT; ++i) acc[m][i] = mma16(a[i], x, acc[m][i]);
      }
    }
    wave_sees_lds();
  }
}

// ---- t / u: 32 rows x up to 64 ranks a workgroup, its waves share the reduction.  Bound by reading X once: 131072 x 512 bf16 in
// 25 us (5.3 TB/s), 65536 x 512 fp32 in 27 (5.0 TB/s); rows of 259 values, which start between lines, 34 us.
constexpr int SH_ROWS = 32, SH_RANKS = 64;

template <typename T, int RT, int NW, bool DROP>
__global__ __launch_bounds__(64 * NW) void k_shrink(const T* __restrict__ X, long long ldx, int K, const T* __restrict__ R, long long ldr,
                                                    long long stride_a, int rank, float factor, Segs sg, KeepArgs ka,
                                                    float* __restrict__ t, int ldt) {
  constexpr int U = strip_units<RT, 2>();
  __shared__ uint4 lds[NW * U];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, l16 = lane & 15, g = lane >> 4;
  const int r0 = blockIdx.x * SH_ROWS, ib = blockIdx.y * SH_RANKS;
  const int r1 = r0 + SH_ROWS < sg.M ? r0 + SH_ROWS : sg.M;
  const KeepKey key = keep_key(ka);
  int q = seg_find(sg, r0);
  for (q = q < 0 ? 0 : q; q < sg.S && sg.row_start[q] < r1; ++q) {
    const Span sp = seg_span(sg, q, r0, r1);
    if (sp.a < 0) continue;
    f32x4 acc[2][RT];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int i = 0; i < RT; ++i) acc[m][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    strip_sum<T, RT, 2, NW, DROP>(acc, R + (long long)sp.a * stride_a + ib * ldr, ldr, rank - ib, X + (long long)r0 * ldx, ldx, sg.M - r0, K,
                                  lds + w * U, w, lane, ka, key, r0);
    f32x4* red = reinterpret_cast<f32x4*>(lds);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int i = 0; i < RT; ++i) red[w * U + (m * RT + i) * 64 + lane] = acc[m][i];
    __syncthreads();
    const float f = factor * (sg.scale != nullptr ? sg.scale[sp.a] : 1.f);
    for (int u = w; u < 2 * RT; u += NW) {
      f32x4 v = red[u * 64 + lane];
#pragma unroll
      for (int o = 1; o < NW; ++o) v += red[o * U + u * 64 + lane];
      const int row = r0 + 16 * (u / RT) + l16, i0 = ib + 16 * (u % RT) + 4 * g;
      if (row >= sp.lo && row < sp.hi && i0 < ldt) {   // ldt is a multiple of 8: four at once
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = i0 + j < rank ? v[j] * f : 0.f;
        *reinterpret_cast<f32x4*>(t + (long long)row * ldt + i0) = v;
      }
    }
    __syncthreads();
  }
}

// A launch takes fewer than 2^32 threads along one dimension of its grid: what may come to more is laid out over y too.
constexpr long long GRID_X = 1 << 22;
inline dim3 grid_of(long long blocks) {
  const long long x = blocks < GRID_X ? blocks : GRID_X;
  return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}
// number of this workgroup in such a grid; the last ones lie past the blocks asked for
__device__ __forceinline__ long long block_of_grid() { return (long long)blockIdx.y * gridDim.x + blockIdx.x; }

// t / u for requests of few rows (single tokens): a wave takes one row and four ranks, its lanes the reduction
constexpr int SR_RANKS = 4;

template <typename T, bool DROP>
__global__ __launch_bounds__(256) void k_shrink_rows(const T* __restrict__ X, long long ldx, int K, const T* __restrict__ R, long long ldr,
                                                     long long stride_a, int rank, float factor, Segs sg, KeepArgs ka,
                                                     float* __restrict__ t, int ldt) {
  const int lane = threadIdx.x & 63, groups = ldt / SR_RANKS;
  const long long id = block_of_grid() * 4 + (threadIdx.x >> 6);
  const int row = (int)(id / groups), i0 = (int)(id % groups) * SR_RANKS;
  if (row >= sg.M) return;
  const int q = seg_find(sg, row);
  if (q < 0) return;
  const Span sp = seg_span(sg, q, row, row + 1);
  if (sp.a < 0) return;
  const KeepKey key = keep_key(ka);
  const T* Ra = R + (long long)sp.a * stride_a;
  float acc[SR_RANKS] = {};
  const T *xr = X + row * ldx, *ar[SR_RANKS];
#pragma unroll
  for (int i = 0; i < SR_RANKS; ++i) ar[i] = Ra + (i0 + i < rank ? i0 + i : rank - 1) * ldr;
  auto step = [&](Frag8<T> x, const Frag8<T> (&a)[SR_RANKS], int k) {
    if (DROP) frag_keep(x, keep8(ka, key, (uint64_t)row, (uint32_t)(k >> 3)));
#pragma unroll
    for (int i = 0; i < SR_RANKS; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[i] = fmaf((float)x.v[j], (float)a[i].v[j], acc[i]);
  };
  int k = 8 * lane;
#pragma unroll 2
  for (; k + 8 <= K; k += 512) {
    Frag8<T> a[SR_RANKS];
    const Frag8<T> x = frag_load(xr + k);
#pragma unroll
    for (int i = 0; i < SR_RANKS; ++i) a[i] = frag_load(ar[i] + k);
    all_loads_first();
    step(x, a, k);
  }
  if (k < K) {
    Frag8<T> a[SR_RANKS];
    const Frag8<T> x = frag_load(xr + k, K - k);
#pragma unroll
    for (int i = 0; i < SR_RANKS; ++i) a[i] = frag_load(ar[i] + k, K - k);
    step(x, a, k);
  }
  const float f = factor * (sg.scale != nullptr ? sg.scale[sp.a] : 1.f);
#pragma unroll
  for (int i = 0; i < SR_RANKS; ++i) {
    float v = acc[i];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    if (lane == i) t[(long long)row * ldt + i0 + i] = i0 + i < rank ? v * f : 0.f;
  }
}

// ---- the projection with the low-rank part: out (M, Nn) = X (M, Kk) W^T (+ bias) + t Bt_a^T, tiles of BM x BN in LDS, rows of
// 128 bytes along the reduction, 16-byte chunks XOR-ed with the row (conflict-free 16-byte reads).  Two LDS buffers and one
// barrier a step: the step after next is on its way to registers while a step is computed.  Bound by the two workgroups a CU that
// its registers allow, neither of which hides all waits of the other: 6001 x 1024 x 4096 fp16 with rank 32 97 us (519 TFLOP/s).
__device__ __forceinline__ f32x16 mma32(uint4 a, uint4 b, f32x16 c, f16) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(uint4 a, uint4 b, f32x16 c, bf16) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(uint4 a, uint4 b, f32x16 c, float) {
  const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], y[j], c, 0, 0, 0);
  return c;
}

// eight 32-bit values as a high and a low bf16 part
__device__ __forceinline__ void split8(const float* v, bf16x8& hi, bf16x8& lo) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    hi[j] = (bf16)v[j];
    const float f = (float)hi[j];
    lo[j] = (bf16)(fabsf(f) < INFINITY ? v[j] - f : 0.f);
  }
}
// the low-rank term of one 32 x 32 block: b (outputs) times v (rows), over 2 V ranks.  Written out for sums in ordinary registers: the
// wide projection keeps its own in all accumulation registers, which the compiler would take for these.  The waits are those
// between dependent products and before a sum is read (sixteen passes at most).
__device__ __forceinline__ f32x16 mma_low(uint4 b, const float (&v)[8], f32x16 c, bf16) {
  bf16x8 hi, lo;
  split8(v, hi, lo);
  asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0\n\ts_nop 9\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %3, %0\n\ts_nop 15\n\ts_nop 3"
               : "+v"(c) : "v"(__builtin_bit_cast(f32x4, b)), "v"(__builtin_bit_cast(f32x4, lo)), "v"(__builtin_bit_cast(f32x4, hi)));
  return c;
}
__device__ __forceinline__ f32x16 mma_low(uint4 b, const float (&v)[8], f32x16 c, f16) {
  bf16x8 hi, lo, bh, bl;
  split8(v, hi, lo);
  const f16x8 x = __builtin_bit_cast(f16x8, b);
  float f[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = (float)x[j];
  split8(f, bh, bl);
  asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %3, %0\n\ts_nop 9\n\tv_mfma_f32_32x32x16_bf16 %0, %2, %4, %0\n\ts_nop 9\n\t"
               "v_mfma_f32_32x32x16_bf16 %0, %1, %4, %0\n\ts_nop 15\n\ts_nop 3"
               : "+v"(c) : "v"(__builtin_bit_cast(f32x4, bh)), "v"(__builtin_bit_cast(f32x4, bl)), "v"(__builtin_bit_cast(f32x4, lo)),
                 "v"(__builtin_bit_cast(f32x4, hi)));
  return c;
}
__device__ __forceinline__ f32x16 mma_low(uint4 b, const float (&v)[4], f32x16 c, float) {
  const f32x4 x = __builtin_bit_cast(f32x4, b);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x2_f32 %0, %1, %2, %0\n\ts_nop 15\n\ts_nop 3" : "+v"(c) : "v"(x[j]), "v"(v[j]));
  return c;
}

struct LowRank {
  const float* t;          // [M][ldt], zeros behind the rank, or nullptr: no adapters at all
  const void* b;           // element (adapter a, output n, i) at a * sa + n * sn + i
  long long sa, sn;
  int rank, ldt;           // ldt: the rank rounded up to 8
};

// What a tile's rows m0 .. m1 - 1 belong to: the first request that may hold some of them, and whether it holds them all
struct Owner { int q, a; bool whole; };
template <typename Starts> __device__ __forceinline__ Owner owner_of(const Segs& sg, const Starts& of, int m0, int m1) {
  Owner o = {of.find(m0), -1, false};
  if (o.q < 0) o.q = 0;
  if (o.q < sg.S) {
    o.whole = of.start(o.q) <= m0 && of.start(o.q + 1) >= m1;
    o.a = of.adapter(o.q);
    if (o.a >= sg.n_adapters) o.a = -1;
  }
  return o;
}
// row_start and adapter where they lie
struct InMemory {
  const Segs& sg;
  __device__ __forceinline__ int find(int row) const { return seg_find(sg, row); }
  __device__ __forceinline__ int start(int q) const { return sg.row_start[q]; }
  __device__ __forceinline__ int adapter(int q) const { return sg.adapter[q]; }
};

// adds the low-rank term to one wave's row of blocks: rows mb .. mb + 31, outputs nw ..
// (`between` is run behind the first loads and before what waits for them)
template <typename T, int NI, typename Starts, typename Between>
__device__ __forceinline__ void low_rank(f32x16 (&sum)[NI], const LowRank& lr, const Segs& sg, const Starts& of, const Owner& own, int Nn, int m1,
                                         int mb, int nw, int lane, Between&& between) {
  constexpr int V = Lines<T>::V;
  const int l32 = lane & 31, h = lane >> 5, row = mb + l32;
  const bool even = lr.rank % V == 0;                 // whole lines of B
  // a half wave whose ranks lie behind the last reads the other half's and gets zeros
  auto ranks = [&](const float* tr, int i0, float (&v)[V]) {
    const int i = i0 + V * h;
    const bool in = i < lr.rank;
    f32x4 t4[V / 4];
#pragma unroll
    for (int j = 0; j < V / 4; ++j) t4[j] = *reinterpret_cast<const f32x4*>(tr + (in ? i : i0) + 4 * j);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = in ? t4[j / 4][j % 4] : 0.f;
  };
  auto outputs = [&](const T* ba, int n, int i0) {
    const int i = i0 + V * h, col = nw + n * 32 + l32;
    const bool in = i < lr.rank;
    const T* bp = ba + (col < Nn ? col : Nn - 1) * lr.sn;
    const uint4 b = even ? line_load(bp + (in ? i : i0)) : line_load(bp + i, lr.rank - i);
    return in ? b : uint4{0, 0, 0, 0};
  };
  if (own.whole) {                                    // one request's: no selection
    if (own.a < 0) { between(); return; }
    const T* ba = static_cast<const T*>(lr.b) + (long long)own.a * lr.sa;
    const float* tr = lr.t + (long long)(row < m1 ? row : m1 - 1) * lr.ldt;
#pragma unroll 1
    for (int i0 = 0; i0 < lr.rank; i0 += 2 * V) {
      float v[V];
      uint4 b[NI];
      ranks(tr, i0, v);
#pragma unroll
      for (int n = 0; n < NI; ++n) b[n] = outputs(ba, n, i0);
      if (i0 == 0) { all_loads_first(); between(); }
#pragma unroll
      for (int n = 0; n < NI; ++n) sum[n] = mma_low(b[n], v, sum[n], T());
    }
    return;
  }
  between();
  const int r1 = mb + 32 < m1 ? mb + 32 : m1;
#pragma unroll 1
  for (int q = own.q; q < sg.S; ++q) {
    const int s0 = of.start(q), s1 = of.start(q + 1), a = of.adapter(q);
    if (s0 >= r1) break;
    if (a < 0 || a >= sg.n_adapters || s1 <= mb || s1 <= s0) continue;
    const bool mine = row >= s0 && row < s1 && row < r1;
    const T* ba = static_cast<const T*>(lr.b) + (long long)a * lr.sa;
    const float* tr = lr.t + (long long)(mine ? row : s0 > mb ? s0 : mb) * lr.ldt;
    f32x16 add[NI];
#pragma unroll
    for (int n = 0; n < NI; ++n) add[n] = sum[n];
#pragma unroll 1
    for (int i0 = 0; i0 < lr.rank; i0 += 2 * V) {
      float v[V];
      uint4 b[NI];
      ranks(tr, i0, v);
#pragma unroll
      for (int n = 0; n < NI; ++n) b[n] = outputs(ba, n, i0);
#pragma unroll
      for (int n = 0; n < NI; ++n) add[n] = mma_low(b[n], v, add[n], T());
    }
#pragma unroll
    for (int n = 0; n < NI; ++n)
#pragma unroll
      for (int j = 0; j < 16; ++j) sum[n][j] = mine ? add[n][j] : sum[n][j];
  }
}

// the low-rank term of a row of blocks of dx, with the mask of x and the factor of what it keeps, added
template <typename T, int NI, typename Starts>
__device__ __forceinline__ void masked_low_rank(f32x16 (&sum)[NI], const LowRank& lr, const Segs& sg, const Starts& of, const KeepArgs& ka, KeepKey key,
                                                const Owner& own, int Nn, int m1, int mb, int nb, int lane) {
  const int l32 = lane & 31, h = lane >> 5;
  f32x16 add[NI];
  uint32_t keep[NI];
#pragma unroll
  for (int n = 0; n < NI; ++n)
#pragma unroll
    for (int j = 0; j < 16; ++j) add[n][j] = 0.f;
  low_rank<T, NI>(add, lr, sg, of, own, Nn, m1, mb, nb, lane, [&]() {
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      // lane h makes the draws of column blocks 2 h and 2 h + 1; its partner holds the other half of each block's columns
      const uint64_t row = (uint64_t)(mb + l32);
      const int cb = (nb >> 3) + 4 * n;
      const uint32_t k2 = keep8(ka, key, row, cb + 2 * h) | keep8(ka, key, row, cb + 2 * h + 1) << 8;
      const uint32_t o2 = __shfl_xor(k2, 32);
      keep[n] = h == 0 ? (k2 | o2 << 16) : (o2 | k2 << 16);
    }
  });
#pragma unroll
  for (int n = 0; n < NI; ++n)
#pragma unroll
    for (int j = 0; j < 16; ++j) sum[n][j] += (keep[n] >> (8 * (j >> 2) + 4 * h + (j & 3))) & 1 ? add[n][j] * ka.up : 0.f;
}

// 16 bytes of results of a 32 x 32 block: outputs 2 V q + V h .. of a lane's row.  A lane holds four outputs of a row and its partner
// (lane ^ 32) the next four; of 16-bit results the two exchange halves of a pair of groups
template <typename T> __device__ __forceinline__ uint4 line_of(const f32x16& sum, int q) {
  if constexpr (sizeof(T) == 2) {
    typedef T Two __attribute__((ext_vector_type(2)));
    uint32_t d[2][2];
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int j = 0; j < 2; ++j) d[e][j] = __builtin_bit_cast(uint32_t, Two{(T)sum[8 * q + 4 * e + 2 * j], (T)sum[8 * q + 4 * e + 2 * j + 1]});
    const auto lo = __builtin_amdgcn_permlane32_swap(d[0][0], d[1][0], false, false);
    const auto hi = __builtin_amdgcn_permlane32_swap(d[0][1], d[1][1], false, false);
    return uint4{lo[0], hi[0], lo[1], hi[1]};
  } else {
    return __builtin_bit_cast(uint4, f32x4{sum[4 * q], sum[4 * q + 1], sum[4 * q + 2], sum[4 * q + 3]});
  }
}
// the first n of 16 bytes of results (n <= 0: none)
template <typename T> __device__ __forceinline__ void store_line(T* o, uint4 v, int n) {
  constexpr int V = Lines<T>::V;
  if (n >= V) {
    *reinterpret_cast<LooseLine<T>*>(o) = __builtin_bit_cast(LooseLine<T>, v);
  } else {
    const Line<T> x = __builtin_bit_cast(Line<T>, v);
#pragma unroll
    for (int j = 0; j < V; ++j) if (j < n) o[j] = x.v[j];
  }
}

// the end of a wave's blocks (rows mw .., outputs nw ..): low-rank term (DROP: with the mask of x, in dx), bias, and out
template <typename T, int NI, int MI, bool DROP>
__device__ __forceinline__ void finish(const f32x16 (&acc)[NI][MI], const LowRank& lr, const Segs& sg, const KeepArgs& ka, const Owner& own, int Nn,
                                       int m1, int mw, int nw, const float* sb, T* out, long long ldo, int lane) {
  const int h = lane >> 5;
  const KeepKey key = keep_key(ka);
#pragma unroll
  for (int m = 0; m < MI; ++m) {
    const int mb = mw + m * 32;
    f32x16 sum[NI];
#pragma unroll
    for (int n = 0; n < NI; ++n)
#pragma unroll
      for (int j = 0; j < 16; ++j) sum[n][j] = acc[n][m][j] + sb[n * 32 + 8 * (j >> 2) + 4 * h + (j & 3)];
    if (lr.t != nullptr && mb < m1) {
      const Owner o = own.whole ? own : owner_of(sg, InMemory{sg}, mb, mb + 32 < m1 ? mb + 32 : m1);
      if (!DROP) {
        low_rank<T, NI>(sum, lr, sg, InMemory{sg}, o, Nn, m1, mb, nw, lane, []() {});
      } else {
        masked_low_rank<T, NI>(sum, lr, sg, InMemory{sg}, ka, key, o, Nn, m1, mb, nw, lane);
      }
    }
    const int row = mb + (lane & 31);
#pragma unroll
    for (int n = 0; n < NI; ++n)
#pragma unroll
      for (int q = 0; q < 16 / Lines<T>::V; ++q) {
        const int col = nw + n * 32 + (2 * q + h) * Lines<T>::V;
        const uint4 v = line_of<T>(sum[n], q);
        if (row < m1) store_line<T>(out + (long long)row * ldo + col, v, Nn - col);
      }
  }
}

template <typename T, int BM, int BN, int WGM, int WGN, bool DROP>
__global__ __launch_bounds__(64 * WGM * WGN, 2) void k_project(const T* __restrict__ X, long long ldx, int Kk, const T* __restrict__ W,
                                                            long long ldw, int Nn, const T* __restrict__ bias, LowRank lr, Segs sg,
                                                            KeepArgs ka, T* __restrict__ out, long long ldo, int tiles_n) {
  constexpr int NT = 64 * WGM * WGN, MI = BM / WGM / 32, NI = BN / WGN / 32, V = Lines<T>::V, KB = Lines<T>::KB;
  constexpr int RX = BM * 8 / NT, RW = BN * 8 / NT;
  __shared__ uint4 lds[2 * (BM + BN) * 8];
  __shared__ float sb[BN];
  uint4 (*sx)[BM * 8] = reinterpret_cast<uint4 (*)[BM * 8]>(lds);
  uint4 (*sw)[BN * 8] = reinterpret_cast<uint4 (*)[BN * 8]>(lds + 2 * BM * 8);
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, wm = w % WGM, wn = w / WGM, l32 = lane & 31, h = lane >> 5;
  // consecutive workgroups go to the eight XCDs in turn: give each XCD a contiguous run of tiles, so that the tiles that share
  // rows of X share an L2
  const int total = gridDim.x, xcd = blockIdx.x & 7, per = total >> 3, extra = total & 7;
  const int tile = xcd * per + (xcd < extra ? xcd : extra) + (blockIdx.x >> 3);
  const int m0 = (tile / tiles_n) * BM, n0 = (tile % tiles_n) * BN;
  const int m1 = m0 + BM < sg.M ? m0 + BM : sg.M;
  const bool busy = n0 + wn * NI * 32 < Nn;           // a wave without outputs loads and waits, and multiplies nothing

  // rows past the end are read as the last one: a row touches its own results alone, and those are not stored
  const int c = tid & 7, rr = tid >> 3;
  const char *bx = reinterpret_cast<const char*>(X + m0 * ldx), *bw = reinterpret_cast<const char*>(W + n0 * ldw);
  uint32_t ox[RX], ow[RW];                            // bytes from the tile's first row: the host keeps these below 2^31
#pragma unroll
  for (int j = 0; j < RX; ++j) {
    const int r = rr + j * (NT / 8);
    ox[j] = ((uint32_t)(m0 + r < sg.M ? r : sg.M - 1 - m0) * (uint32_t)ldx + c * V) * sizeof(T);
  }
#pragma unroll
  for (int j = 0; j < RW; ++j) {
    const int r = rr + j * (NT / 8);
    ow[j] = ((uint32_t)(n0 + r < Nn ? r : Nn - 1 - n0) * (uint32_t)ldw + c * V) * sizeof(T);
  }
  uint4 gx[RX], gw[RW];
  auto fetch = [&](int s) {
    const size_t k = (size_t)s * 128;
#pragma unroll
    for (int j = 0; j < RX; ++j) gx[j] = line_load(reinterpret_cast<const T*>(bx + k + ox[j]));
#pragma unroll
    for (int j = 0; j < RW; ++j) gw[j] = line_load(reinterpret_cast<const T*>(bw + k + ow[j]));
  };
  auto stash = [&](int buf) {
#pragma unroll
    for (int j = 0; j < RX; ++j) { const int r = rr + j * (NT / 8); sx[buf][r * 8 + (c ^ (r & 7))] = gx[j]; }
#pragma unroll
    for (int j = 0; j < RW; ++j) { const int r = rr + j * (NT / 8); sw[buf][r * 8 + (c ^ (r & 7))] = gw[j]; }
  };
  const int full = Kk / KB, rest = Kk - full * KB;
  if (full > 0) fetch(0);
  if (tid < BN) sb[tid] = bias != nullptr && n0 + tid < Nn ? (float)bias[n0 + tid] : 0.f;
  if (rest > 0) {                                     // what is left of the reduction goes first, through the second buffer
    const size_t k = (size_t)full * 128;
    const int n = rest - c * V;
#pragma unroll 1
    for (int r = rr; r < BM; r += NT / 8) {
      const uint32_t o = ((uint32_t)(m0 + r < sg.M ? r : sg.M - 1 - m0) * (uint32_t)ldx + c * V) * sizeof(T);
      sx[1][r * 8 + (c ^ (r & 7))] = line_load(reinterpret_cast<const T*>(bx + k + o), n);
    }
#pragma unroll 1
    for (int r = rr; r < BN; r += NT / 8) {
      const uint32_t o = ((uint32_t)(n0 + r < Nn ? r : Nn - 1 - n0) * (uint32_t)ldw + c * V) * sizeof(T);
      sw[1][r * 8 + (c ^ (r & 7))] = line_load(reinterpret_cast<const T*>(bw + k + o), n);
    }
  }

  f32x16 acc[NI][MI];
#pragma unroll
  for (int n = 0; n < NI; ++n)
#pragma unroll
    for (int m = 0; m < MI; ++m)
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[n][m][j] = 0.f;

  Owner own = {0, -1, false};
  if (lr.t != nullptr && busy) own = owner_of(sg, InMemory{sg}, m0, m1);

  const int rx = (wm * MI * 32 + l32) * 8, rw = (wn * NI * 32 + l32) * 8, sel = l32 & 7;    // rows of a block differ by 32: one XOR
  auto chunk = [&](int buf, int kk) {                 // 2 V values of the reduction
    uint4 fx[MI], fw[NI];
    const int at = (2 * kk + h) ^ sel;
#pragma unroll
    for (int m = 0; m < MI; ++m) fx[m] = sx[buf][rx + m * 256 + at];
#pragma unroll
    for (int n = 0; n < NI; ++n) fw[n] = sw[buf][rw + n * 256 + at];
#pragma unroll
    for (int n = 0; n < NI; ++n)
#pragma unroll
      for (int m = 0; m < MI; ++m) acc[n][m] = mma32(fw[n], fx[m], acc[n][m], T());
  };
  if (full > 0) {
    stash(0);
    if (full > 1) fetch(1);
  }
  __syncthreads();
  if (rest > 0) {
    if (busy) {
#pragma unroll 1
      for (int kk = 0; kk * 2 * V < rest; ++kk) chunk(1, kk);
    }
    __syncthreads();
  }
  for (int s = 0; s < full; ++s) {
    const int buf = s & 1;
    if (s + 1 < full) {
      stash(buf ^ 1);
      if (s + 2 < full) fetch(s + 2);
    }
    if (busy) {
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) chunk(buf, kk);
    }
    __syncthreads();
  }
  if (!busy) return;

  finish<T, NI, MI, DROP>(acc, lr, sg, ka, own, Nn, m1, m0 + wm * MI * 32, n0 + wn * NI * 32, sb + wn * NI * 32, out, ldo, lane);
}

// ---- the same for many tiles: 256 x 256, four waves of 128 x 128 (one a SIMD, with all its registers), one workgroup a CU that goes
// from tile to tile.
//
// Bound by the matrix cores if everything else runs in their shadow: a wave has the fragments of the next chunk of the reduction on
// their way from the LDS while it multiplies this one, and between the products writes its part of the next step into the other
// buffer and sends for the step after that; one barrier a step, behind which the next step's first fragments are read.  128 x 128
// outputs a wave need half an LDS byte for each that 128 x 64 need three quarters of.  Loads run on across tiles: a new tile's
// first steps are under way while the last one is finished and stored.
// Measured without adapters: 8192 x 4096 x 4096 bf16 243 us (1131 TFLOP/s), 131072 x 512 x 512 bf16 89 us (half of it the way in and
// out of 1024 tiles), 65536 x 512 x 512 fp32 302 us (114 TFLOP/s).  With them: the first at rank 64 278 us, the last at rank 16 302 us
// where requests end with tiles and 339 where they end anywhere (rows of several requests are finished block by block).
constexpr int WIDE = 256, LDS_REQUESTS = 256;

// The sums of the wide projection, by the names of their registers: block (n, m) of a wave is a[16 (4 n + m)] .. + 15, all 256
// accumulation registers.  The compiler is not asked to place them: as variables they are copied wherever two paths meet, there
// is no register left to copy through, and sums travel through memory (measured: 13 us a tile instead of 3).  It has no other use
// for these registers, since what it keeps fits the 256 others.  What it cannot see it does not wait for: two products on the
// same sum lie at least two products apart (a product passes its sum on to the next by itself), and sums_done() comes before the
// sums are read.
#define HM_ALL_SUMS \
  "a0", "a1", "a2", "a3", "a4", "a5", "a6", "a7", "a8", "a9", "a10", "a11", "a12", "a13", "a14", "a15", "a16", "a17", "a18", \
  "a19", "a20", "a21", "a22", "a23", "a24", "a25", "a26", "a27", "a28", "a29", "a30", "a31", "a32", "a33", "a34", "a35", "a36", \
  "a37", "a38", "a39", "a40", "a41", "a42", "a43", "a44", "a45", "a46", "a47", "a48", "a49", "a50", "a51", "a52", "a53", "a54", \
  "a55", "a56", "a57", "a58", "a59", "a60", "a61", "a62", "a63", "a64", "a65", "a66", "a67", "a68", "a69", "a70", "a71", "a72", \
  "a73", "a74", "a75", "a76", "a77", "a78", "a79", "a80", "a81", "a82", "a83", "a84", "a85", "a86", "a87", "a88", "a89", "a90", \
  "a91", "a92", "a93", "a94", "a95", "a96", "a97", "a98", "a99", "a100", "a101", "a102", "a103", "a104", "a105", "a106", "a107", \
  "a108", "a109", "a110", "a111", "a112", "a113", "a114", "a115", "a116", "a117", "a118", "a119", "a120", "a121", "a122", "a123", \
  "a124", "a125", "a126", "a127", "a128", "a129", "a130", "a131", "a132", "a133", "a134", "a135", "a136", "a137", "a138", "a139", \
  "a140", "a141", "a142", "a143", "a144", "a145", "a146", "a147", "a148", "a149", "a150", "a151", "a152", "a153", "a154", "a155", \
  "a156", "a157", "a158", "a159", "a160", "a161", "a162", "a163", "a164", "a165", "a166", "a167", "a168", "a169", "a170", "a171", \
  "a172", "a173", "a174", "a175", "a176", "a177", "a178", "a179", "a180", "a181", "a182", "a183", "a184", "a185", "a186", "a187", \
  "a188", "a189", "a190", "a191", "a192", "a193", "a194", "a195", "a196", "a197", "a198", "a199", "a200", "a201", "a202", "a203", \
  "a204", "a205", "a206", "a207", "a208", "a209", "a210", "a211", "a212", "a213", "a214", "a215", "a216", "a217", "a218", "a219", \
  "a220", "a221", "a222", "a223", "a224", "a225", "a226", "a227", "a228", "a229", "a230", "a231", "a232", "a233", "a234", "a235", \
  "a236", "a237", "a238", "a239", "a240", "a241", "a242", "a243", "a244", "a245", "a246", "a247", "a248", "a249", "a250", "a251", \
  "a252", "a253", "a254", "a255"
__device__ __forceinline__ void sums_clear() {
  asm volatile("" ::: HM_ALL_SUMS);
#pragma unroll
  for (int i = 0; i < 256; ++i) asm volatile("v_accvgpr_write_b32 a[%0], 0" ::"i"(i));
  asm volatile("s_nop 7");
}
__device__ __forceinline__ void sums_done() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }   // more than the sixteen passes of the last product
__device__ __forceinline__ void sums_used() { asm volatile("" ::: HM_ALL_SUMS); }
__device__ __forceinline__ f32x16 sums_of(int n, int m) {
  f32x16 v;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    float x;
    asm volatile("v_accvgpr_read_b32 %0, a[%1]" : "=v"(x) : "i"(16 * (4 * n + m) + j));
    v[j] = x;
  }
  return v;
}
__device__ __forceinline__ void mma_sums(int n, int m, uint4 a, uint4 b, f16) {
  asm volatile("v_mfma_f32_32x32x16_f16 a[%2:%3], %0, %1, a[%2:%3]" ::"v"(__builtin_bit_cast(f32x4, a)), "v"(__builtin_bit_cast(f32x4, b)),
               "i"(16 * (4 * n + m)), "i"(16 * (4 * n + m) + 15));
}
__device__ __forceinline__ void mma_sums(int n, int m, uint4 a, uint4 b, bf16) {
  asm volatile("v_mfma_f32_32x32x16_bf16 a[%2:%3], %0, %1, a[%2:%3]" ::"v"(__builtin_bit_cast(f32x4, a)), "v"(__builtin_bit_cast(f32x4, b)),
               "i"(16 * (4 * n + m)), "i"(16 * (4 * n + m) + 15));
}
__device__ __forceinline__ void mma_sums(int n, int m, float a, float b) {
  asm volatile("v_mfma_f32_32x32x2_f32 a[%2:%3], %0, %1, a[%2:%3]" ::"v"(a), "v"(b), "i"(16 * (4 * n + m)), "i"(16 * (4 * n + m) + 15));
}

// the same of fragments that vector instructions have just written: those must lie two wait states back
__device__ __forceinline__ void mma_sums_late(int n, int m, bf16x8 a, bf16x8 b) {
  asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 a[%2:%3], %0, %1, a[%2:%3]" ::"v"(a), "v"(b), "i"(16 * (4 * n + m)), "i"(16 * (4 * n + m) + 15));
}
__device__ __forceinline__ void mma_sums_late(int n, int m, float a, float b) {
  asm volatile("s_nop 1\n\tv_mfma_f32_32x32x2_f32 a[%2:%3], %0, %1, a[%2:%3]" ::"v"(a), "v"(b), "i"(16 * (4 * n + m)), "i"(16 * (4 * n + m) + 15));
}

// the low-rank term of row blocks FIRST .. LAST - 1 of a wave's 128 x 128 outputs, which belong to adapter a, added where the sums are
template <typename T, int FIRST, int LAST>
__device__ __forceinline__ void low_rank_here(const LowRank& lr, int a, int Nn, int m1, int mw, int nw, int lane) {
  constexpr int V = Lines<T>::V, MB = LAST - FIRST;
  const int l32 = lane & 31, h = lane >> 5;
  const bool even = lr.rank % V == 0;                 // whole lines of B
  const T* ba = static_cast<const T*>(lr.b) + (long long)a * lr.sa;
#pragma unroll 1
  for (int i0 = 0; i0 < lr.rank; i0 += 2 * V) {
    const int i = i0 + V * h;
    const bool in = i < lr.rank;                      // a half wave whose ranks lie behind the last reads the other half's and gets zeros
    uint4 b[4];
    f32x4 t4[MB][V / 4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int col = nw + n * 32 + l32;
      const T* bp = ba + (col < Nn ? col : Nn - 1) * lr.sn;
      b[n] = even ? line_load(bp + (in ? i : i0)) : line_load(bp + i, lr.rank - i);
    }
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      const int row = mw + (FIRST + m) * 32 + l32;
      const float* tr = lr.t + (long long)(row < m1 ? row : m1 - 1) * lr.ldt + (in ? i : i0);
#pragma unroll
      for (int j = 0; j < V / 4; ++j) t4[m][j] = *reinterpret_cast<const f32x4*>(tr + 4 * j);
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) if (!in) b[n] = uint4{0, 0, 0, 0};
    // (two products on the same sum lie at least two products apart)
    if constexpr (sizeof(T) == 2) {
      bf16x8 hi[MB], lo[MB];
#pragma unroll
      for (int m = 0; m < MB; ++m) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = in ? t4[m][j / 4][j % 4] : 0.f;
        split8(v, hi[m], lo[m]);
      }
#pragma unroll
      for (int n2 = 0; n2 < 4; n2 += 2) {
        bf16x8 bh[2], bl[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          if constexpr (__is_same(T, f16)) {
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = (float)__builtin_bit_cast(f16x8, b[n2 + n])[j];
            split8(f, bh[n], bl[n]);
          } else {
            bh[n] = __builtin_bit_cast(bf16x8, b[n2 + n]);
          }
        }
#pragma unroll
        for (int part = 0; part < (__is_same(T, f16) ? 3 : 2); ++part)
#pragma unroll
          for (int m = 0; m < MB; ++m)
#pragma unroll
            for (int n = 0; n < 2; ++n)
              mma_sums_late(n2 + n, FIRST + m, __is_same(T, f16) && part == 1 ? bl[n] : bh[n], part == 0 ? lo[m] : hi[m]);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
          for (int n = 0; n < 4; ++n) mma_sums_late(n, FIRST + m, __builtin_bit_cast(f32x4, b[n])[j], in ? t4[m][0][j] : 0.f);
    }
  }
}

template <int N> struct Number { static constexpr int value = N; };

struct InLds {
  const Segs& sg;
  const int (*at)[LDS_REQUESTS];
  int lane;
  __device__ __forceinline__ int find(int row) const {
    int n = 0;
    for (int q = 0; q < sg.S; q += 64) n += __popcll(__ballot(q + lane < sg.S && at[0][q + lane] <= row));
    return n - 1;
  }
  __device__ __forceinline__ int start(int q) const { return __builtin_amdgcn_readfirstlane(at[0][q]); }
  __device__ __forceinline__ int adapter(int q) const { return __builtin_amdgcn_readfirstlane(at[1][q]); }
};

// a row's last n values (n = 1 .. V - 1), read as the 16 bytes that end with the row: moved down, zeros above; n <= 0: zeros
template <typename T> __device__ __forceinline__ uint4 line_down(uint4 q, int n) {
  constexpr int V = Lines<T>::V;
  uint64_t lo = q.x | (uint64_t)q.y << 32, hi = q.z | (uint64_t)q.w << 32;
  const int bits = (n >= V ? 0 : V - n) * 8 * (int)sizeof(T);
  const bool far = bits >= 64;
  const uint64_t a = far ? hi : lo, b = far ? 0 : hi;
  const int r = bits & 63;
  lo = a >> r | (r != 0 ? b << (64 - r) : 0);
  hi = b >> r;
  if (n <= 0) lo = hi = 0;
  return uint4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}

// `v`, which the compiler takes for a new value
__device__ __forceinline__ int fresh(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

template <typename T, bool DROP>
__global__ __launch_bounds__(256, 1) void k_project_wide(const T* __restrict__ X, long long ldx, int Kk, const T* __restrict__ W, long long ldw,
                                                         int Nn, const T* __restrict__ bias, LowRank lr, Segs sg, KeepArgs ka,
                                                         T* __restrict__ out, long long ldo, int tiles_m, int tiles_n) {
  constexpr int MI = 4, NI = 4, V = Lines<T>::V, KB = Lines<T>::KB;
  __shared__ uint4 lds[2][2 * WIDE * 8];              // X lines, then W lines
  __shared__ uint4 stage[4][256];                     // 32 lines of results a wave
  __shared__ float sb[4][WIDE / 2];                   // the bias of each wave's outputs, written and read by that wave alone
  __shared__ int starts[2][LDS_REQUESTS];             // row_start, and the adapter of each request, where they are few
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), wm = w & 1, wn = w >> 1;
  const int lane = tid & 63, l32 = lane & 31, h = lane >> 5;
  // workgroups go to the eight XCDs in turn: each XCD takes a contiguous run of tiles, its 32 workgroups neighbours in it, in
  // bands of eight tiles of rows (eight by four tiles at a time share what their L2 holds)
  const int total = tiles_m * tiles_n, xcd = blockIdx.x & 7, each = total >> 3, extra = total & 7;
  const int first = xcd * each + (xcd < extra ? xcd : extra), end = first + each + (xcd < extra ? 1 : 0);
  auto place = [&](int tile, int& m0, int& n0) {
    const int band = tile / (8 * tiles_n), in = tile - band * 8 * tiles_n;
    const int high = tiles_m - band * 8 < 8 ? tiles_m - band * 8 : 8;
    m0 = (band * 8 + in % high) * WIDE;
    n0 = in / high * WIDE;
  };
  const int full = Kk / KB, rest = Kk - full * KB, steps = full + (rest > 0);
  const int rr = tid >> 3, c = tid & 7;
  // the last step of a row that does not end with a line: the lane reads the 16 bytes that end with the row (or, where it has no
  // value left, some of the step before) and moves them down when it writes them
  const int left = rest - c * V;
  const uint32_t tail_back = left >= V ? 0 : left > 0 ? (V - left) * (int)sizeof(T) : 128;
  // where the loads are: tile, step, and what belongs to them (128 bytes before the step, for tail_back).  Rows past the end are
  // read as the last one: a row touches its own results alone.  Behind the last tile its own steps are read again, and not used
  int f_tile = first + (blockIdx.x >> 3), f_step = 0;
  const char *fx, *fw;
  uint32_t ox[8], ow[8], back = 128;
  auto aim = [&]() {
    int m0, n0;
    place(f_tile, m0, n0);
    fx = reinterpret_cast<const char*>(X + m0 * ldx) - 128;
    fw = reinterpret_cast<const char*>(W + n0 * ldw) - 128;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int r = rr + 32 * j;
      ox[j] = ((uint32_t)(m0 + r < sg.M ? r : sg.M - 1 - m0) * (uint32_t)ldx + c * V) * sizeof(T);
      ow[j] = ((uint32_t)(n0 + r < Nn ? r : Nn - 1 - n0) * (uint32_t)ldw + c * V) * sizeof(T);
    }
  };
  uint4 gl[16];                                       // eight lines of X, eight of W
  auto fetch = [&](int j) {
    gl[j] = j < 8 ? line_load(reinterpret_cast<const T*>(fx + (ox[j & 7] + back))) : line_load(reinterpret_cast<const T*>(fw + (ow[j & 7] + back)));
  };
  auto next = [&]() {
    fx += 128;
    fw += 128;
    if (++f_step == steps) {
      asm volatile("; another tile");                 // keeps this a branch: its 140 instructions would be run at every step
      f_step = 0;
      if (f_tile + 32 < end) f_tile += 32;
      aim();
    }
    back = f_step < full ? 128 : 128 - tail_back;
  };
  const int to = rr * 8 + (c ^ (rr & 7));             // rows of a thread differ by 32: one XOR
  auto stash = [&](int buf, int j) {
    lds[buf][(j < 8 ? 0 : WIDE * 8) + to + (j & 7) * 256] = gl[j];
  };
  int tile = f_tile;
  if (tile >= end) return;
  const bool cached = sg.S < LDS_REQUESTS;
  if (cached && lr.t != nullptr) {
    if (tid <= sg.S) starts[0][tid] = sg.row_start[tid];
    if (tid < sg.S) starts[1][tid] = sg.adapter[tid];
  }
  aim();
#pragma unroll
  for (int j = 0; j < 16; ++j) fetch(j);
  next();
#pragma unroll
  for (int j = 0; j < 16; ++j) stash(0, j);           // the host keeps full >= 1
#pragma unroll
  for (int j = 0; j < 16; ++j) fetch(j);
  int s_step = f_step;                                // step that gl holds
  next();
  __syncthreads();
  const int rx = (wm * 128 + l32) * 8, rw = WIDE * 8 + (wn * 128 + l32) * 8, sel = l32 & 7;
  uint4 fr[2][8];                                     // fragments of this chunk and the next: four of W, four of X
  auto read = [&](int buf, int kk, int set, int i) {
    const int at = (2 * kk + h) ^ sel;
    fr[set][i] = lds[buf][(i < 4 ? rw + i * 256 : rx + (i - 4) * 256) + at];
  };
  int buf = 0;
  for (; tile < end; tile += 32) {
    int m0, n0;
    place(tile, m0, n0);
    const int m1 = m0 + WIDE < sg.M ? m0 + WIDE : sg.M;
    const int mw = m0 + wm * 128, nw = n0 + wn * 128;
    const bool busy = nw < Nn;                        // a wave without outputs keeps step, and stores nothing
    auto owner = [&](int r0, int r1, int ln) { return cached ? owner_of(sg, InLds{sg, starts, ln}, r0, r1) : owner_of(sg, InMemory{sg}, r0, r1); };
    Owner own = {0, -1, false};
    if (lr.t != nullptr) own = owner(m0, m1, fresh(tid) & 63);
    sums_clear();
    // waves finish a tile at different times, with no barrier between that and the next tile: what one of them adds there must not
    // be written by another
    if (bias != nullptr) {
      const int ln = fresh(tid) & 63;
#pragma unroll
      for (int e = 0; e < 2; ++e) sb[w][64 * e + ln] = nw + 64 * e + ln < Nn ? (float)bias[nw + 64 * e + ln] : 0.f;
    }
    // (the last step of the tile before read these too; across its end they would take 32 registers)
#pragma unroll
    for (int i = 0; i < 8; ++i) read(buf, 0, 0, i);
    for (int s = 0; s < steps; ++s) {
      if (s_step >= full) {
        const int n = rest - (fresh(tid) & 7) * V;
#pragma unroll
        for (int j = 0; j < 16; ++j) gl[j] = line_down<T>(gl[j], n);
      }
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const int now = kk & 1;
        if (kk == 3) __syncthreads();                 // the next step lies in the LDS, and no fragment of the one before this is waited for
#pragma unroll
        for (int j = 0; j < (sizeof(T) == 2 ? 1 : 4); ++j) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              // at most two memory instructions between two products: more take longer to send than a product lasts
              if (j == 0 && e == 0) {
                if (kk < 3) read(buf, kk + 1, now ^ 1, i);
                else read(buf ^ 1, 0, now ^ 1, i);
              } else if (j == 0 && (kk == 1 || kk == 2)) {
                stash(buf ^ 1, (kk - 1) * 8 + i);
                fetch((kk - 1) * 8 + i);
              }
              __builtin_amdgcn_sched_barrier(0);
              const int n = (2 * i + e) >> 2, m = (2 * i + e) & 3;
              if constexpr (sizeof(T) == 2) {
                mma_sums(n, m, fr[now][n], fr[now][4 + m], T());
              } else {
                mma_sums(n, m, __builtin_bit_cast(f32x4, fr[now][n])[j], __builtin_bit_cast(f32x4, fr[now][4 + m])[j]);
              }
              __builtin_amdgcn_sched_barrier(0);
            }
          }
        }
      }
      s_step = f_step;
      next();
      buf ^= 1;
    }
    // the low-rank term comes after the main loop: before it, its loads would stand in line behind the stores of the tile before
    // row blocks of 32 that lie in one request get their low-rank term here; bit m of `open`: block m does not
    unsigned open = 0;
    if (lr.t != nullptr) {
      const int ln = fresh(tid) & 63;
      if (DROP || !busy) {
        open = 15;
      } else if (own.whole) {
        if (own.a >= 0) {
          if constexpr (__is_same(T, f16)) {          // (its weights take two parts: half the rows at a time fit the registers)
            low_rank_here<T, 0, 2>(lr, own.a, Nn, m1, mw, nw, ln);
            low_rank_here<T, 2, 4>(lr, own.a, Nn, m1, mw, nw, ln);
          } else {
            low_rank_here<T, 0, 4>(lr, own.a, Nn, m1, mw, nw, ln);
          }
        }
      } else {
        auto block = [&](auto of) {
          constexpr int M = decltype(of)::value;
          const int r0 = mw + M * 32, r1 = r0 + 32 < m1 ? r0 + 32 : m1;
          if (r0 >= m1) return;
          const Owner o = owner(r0, r1, ln);
          if (!o.whole) open |= 1u << M;
          else if (o.a >= 0) low_rank_here<T, M, M + 1>(lr, o.a, Nn, m1, mw, nw, ln);
        };
        block(Number<0>()); block(Number<1>()); block(Number<2>()); block(Number<3>());
      }
    }
    sums_done();
    if (!busy) continue;
    // 32 rows of 128 bytes at a time (two blocks of 16-bit results, one of fp32), through the wave's own part of the LDS: in the
    // layout of the products a row's results leave in pieces of 32 bytes, which the memory path takes four times as long for
    constexpr int PAIR = sizeof(T) == 2 ? 2 : 1;
    const KeepKey key = keep_key(ka);
#pragma unroll 1
    for (int k = 0; k < NI * MI; k += PAIR) {         // block k: outputs k % 4, rows k / 4
      const int mb = mw + (k >> 2) * 32, nb = nw + (k & 3) * 32, ln = fresh(tid) & 63, l32 = ln & 31, h = ln >> 5;
      if (mb >= m1 || nb >= Nn) continue;
      f32x16 sum[PAIR];
#define HM_BLOCK(U)                                                       \
      case U:                                                             \
        sum[0] = sums_of(U & 3, U >> 2);                                  \
        if constexpr (PAIR == 2) sum[PAIR - 1] = sums_of((U + 1) & 3, U >> 2); \
        break;
      if constexpr (PAIR == 2) {
        switch (k) { HM_BLOCK(0) HM_BLOCK(2) HM_BLOCK(4) HM_BLOCK(6) HM_BLOCK(8) HM_BLOCK(10) HM_BLOCK(12) HM_BLOCK(14) }
      } else {
        switch (k) {
          HM_BLOCK(0) HM_BLOCK(1) HM_BLOCK(2) HM_BLOCK(3) HM_BLOCK(4) HM_BLOCK(5) HM_BLOCK(6) HM_BLOCK(7)
          HM_BLOCK(8) HM_BLOCK(9) HM_BLOCK(10) HM_BLOCK(11) HM_BLOCK(12) HM_BLOCK(13) HM_BLOCK(14) HM_BLOCK(15)
        }
      }
#undef HM_BLOCK
      if (DROP ? lr.t != nullptr : open >> (k >> 2) & 1) {       // a mask, or several requests' rows
        const Owner o = own.whole ? own : owner(mb, mb + 32 < m1 ? mb + 32 : m1, ln);
        auto add = [&](const auto& of) {
          if constexpr (DROP) masked_low_rank<T, PAIR>(sum, lr, sg, of, ka, key, o, Nn, m1, mb, nb, ln);
          else low_rank<T, PAIR>(sum, lr, sg, of, o, Nn, m1, mb, nb, ln, []() {});
        };
        if (cached) add(InLds{sg, starts, ln});
        else add(InMemory{sg});
      }
      if (bias != nullptr) {                          // a lane's outputs are nb + 32 e + 8 (j / 4) + 4 h + j % 4
        const float* b = sb[w] + nb - nw + 4 * h;
#pragma unroll
        for (int e = 0; e < PAIR; ++e)
#pragma unroll
          for (int j = 0; j < 16; ++j) sum[e][j] += b[e * 32 + 8 * (j >> 2) + (j & 3)];
      }
#pragma unroll
      for (int e = 0; e < PAIR; ++e)
#pragma unroll
        for (int q = 0; q < 4 / PAIR; ++q) stage[w][l32 * 8 + ((e * 4 + 2 * q + h) ^ (l32 & 7))] = line_of<T>(sum[e], q);
      wave_sees_lds();
      uint4 line[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) { const int r = i * 8 + (ln >> 3); line[i] = stage[w][r * 8 + ((ln & 7) ^ (r & 7))]; }
      const int col = nb + (ln & 7) * V;
      T* o = out + (long long)(mb + (ln >> 3)) * ldo + col;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (mb + i * 8 + (ln >> 3) < m1) store_line<T>(o, line[i], Nn - col);
        o += 8 * ldo;
      }
      wave_sees_lds();
    }
    sums_used();
  }
}

// ---- few rows: the weights are read once for each 64 rows, sixteen outputs a workgroup, its waves share the reduction
// (up to 256 rows: 37 us of 256 rows x 4096 x 4096 bf16 against 56 of the tiles of 64, 21 against 54 of 128 rows; 64 rows with
// 48 adapters of rank 16 13 us, bound by the way of W through the LDS, 2.6 TB/s).  Forward alone: dx of few rows takes the tiles of
// 64, which have the mask of x (54 of the 317 us of a training call of 128 single rows x 4096 x 4096).
constexpr int FEW_ROWS = 256, FEW_WAVES = 8;

template <typename T, int MT>
__global__ __launch_bounds__(64 * FEW_WAVES) void k_project_few(const T* __restrict__ X, long long ldx, int K, const T* __restrict__ W,
                                                                long long ldw, int N, const T* __restrict__ bias, LowRank lr, Segs sg,
                                                                T* __restrict__ out, long long ldo) {
  constexpr int U = strip_units<1, MT>();
  __shared__ uint4 lds[FEW_WAVES * U];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, l16 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  // wave w finishes rows m0 + 16 w .. m0 + 16 w + 15, lane: row m0 + 16 w + l16, outputs n0 + 4 g .. + 3.  Its adapter: how many requests start
  // at or before the row, 64 of them looked at at a time by all lanes
  const int m0 = blockIdx.y * 64, row = m0 + 16 * w + l16, col = n0 + 4 * g;
  int a = -1;
  if (lr.t != nullptr && w < MT) {
    int before = 0;
    for (int s0 = 0; s0 < sg.S; s0 += 64) {
      const int start = s0 + lane < sg.S ? sg.row_start[s0 + lane] : 0x7fffffff;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int n = __popcll(__ballot(start <= m0 + 16 * w + r));
        before += l16 == r ? n : 0;
      }
    }
    if (before > 0 && row < sg.M) a = seg_span(sg, before - 1, row, row + 1).a;
  }
  f32x4 acc[MT][1];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m][0] = f32x4{0.f, 0.f, 0.f, 0.f};
  strip_sum<T, 1, MT, FEW_WAVES, false>(acc, W + (long long)n0 * ldw, ldw, N - n0, X + (long long)m0 * ldx, ldx, sg.M - m0, K, lds + w * U, w, lane, KeepArgs{}, KeepKey{}, 0);
  f32x4* red = reinterpret_cast<f32x4*>(lds);
#pragma unroll
  for (int m = 0; m < MT; ++m) red[w * U + m * 64 + lane] = acc[m][0];
  __syncthreads();
  if (w >= MT || row >= sg.M) return;
  f32x4 v = red[w * 64 + lane];
#pragma unroll
  for (int u = 1; u < FEW_WAVES; ++u) v += red[u * U + w * 64 + lane];
  if (a >= 0) {
    const T* b = static_cast<const T*>(lr.b) + (long long)a * lr.sa;
    const float* tr = lr.t + (long long)row * lr.ldt;
    if (lr.rank % 8 == 0) {
      for (int i = 0; i < lr.rank; i += 8) {
        const f32x4 t0 = *reinterpret_cast<const f32x4*>(tr + i), t1 = *reinterpret_cast<const f32x4*>(tr + i + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const Frag8<T> f = frag_load(b + (col + j < N ? col + j : N - 1) * lr.sn + i);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[j] = fmaf(t1[e], (float)f.v[e + 4], fmaf(t0[e], (float)f.v[e], v[j]));
        }
      }
    } else {
      for (int i = 0; i < lr.rank; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = fmaf(tr[i], (float)b[(col + j < N ? col + j : N - 1) * lr.sn + i], v[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (col + j < N) out[row * ldo + col + j] = (T)(v[j] + (bias != nullptr ? (float)bias[col + j] : 0.f));
}

// ---- sums over rows: G_a[p][i] = sum over the rows m of adapter a of X[m][p] t[m][i], 128 columns p and up to 64 ranks a
// workgroup.  The reduction runs along the rows, while a row lies along its columns.  A lane loads eight columns of each of its
// rows (whole lines), so what the matrix cores need -- consecutive rows of one column -- is in its own registers:
//   fp32    four rows a wave and step, 16 x 16 x 4 products, column j of every lane at a time;
//   16 bit  32 rows a wave and step (eight a lane), turned 8 x 8 in registers, 16 x 16 x 32 bf16 products with t split in two
//           (an eighth of the matrix time of the fp32 products, which bounded ranks over 16).
// About 1024 workgroups, each a run of rows; partial sums of (run, request) pairs in slots, added in order by k_outer_sum.  Bound by the
// time that loads take to come back: 2.7 TB/s over x and dy of 131072 rows (76 us).  The next step's loads sent ahead of this one's
// products cost the registers of a third workgroup a CU and take 92 us; four workgroups a CU spill.  Requests of one row each are
// taken one after the other, with one wave at work: 202 us of 128 rows x (4096 + 4096).
constexpr int OU_COLS = 128;

template <typename T, int RT> struct OuterSum {
  const T* X;
  const float* t;
  const KeepArgs& ka;
  KeepKey key;
  long long ldx;
  int P, p, ldt, g;
  int at[RT];              // ranks past the rank are read as the last one: not stored
  bool drop;
  __device__ __forceinline__ OuterSum(const T* X_, long long ldx_, int P_, const float* t_, int ldt_, int ib, int p_, int lane, bool drop_,
                                      const KeepArgs& ka_)
      : X(X_), t(t_), ka(ka_), key(keep_key(ka_)), ldx(ldx_), P(P_), p(p_), ldt(ldt_), g(lane >> 4), drop(drop_) {
#pragma unroll
    for (int i = 0; i < RT; ++i) { const int r = ib + 16 * i + (lane & 15); at[i] = r < ldt ? r : ldt - 1; }
  }
  __device__ __forceinline__ void mask(Frag8<T>& x, int m) const {
    uint32_t keep = keep8(ka, key, (uint64_t)m, (uint32_t)(p >> 3));
    if (p & 7) keep = (keep | keep8(ka, key, (uint64_t)m, (uint32_t)(p >> 3) + 1) << 8) >> (p & 7);
    frag_keep(x, keep);
  }
  // adds rows [lo, hi) to the sums of the four waves
  __device__ __forceinline__ void rows(f32x4 (&acc)[8][RT], int lo, int hi, int w) const;
  template <bool ALL> __device__ __forceinline__ void group(f32x4 (&acc)[8][RT], int m0, int hi) const;
};

__device__ __forceinline__ f32x4 mma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma_outer(bf16x8 x, bf16x8 hi, bf16x8 lo, f32x4 c) { return mma16(x, hi, mma16(x, lo, c)); }
__device__ __forceinline__ f32x4 mma_outer(f16x8 x, bf16x8 hi, bf16x8 lo, f32x4 c) {
  float f[8];
  bf16x8 xh, xl;
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = (float)x[j];
  split8(f, xh, xl);
  return mma16(xh, hi, mma16(xl, hi, mma16(xh, lo, c)));
}

// one step of a wave; ALL: every row lies before hi and a lane has its eight columns
template <typename T, int RT>
template <bool ALL>
__device__ __forceinline__ void OuterSum<T, RT>::group(f32x4 (&acc)[8][RT], int m0, int hi) const {
  constexpr int R = sizeof(T) == 2 ? 8 : 1;            // rows of a lane
  Frag8<T> x[R];
  float tv[RT][R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int m = m0 + R * g + r;
    if (ALL) {
      x[r] = frag_load(X + m * ldx + p);
#pragma unroll
      for (int i = 0; i < RT; ++i) tv[i][r] = t[(long long)m * ldt + at[i]];
    } else {
      const bool in = m < hi;
      x[r] = frag_load(X + (in ? m : m0) * ldx + p, in ? P - p : 0);
#pragma unroll
      for (int i = 0; i < RT; ++i) tv[i][r] = in ? t[(long long)m * ldt + at[i]] : 0.f;
    }
  }
  if (sizeof(T) == 2) all_loads_first();
  if (drop) {
#pragma unroll
    for (int r = 0; r < R; ++r) mask(x[r], m0 + R * g + r);
  }
  if constexpr (sizeof(T) == 2) {
    bf16x8 th[RT], tl[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) split8(tv[i], th[i], tl[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      decltype(x[0].v) col;
#pragma unroll
      for (int r = 0; r < 8; ++r) col[r] = x[r].v[j];
#pragma unroll
      for (int i = 0; i < RT; ++i) acc[j][i] = mma_outer(col, th[i], tl[i], acc[j][i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[0].v[j], tv[i][0], acc[j][i], 0, 0, 0);
  }
}

template <typename T, int RT>
__device__ __forceinline__ void OuterSum<T, RT>::rows(f32x4 (&acc)[8][RT], int lo, int hi, int w) const {
  constexpr int STEP = sizeof(T) == 2 ? 32 : 4;        // rows of a wave and step
  int m0 = lo + STEP * w;
  if (P >= 8) {
    if constexpr (sizeof(T) == 4) {
      for (; m0 + 12 * STEP + STEP <= hi; m0 += 16 * STEP) {                   // the loads of four steps in flight
#pragma unroll
        for (int u = 0; u < 4; ++u) group<true>(acc, m0 + 4 * STEP * u, hi);
      }
    }
    for (; m0 + STEP <= hi; m0 += 4 * STEP) group<true>(acc, m0, hi);
  }
  for (; m0 < hi; m0 += 4 * STEP) group<false>(acc, m0, hi);
}

// first of the eight columns of a lane: the last lanes of a row share its last eight (they come to the same bits)
__device__ __forceinline__ int outer_col(int P, int pb, int l16) {
  const int p = pb * OU_COLS + 8 * l16;
  return p + 8 <= P || P < 8 ? p : P - 8;
}

// one job of the sums: dA (X = x, t = u) or dB (X = dy, t = t)
struct Outer {
  const void* X;
  long long ldx;
  int P;                   // columns
  const float* t;
  int ldt;
  void* out;               // element (a, p, i) at a * oa + p * op + i * oi
  long long oa, op, oi;
  float* part;             // [slot][column block][rank chunk][tile (j, i)][lane] f32x4
  int blocks;              // column blocks
  int drop;
  float factor;
};

template <int RT> __device__ __forceinline__ size_t part_at(const Outer& o, int slot, int pb, int rc, int chunks) {
  return (((size_t)slot * o.blocks + pb) * chunks + rc) * (8 * RT * 64);
}

// value q of tile (j, i) in `lane`: column outer_col(4 (lane / 16) + q) + j, rank ib + 16 i + lane % 16
template <typename T, int RT>
__device__ __forceinline__ void outer_store(const Outer& o, f32x4 v, int tile, int lane, int a, int pb, int ib, int rank) {
  const int j = tile / RT, i = ib + 16 * (tile % RT) + (lane & 15);
  if (i >= rank) return;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int p = outer_col(o.P, pb, 4 * (lane >> 4) + q) + j;
    if (p < o.P) static_cast<T*>(o.out)[a * o.oa + p * o.op + i * o.oi] = (T)(v[q] * o.factor);
  }
}

// partial sums of a run of rows, one slot for each (run, request) pair: run + request numbers it, for a step to the next pair
// raises one of the two
template <typename T, int RT>
__device__ __forceinline__ void outer_run(const Outer& o, const Segs& sg, const KeepArgs& ka, int rank, int rows_per_run, f32x4 (*red)[8][64]) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, l16 = lane & 15;
  const int pb = blockIdx.x, run = blockIdx.y, chunks = (rank + 63) / 64;
  const int r0 = run * rows_per_run, r1 = sg.M - r0 < rows_per_run ? sg.M : r0 + rows_per_run;
  int q = seg_find(sg, r0);
  for (q = q < 0 ? 0 : q; q < sg.S && sg.row_start[q] < r1; ++q) {
    const Span sp = seg_span(sg, q, r0, r1);
    if (sp.a < 0) continue;
    for (int rc = 0; rc < chunks; ++rc) {
      f32x4 acc[8][RT];
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < RT; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
      OuterSum<T, RT>(static_cast<const T*>(o.X), o.ldx, o.P, o.t, o.ldt, 64 * rc, outer_col(o.P, pb, l16), lane, o.drop != 0, ka)
          .rows(acc, sp.lo, sp.hi, w);
      f32x4* to = reinterpret_cast<f32x4*>(o.part) + part_at<RT>(o, run + q, pb, rc, chunks);
#pragma unroll
      for (int i = 0; i < RT; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) red[w][j][lane] = acc[j][i];
        __syncthreads();
        for (int j = w; j < 8; j += 4)
          to[(j * RT + i) * 64 + lane] = (red[0][j][lane] + red[1][j][lane]) + (red[2][j][lane] + red[3][j][lane]);
        __syncthreads();
      }
    }
  }
}

template <typename T, int RT>
__global__ __launch_bounds__(256) void k_outer(Outer oa, Outer ob, Segs sg, KeepArgs ka, int rank, int rows_per_run) {
  __shared__ f32x4 red[4][8][64];
  const Outer& o = blockIdx.z == 0 ? oa : ob;
  if ((int)blockIdx.x >= o.blocks) return;
  outer_run<T, RT>(o, sg, ka, rank, rows_per_run, red);
}

// requests of an adapter in ascending order, 256 looked at a time (by the first 256 threads)
struct ReqList { int n; int q[256]; };
__device__ __forceinline__ void list_requests(const Segs& sg, int a, int base, ReqList* l) {
  __shared__ int cnt[4];
  const int q = base + threadIdx.x, w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const bool is = w < 4 && q < sg.S && sg.adapter[q] == a && sg.row_start[q] < sg.row_start[q + 1];
  const unsigned long long b = __ballot(is);
  __syncthreads();                                     // the list of the last step is read
  if (lane == 0 && w < 4) cnt[w] = __popcll(b);
  __syncthreads();
  int at = 0;
  for (int i = 0; i < 4; ++i) at += i < w ? cnt[i] : 0;
  if (is) l->q[at + __popcll(b & ((1ull << lane) - 1))] = q;
  if (threadIdx.x == 0) l->n = cnt[0] + cnt[1] + cnt[2] + cnt[3];
  __syncthreads();
}

// n <= 8 values side by side
template <typename T> struct alignas(sizeof(T)) Eight { T v[8]; };
template <typename T> __device__ __forceinline__ void store_eight(T* o, const float (&v)[8], int n) {
  Eight<T> u;
#pragma unroll
  for (int j = 0; j < 8; ++j) u.v[j] = (T)v[j];
  if (n >= 8) {
    *reinterpret_cast<Eight<T>*>(o) = u;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) if (j < n) o[j] = u.v[j];
  }
}

// sums the slots of an adapter, in order of requests and runs: their numbers are listed first, so that many loads are under way.
// 128 columns x 16 ranks a workgroup, results out through the LDS: as the products lie, each would be a store of its own
constexpr int SLOTS = 2048;
template <typename T, int RT>
__global__ __launch_bounds__(512) void k_outer_sum(Outer oa, Outer ob, Segs sg, int rank, int rows_per_run) {
  __shared__ ReqList list;
  __shared__ int slot[SLOTS], total[2][256];
  __shared__ float sums[16][OU_COLS + 1];
  const Outer& o = blockIdx.z == 0 ? oa : ob;
  const int chunks = (rank + 63) / 64, parts = RT;    // eight tiles a workgroup, one a wave
  const int a = blockIdx.y, per = o.blocks * chunks * parts;
  if ((int)blockIdx.x >= per) return;
  const int pb = blockIdx.x / (chunks * parts), rc = blockIdx.x / parts % chunks, i16 = blockIdx.x % parts;
  const int lane = threadIdx.x & 63, tid = threadIdx.x, w = tid >> 6;
  const f32x4* at = reinterpret_cast<const f32x4*>(o.part) + part_at<RT>(o, 0, pb, rc, chunks) + (w * RT + i16) * 64 + lane;
  const size_t step = part_at<RT>(o, 1, 0, 0, chunks);
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int base = 0; base < sg.S; base += 256) {
    list_requests(sg, a, base, &list);
    // runs of request `tid` of the list, and how many come before
    int first = 0, count = 0;
    if (tid < list.n) {
      const int q = list.q[tid], lo = sg.row_start[q] > 0 ? sg.row_start[q] : 0, hi = sg.row_start[q + 1] < sg.M ? sg.row_start[q + 1] : sg.M;
      if (lo < hi) { first = lo / rows_per_run; count = (hi - 1) / rows_per_run - first + 1; }
    }
    if (tid < 256) total[0][tid] = count;
    __syncthreads();
    int now = 0;
    for (int d = 1; d < 256; d <<= 1) {
      if (tid < 256) total[now ^ 1][tid] = total[now][tid] + (tid >= d ? total[now][tid - d] : 0);
      now ^= 1;
      __syncthreads();
    }
    const int all = total[now][255], before = total[now][tid & 255] - count;
    for (int b0 = 0; b0 < all; b0 += SLOTS) {
      for (int i = 0; i < count; ++i)
        if (before + i >= b0 && before + i < b0 + SLOTS) slot[before + i - b0] = first + i + list.q[tid];
      __syncthreads();
      const int n = all - b0 < SLOTS ? all - b0 : SLOTS;
      int i = 0;
      for (; i + 8 <= n; i += 8) {
        f32x4 x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = at[step * slot[i + u]];
#pragma unroll
        for (int u = 0; u < 8; ++u) v += x[u];
      }
      for (; i < n; ++i) v += at[step * slot[i]];
      __syncthreads();
    }
  }
  // value q of tile j in a lane: column 8 (4 (lane / 16) + q) + j of the block, rank lane % 16
#pragma unroll
  for (int q = 0; q < 4; ++q) sums[lane & 15][8 * (4 * (lane >> 4) + q) + w] = v[q] * o.factor;
  __syncthreads();
  if (tid >= 256) return;
  const int r0 = 64 * rc + 16 * i16;
  float u[8];
  if (o.op == 1) {                                    // columns side by side: a thread takes eight of a rank
    const int r = tid >> 4, c = tid & 15, p = outer_col(o.P, pb, c);
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = sums[r][8 * c + j];
    if (r0 + r < rank) store_eight(static_cast<T*>(o.out) + a * o.oa + p + (r0 + r) * o.oi, u, o.P - p);
  } else {                                            // ranks side by side: eight of a column
    const int col = tid >> 1, r = 8 * (tid & 1), p = outer_col(o.P, pb, col >> 3) + (col & 7);
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = sums[r + j][col];
    if (p < o.P) store_eight(static_cast<T*>(o.out) + a * o.oa + p * o.op + r0 + r, u, rank - r0 - r);
  }
}

// the same without partial sums, for so many requests that their slots would not fit: a workgroup sums all rows of an adapter
template <typename T, int RT>
__global__ __launch_bounds__(256) void k_outer_direct(Outer oa, Outer ob, Segs sg, KeepArgs ka, int rank) {
  __shared__ ReqList list;
  __shared__ f32x4 red[4][8][64];
  const Outer& o = blockIdx.z == 0 ? oa : ob;
  const int chunks = (rank + 63) / 64, a = blockIdx.y, pb = blockIdx.x / chunks, ib = 64 * (blockIdx.x % chunks);
  if (pb >= o.blocks) return;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, l16 = lane & 15;
  f32x4 acc[8][RT];
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int i = 0; i < RT; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int base = 0; base < sg.S; base += 256) {
    list_requests(sg, a, base, &list);
    for (int e = 0; e < list.n; ++e) {
      const int q = list.q[e];
      const int lo = sg.row_start[q] > 0 ? sg.row_start[q] : 0, hi = sg.row_start[q + 1] < sg.M ? sg.row_start[q + 1] : sg.M;
      OuterSum<T, RT>(static_cast<const T*>(o.X), o.ldx, o.P, o.t, o.ldt, ib, outer_col(o.P, pb, l16), lane, o.drop != 0, ka)
          .rows(acc, lo, hi, w);
    }
  }
#pragma unroll
  for (int i = 0; i < RT; ++i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) red[w][j][lane] = acc[j][i];
    __syncthreads();
    for (int j = w; j < 8; j += 4)
      outer_store<T, RT>(o, (red[0][j][lane] + red[1][j][lane]) + (red[2][j][lane] + red[3][j][lane]), j * RT + i, lane, a, pb, ib, rank);
    __syncthreads();
  }
}

// ---- transposes for the backward pass, up to three in one launch: out[z][c][r] = in[z][r][c] (rows x cols), rows of out padded
// with zeros to ldo
struct Turn {
  const void* in;
  long long ldi, si;
  int rows, cols;
  void* out;
  long long ldo, so;
  int first, across, down; // first workgroup of the job, workgroups along the columns and the rows
};
struct Turns { Turn job[3]; int n, blocks; };

template <typename T> __global__ __launch_bounds__(256) void k_turn(Turns all) {
  __shared__ T tile[64][66];
  const long long block = block_of_grid();
  if (block >= all.blocks) return;
  int at = 0;
  while (at + 1 < all.n && (int)block >= all.job[at + 1].first) ++at;
  const Turn& jb = all.job[at];
  const int id = (int)block - jb.first, bx = id % jb.across, by = id / jb.across % jb.down, z = id / (jb.across * jb.down);
  const T* i = static_cast<const T*>(jb.in) + z * jb.si;
  T* o = static_cast<T*>(jb.out) + z * jb.so;
  const int c0 = bx * 64, r0 = by * 64, x = (threadIdx.x & 7) * 8, y = threadIdx.x >> 3;    // eight values a thread
#pragma unroll
  for (int j = y; j < 64; j += 32) {
    const int n = r0 + j < jb.rows ? jb.cols - c0 - x : 0;
    const T* p = i + (r0 + j) * jb.ldi + c0 + x;
    Frag8<T> f;
    if (n >= 8) f = frag_load(p);
    else f = frag_load(p, n);
#pragma unroll
    for (int e = 0; e < 8; ++e) tile[j][x + e] = f.v[e];
  }
  __syncthreads();
#pragma unroll
  for (int j = y; j < 64; j += 32) {
    if (c0 + j < jb.cols && r0 + x < jb.ldo) {         // ldo is a multiple of eight
      Pack8<T> u;
#pragma unroll
      for (int e = 0; e < 8; ++e) u.v[e] = tile[x + e][j];
      *reinterpret_cast<Pack8<T>*>(o + (c0 + j) * jb.ldo + r0 + x) = u;
    }
  }
}

// ---- host side

int pad8(int v) { return (v + 7) & ~7; }
size_t up256(size_t v) { return (v + 255) & ~size_t(255); }
size_t type_size(int type) { return type == HM_TYPE_F32 ? 4 : 2; }

struct Plan {
  int rt, chunks, rows_per_run, runs, direct;
  long long npad, rpad;
  size_t wt, bt, at, u, pa, pb, total;       // offsets into the workspace
};

constexpr size_t MAX_PART = size_t(512) << 20;

Plan make_plan(const hm_adapter_args& g) {
  Plan p;
  p.rt = g.rank <= 16 ? 1 : g.rank <= 32 ? 2 : 4;
  p.chunks = (g.rank + 63) / 64;
  const int ba = (g.k + OU_COLS - 1) / OU_COLS, bb = (g.n + OU_COLS - 1) / OU_COLS, blocks = ba > bb ? ba : bb;
  // about 1024 workgroups for each of the two sums (a CU holds three), a quarter of that for ranks over 32 (a CU holds one, and a
  // run's partial sums are as large as 512 of its rows), runs of at least 64 rows
  long long runs = (1024 / p.rt + blocks - 1) / blocks, most = (g.rows + 63) / 64;
  runs = runs < most ? runs : most;
  if (runs < 1) runs = 1;
  long long per = (g.rows + runs - 1) / runs;
  per = (per + 15) & ~15ll;
  if (per < 16) per = 16;
  p.rows_per_run = (int)per;
  p.runs = (int)((g.rows + per - 1) / per);
  p.npad = (g.n + 7) & ~7ll;
  p.rpad = pad8(g.rank);
  const size_t slot = (size_t)p.chunks * 8 * p.rt * 64 * sizeof(f32x4), slots = (size_t)p.runs + g.segments;
  p.direct = slots * slot * (ba + bb) > MAX_PART;
  size_t at = 0;
  p.wt = at; at = up256(at + (size_t)g.k * p.npad * type_size(g.type));
  p.bt = at; at = up256(at + (size_t)g.adapters * g.rank * p.npad * type_size(g.type));
  p.at = at; at = up256(at + (size_t)g.adapters * g.k * p.rpad * type_size(g.type));
  p.u = at;  at = up256(at + (size_t)g.rows * p.rpad * sizeof(float));
  p.pa = at; at = up256(at + (p.direct ? 0 : slots * slot * ba));
  p.pb = at; at = up256(at + (p.direct ? 0 : slots * slot * bb));
  p.total = at;
  return p;
}

int check_args(const char* name, const hm_adapter_args* g, KeepArgs* ka) {
  if (g == nullptr) { hm_set_error("%s: null argument", name); return -1; }
  if (g->type < HM_TYPE_F32 || g->type > HM_TYPE_BF16) { hm_set_error("%s: unknown element type %d", name, g->type); return -1; }
  if (g->rows < 0 || g->rows > HM_ADAPTER_MAX_ROWS) {
    hm_set_error("%s: %lld rows, at most %d are taken", name, g->rows, HM_ADAPTER_MAX_ROWS); return -1; }
  if (g->k < 1 || g->n < 1 || g->k > HM_ADAPTER_MAX_WIDTH || g->n > HM_ADAPTER_MAX_WIDTH) {
    hm_set_error("%s: k = %d and n = %d must be in 1 .. %d", name, g->k, g->n, HM_ADAPTER_MAX_WIDTH); return -1; }
  if (g->rank < 1 || g->rank > HM_ADAPTER_MAX_RANK) {
    hm_set_error("%s: rank %d must be in 1 .. %d", name, g->rank, HM_ADAPTER_MAX_RANK); return -1; }
  if (g->adapters < 0 || g->segments < 0 || g->adapters > HM_ADAPTER_MAX_COUNT || g->segments > HM_ADAPTER_MAX_ROWS) {
    hm_set_error("%s: %d adapters (0 .. %d) and %d requests (0 .. %d) asked for", name, g->adapters, HM_ADAPTER_MAX_COUNT, g->segments,
                 HM_ADAPTER_MAX_ROWS); return -1; }
  if (!keep_args(ka, g->p, g->seed, g->d_seed, g->tag, g->row0)) {
    hm_set_error("%s: p must be in [0, 1], got %g", name, g->p); return -1; }
  if (g->rows > 0 && (g->d_x == nullptr || g->d_w == nullptr)) { hm_set_error("%s: null argument", name); return -1; }
  if (g->adapters > 0 && g->segments > 0 &&
      (g->d_a == nullptr || g->d_b == nullptr || g->d_row_start == nullptr || g->d_adapter == nullptr)) {
    hm_set_error("%s: null argument", name); return -1; }
  if ((g->rows > 1 && g->ld_x < g->k) || (g->n > 1 && g->ld_w < g->k)) {
    hm_set_error("%s: a row stride is less than k = %d", name, g->k); return -1; }
  if (g->ld_x > HM_ADAPTER_MAX_STRIDE || g->ld_w > HM_ADAPTER_MAX_STRIDE) {
    hm_set_error("%s: a row stride is over %d", name, HM_ADAPTER_MAX_STRIDE); return -1; }
  return 0;
}

Segs segs_of(const hm_adapter_args& g) {
  return {g.d_row_start, g.d_adapter, g.d_scale, g.adapters > 0 ? g.segments : 0, g.adapters, (int)g.rows};
}

// requests of fewer than eight rows on average: a wave per row.  A matrix product of the tiled kernel would be filled to less than
// a quarter, once for each request in its 32 rows.
bool few_rows_each(const hm_adapter_args& g) { return g.rows < 8ll * g.segments; }

template <typename T>
int shrink(const hm_adapter_args& g, const T* X, long long ldx, int K, const T* R, long long ldr, long long stride_a, bool drop,
           const KeepArgs& ka, float* t, hipStream_t st) {
  const Segs sg = segs_of(g);
  const float f = drop ? ka.up : 1.f;
  if (few_rows_each(g)) {
    const long long waves = g.rows * (pad8(g.rank) / SR_RANKS);
    const dim3 grid = grid_of((waves + 3) / 4);
    if (drop) hipLaunchKernelGGL((k_shrink_rows<T, true>), grid, dim3(256), 0, st, X, ldx, K, R, ldr, stride_a, g.rank, f, sg, ka, t, pad8(g.rank));
    else hipLaunchKernelGGL((k_shrink_rows<T, false>), grid, dim3(256), 0, st, X, ldx, K, R, ldr, stride_a, g.rank, f, sg, ka, t, pad8(g.rank));
  } else {
    const dim3 grid((unsigned)((g.rows + SH_ROWS - 1) / SH_ROWS), (g.rank + SH_RANKS - 1) / SH_RANKS);
#define HM_GO(RT, NW, D) hipLaunchKernelGGL((k_shrink<T, RT, NW, D>), grid, dim3(64 * NW), 0, st, X, ldx, K, R, ldr, stride_a, g.rank, f, sg, ka, t, pad8(g.rank))
#define HM_GO_RT(RT) if (wide) { if (drop) HM_GO(RT, 8, true); else HM_GO(RT, 8, false); } else { if (drop) HM_GO(RT, 4, true); else HM_GO(RT, 4, false); }
    const bool wide = K > 8 * Lines<T>::KB;            // more than eight lines: eight waves share them instead of four
    if (g.rank <= 16) { HM_GO_RT(1) }
    else if (g.rank <= 32) { HM_GO_RT(2) }
    else { HM_GO_RT(4) }
#undef HM_GO_RT
#undef HM_GO
  }
  HM_CHECK_HIP(hipGetLastError());
  return 0;
}

// Outputs a side of a workgroup's tile: 256 (k_project_wide: whole rounds of one workgroup a CU count, the last one is as long as the
// others), 128 (two a CU) or 64 (five).  By the time that a round of each takes, in us, with s steps of 128 bytes along the reduction:
//   16 bits  wide 14 + 1.67 s a round of 256 tiles, 128: 4.7 + 1.29 s a round of 512; 64 where those of 128 would not fill the CUs once
//            (512 x 4096 x 4096: 49 against 60) or half of each would lie beside the outputs
//   fp32     wide 38 + 6.8 s a round, 64: 2.97 s a round of 1280 (128 takes as long from 2048 rows of 512 on, twice as long below)
// The rule knows neither the rank nor where requests end, so it tells the sides apart rather than the time.  Kernel times of sides
// 256 / 128 / 64 (fp32: 256 / 64) with requests of equal lengths, and what the rule says of the two that it compares:
//   131072 x 512 x 512 bf16 rank 8    96 / 115 / 143 (109, 122)     8192 x 4096 x 4096 bf16 rank 64  278 / 386 / 598 (242, 351)
//   131072 x 512 x 259 bf16 rank 8    93 /  96 /  96 (109,  92)     6001 x 1024 x 4096 fp16 rank 32  106 /  97 / 127 ( 81,  76)
//    65536 x 512 x 253 fp16 rank 16   35 /  40 /  48 ( 27,  32)    52000 x 512 x 512 bf16 rank 16     60 /  52 /  60 ( 55,  50)
//    65536 x 512 x 512 fp32 rank 16  302 / 320       (294, 309)    32768 x 512 x 512 fp32 rank 4     141 / 155       (147, 157)
// Requests that end inside tiles cost the wide tile most: 65536 x 512 x 253 takes 55 us then, 65536 x 512 x 512 fp32 339.
int pick_tile(long long rows, int n, int k, int size) {
  auto tiles = [&](int t) { return ((rows + t - 1) / t) * ((n + t - 1) / t); };
  const int line = 128 / size;
  const double s = (k + line - 1) / line, rounds = (double)((tiles(256) + 255) / 256);
  double wide, other;
  int small;
  if (size == 2) {
    wide = rounds * (14 + 1.67 * s);
    const double r = tiles(128) / 512.0;
    other = (r < 1 ? 1 : r) * (4.7 + 1.29 * s) + 2;
    small = tiles(128) < 256 || n <= 64 ? 64 : 128;
  } else {
    wide = rounds * (38 + 6.8 * s);
    const double r = tiles(64) / 1280.0;
    other = (r < 1 ? 1 : r) * 2.97 * s + 5;
    small = 64;
  }
  return k >= line && tiles(256) >= 64 && wide < other ? 256 : small;
}

int g_tile = 0;            // hm_debug_set_adapter_tile

template <typename T> int tile_of(long long rows, int Nn, int Kk) {
  if (g_tile != 0 && (g_tile != WIDE || Kk >= Lines<T>::KB)) return g_tile == 128 && sizeof(T) == 4 ? 64 : g_tile;
  return pick_tile(rows, Nn, Kk, sizeof(T));
}

// Tiles of 64 or 128 are a workgroup of 256 threads each, of which a launch takes fewer than 2^32 along a dimension: 2^36 fp32 outputs
// (275 GB) of a short reduction come to more, and are refused before anything is launched.
template <typename T> int check_tiles(const char* name, long long rows, int Nn, int Kk) {
  const int tile = tile_of<T>(rows, Nn, Kk);
  if (tile != WIDE && ((rows + tile - 1) / tile) * ((Nn + tile - 1) / tile) >= 1ll << 24) {
    hm_set_error("%s: %lld x %d outputs are too many for one call", name, rows, Nn); return -1; }
  return 0;
}

template <typename T>
int project(const hm_adapter_args& g, const T* X, long long ldx, int Kk, const T* W, long long ldw, int Nn, const T* bias,
            const LowRank& lr, bool drop, const KeepArgs& ka, T* out, long long ldo, hipStream_t st) {
  const Segs sg = segs_of(g);
#define HM_GO(BM, BN, WGM, WGN, D)                                                                                                   \
  hipLaunchKernelGGL((k_project<T, BM, BN, WGM, WGN, D>), dim3((unsigned)(((g.rows + BM - 1) / BM) * ((Nn + BN - 1) / BN))),         \
                     dim3(64 * WGM * WGN), 0, st, X, ldx, Kk, W, ldw, Nn, bias, lr, sg, ka, out, ldo, (Nn + BN - 1) / BN)
  const int tile = tile_of<T>(g.rows, Nn, Kk);
  if (tile == WIDE) {
    const int tm = (int)((g.rows + WIDE - 1) / WIDE), tn = (Nn + WIDE - 1) / WIDE;
    const dim3 grid((long long)tm * tn < 256 ? tm * tn : 256);
    if (drop) hipLaunchKernelGGL((k_project_wide<T, true>), grid, dim3(256), 0, st, X, ldx, Kk, W, ldw, Nn, bias, lr, sg, ka, out, ldo, tm, tn);
    else hipLaunchKernelGGL((k_project_wide<T, false>), grid, dim3(256), 0, st, X, ldx, Kk, W, ldw, Nn, bias, lr, sg, ka, out, ldo, tm, tn);
  } else if (tile == 128) {
    if constexpr (sizeof(T) == 2) { if (drop) HM_GO(128, 128, 2, 2, true); else HM_GO(128, 128, 2, 2, false); }
  } else {
    if (drop) HM_GO(64, 64, 2, 2, true); else HM_GO(64, 64, 2, 2, false);
  }
#undef HM_GO
  HM_CHECK_HIP(hipGetLastError());
  return 0;
}

template <typename T> int forward(const hm_adapter_args& g, const KeepArgs& ka, void* d_y, long long ld_y, float* d_t, hipStream_t st) {
  const T *X = static_cast<const T*>(g.d_x), *W = static_cast<const T*>(g.d_w), *A = static_cast<const T*>(g.d_a);
  const T* bias = static_cast<const T*>(g.d_bias);
  T* y = static_cast<T*>(d_y);
  const bool any = g.adapters > 0 && g.segments > 0, few = g.rows <= FEW_ROWS && g_tile == 0;
  if (!few && check_tiles<T>("hm_adapter_linear", g.rows, g.n, g.k)) return -1;
  if (any) {
    const int rc = shrink<T>(g, X, g.ld_x, g.k, A, g.k, (long long)g.rank * g.k, ka.threshold != 0, ka, d_t, st);
    if (rc) return rc;
  }
  const LowRank lr = {any ? d_t : nullptr, g.d_b, (long long)g.n * g.rank, g.rank, g.rank, pad8(g.rank)};
  if (few) {
    const dim3 grid((g.n + 15) / 16, (unsigned)((g.rows + 63) / 64));
    const Segs sg = segs_of(g);
#define HM_GO(MT) hipLaunchKernelGGL((k_project_few<T, MT>), grid, dim3(64 * FEW_WAVES), 0, st, X, g.ld_x, g.k, W, g.ld_w, g.n, bias, lr, sg, y, ld_y)
    if (g.rows <= 16) HM_GO(1);
    else if (g.rows <= 32) HM_GO(2);
    else HM_GO(4);
#undef HM_GO
    HM_CHECK_HIP(hipGetLastError());
    return 0;
  }
  return project<T>(g, X, g.ld_x, g.k, W, g.ld_w, g.n, bias, lr, false, ka, y, ld_y, st);
}

void add_turn(Turns* all, const void* in, long long ldi, long long si, int rows, int cols, void* out, long long ldo,
              long long so, int count) {
  const Turn t = {in, ldi, si, rows, cols, out, ldo, so, all->blocks, (cols + 63) / 64, (int)((ldo + 63) / 64)};
  all->job[all->n++] = t;
  all->blocks += t.across * t.down * count;           // at most 2^28 of the adapters' A and B each, 2^20 of the weight
}

template <typename T>
int backward(const hm_adapter_args& g, const KeepArgs& ka, const void* d_dy, long long ld_dy, const float* d_t, void* d_dx,
             long long ld_dx, void* d_da, void* d_db, char* ws, hipStream_t st) {
  const Plan p = make_plan(g);
  const T *X = static_cast<const T*>(g.d_x), *W = static_cast<const T*>(g.d_w), *dy = static_cast<const T*>(d_dy);
  T *wt = reinterpret_cast<T*>(ws + p.wt), *bt = reinterpret_cast<T*>(ws + p.bt), *at = reinterpret_cast<T*>(ws + p.at);
  float* u = reinterpret_cast<float*>(ws + p.u);
  const bool any = g.adapters > 0 && g.segments > 0 && g.rows > 0;
  const bool want_u = any && (d_dx != nullptr || d_da != nullptr), want_dx = d_dx != nullptr && g.rows > 0;
  if (want_dx && check_tiles<T>("hm_adapter_linear_backward", g.rows, g.k, g.n)) return -1;
  Turns turns = {};
  if (want_u) add_turn(&turns, g.d_b, g.rank, (long long)g.n * g.rank, g.n, g.rank, bt, p.npad, g.rank * p.npad, g.adapters);
  if (want_dx) add_turn(&turns, W, g.ld_w, 0, g.n, g.k, wt, p.npad, 0, 1);
  if (want_dx && any) add_turn(&turns, g.d_a, g.k, (long long)g.rank * g.k, g.rank, g.k, at, p.rpad, g.k * p.rpad, g.adapters);
  if (turns.n > 0) {
    hipLaunchKernelGGL((k_turn<T>), grid_of(turns.blocks), dim3(256), 0, st, turns);
    HM_CHECK_HIP(hipGetLastError());
  }
  int rc;
  if (want_u && (rc = shrink<T>(g, dy, ld_dy, g.n, bt, p.npad, g.rank * p.npad, false, ka, u, st))) return rc;
  if (want_dx) {
    const LowRank lr = {any ? u : nullptr, at, g.k * p.rpad, p.rpad, g.rank, pad8(g.rank)};
    if ((rc = project<T>(g, dy, ld_dy, g.n, wt, p.npad, g.k, nullptr, lr, ka.threshold != 0, ka, static_cast<T*>(d_dx), ld_dx, st))) return rc;
  }
  if (g.adapters > 0 && (d_da != nullptr || d_db != nullptr)) {
    const Segs sg = segs_of(g);
    Outer oa = {X, g.ld_x, d_da != nullptr ? g.k : 0, u, pad8(g.rank), d_da, (long long)g.rank * g.k, 1, g.k, reinterpret_cast<float*>(ws + p.pa),
                d_da != nullptr ? (g.k + OU_COLS - 1) / OU_COLS : 0, ka.threshold != 0, ka.up};
    Outer ob = {dy, ld_dy, d_db != nullptr ? g.n : 0, d_t, pad8(g.rank), d_db, (long long)g.n * g.rank, g.rank, 1, reinterpret_cast<float*>(ws + p.pb),
                d_db != nullptr ? (g.n + OU_COLS - 1) / OU_COLS : 0, 0, 1.f};
    const int blocks = oa.blocks > ob.blocks ? oa.blocks : ob.blocks;   // column blocks
#define HM_GO(RT)                                                                                                                    \
    if (p.direct) {                                                                                                                  \
      hipLaunchKernelGGL((k_outer_direct<T, RT>), dim3(blocks * p.chunks, g.adapters, 2), dim3(256), 0, st, oa, ob, sg, ka, g.rank); \
    } else {                                                                                                                         \
      if (any) hipLaunchKernelGGL((k_outer<T, RT>), dim3(blocks, p.runs, 2), dim3(256), 0, st, oa, ob, sg, ka, g.rank, p.rows_per_run); \
      hipLaunchKernelGGL((k_outer_sum<T, RT>), dim3(blocks * p.chunks * RT, g.adapters, 2), dim3(512), 0, st, oa, ob, sg, g.rank, p.rows_per_run); \
    }
    if (p.rt == 1) { HM_GO(1) } else if (p.rt == 2) { HM_GO(2) } else { HM_GO(4) }
#undef HM_GO
    HM_CHECK_HIP(hipGetLastError());
  }
  return 0;
}

}  // namespace

extern "C" void hm_debug_set_adapter_tile(int tile) { g_tile = tile == 64 || tile == 128 || tile == WIDE ? tile : 0; }

extern "C" int hm_adapter_linear(const hm_adapter_args* g, void* d_y, long long ld_y, float* d_t, void* stream) {
  KeepArgs ka;
  const int rc = check_args("hm_adapter_linear", g, &ka);
  if (rc) return rc;
  if (g->rows == 0) return 0;
  if (d_y == nullptr || (d_t == nullptr && g->adapters > 0 && g->segments > 0)) { hm_set_error("hm_adapter_linear: null argument"); return -1; }
  if (g->rows > 1 && ld_y < g->n) { hm_set_error("hm_adapter_linear: row stride %lld of the output is less than n = %d", ld_y, g->n); return -1; }
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (g->type == HM_TYPE_F32) return forward<float>(*g, ka, d_y, ld_y, d_t, st);
  if (g->type == HM_TYPE_F16) return forward<f16>(*g, ka, d_y, ld_y, d_t, st);
  return forward<bf16>(*g, ka, d_y, ld_y, d_t, st);
}

extern "C" long long hm_adapter_linear_backward_bytes(const hm_adapter_args* g) {
  KeepArgs ka;
  hm_adapter_args h;
  if (g != nullptr) {                                  // sizes alone count here
    h = *g;
    h.rows = 0; h.segments = 0; h.ld_x = g->k; h.ld_w = g->k;
    if (g->rows < 0 || g->rows > HM_ADAPTER_MAX_ROWS || g->segments < 0 || g->segments > HM_ADAPTER_MAX_ROWS) h.rows = -1;
  }
  if (check_args("hm_adapter_linear_backward_bytes", g != nullptr ? &h : nullptr, &ka)) return -1;
  return (long long)make_plan(*g).total;
}

extern "C" int hm_adapter_linear_backward(const hm_adapter_args* g, const void* d_dy, long long ld_dy, const float* d_t, void* d_dx,
                                          long long ld_dx, void* d_da, void* d_db, void* d_ws, long long ws_bytes, void* stream) {
  KeepArgs ka;
  const int rc = check_args("hm_adapter_linear_backward", g, &ka);
  if (rc) return rc;
  const bool any = g->rows > 0 && g->adapters > 0 && g->segments > 0;
  if ((g->rows > 0 && d_dy == nullptr) || (any && d_db != nullptr && d_t == nullptr)) {
    hm_set_error("hm_adapter_linear_backward: null argument"); return -1; }
  if (g->rows > 1 && (ld_dy < g->n || (d_dx != nullptr && ld_dx < g->k))) {
    hm_set_error("hm_adapter_linear_backward: a row stride is less than the columns"); return -1; }
  if (ld_dy > HM_ADAPTER_MAX_STRIDE) { hm_set_error("hm_adapter_linear_backward: a row stride is over %d", HM_ADAPTER_MAX_STRIDE); return -1; }
  const Plan p = make_plan(*g);
  if (d_ws == nullptr || ws_bytes < (long long)p.total) {
    hm_set_error("hm_adapter_linear_backward: workspace of %lld bytes, %lld are needed", d_ws == nullptr ? 0ll : ws_bytes, (long long)p.total); return -1; }
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(d_ws);
  if (g->type == HM_TYPE_F32) return backward<float>(*g, ka, d_dy, ld_dy, d_t, d_dx, ld_dx, d_da, d_db, ws, st);
  if (g->type == HM_TYPE_F16) return backward<f16>(*g, ka, d_dy, ld_dy, d_t, d_dx, ld_dx, d_da, d_db, ws, st);
  return backward<bf16>(*g, ka, d_dy, ld_dy, d_t, d_dx, ld_dx, d_da, d_db, ws, st);
}
