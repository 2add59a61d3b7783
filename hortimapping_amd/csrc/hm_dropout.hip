// Dropout with a mask that is never stored: y = keep ? act(x) * up : 0, keep from hm_keep.h, act the identity or ReLU (the
// reference's hidden layers are Linear -> ReLU -> dropout in training, deepsdf/networks/deep_sdf_decoder.py:96-104).
//
// Backward: identity form  dx = keep ? dy * up : 0 -- the draws are made again from the counters;
//           ReLU form      dx = y == 0 ? 0 : dy * up -- y (kept anyway: the next layer's input) is zero exactly where the
//           ReLU or the mask removed the value (up >= 1: no kept value rounds to zero), so nothing is drawn.
// A NaN passes where it is kept; where it is dropped the result is 0 (a selection, not a product with 0).
//
// One thread takes one block of eight columns (one generator call), so a row of any length starts its own blocks; odd rows
// (253 columns) are read at the alignment they have, the last block of a row in pieces of 4, 2 and 1.
//
// Bound by memory: 131072 x 512 fp32 with ReLU forward 97 us (5.5 TB/s), backward 149 us (5.4 TB/s), without ReLU 101 us either way
// (5.3); 32768 x 512 fp16 15 us (4.5).  131072 x 253 bf16, every row at another alignment: 31 to 37 us forward, 35 to 48 us
// backward with ReLU (on different cards), 30 us either way without.  (Contiguous tensors whose backward pass draws nothing could be
// taken as one long row, every access aligned; they are not.)  A generator call's ten rounds hide behind the loads: four blocks a
// thread (DR_PER) keep enough of these in flight.
#include "hm_internal.h"
#include "hm_keep.h"
#include "../../include/hortimapping_amd.h"

using namespace hm;

namespace {

constexpr int DR_THREADS = 256;
constexpr int DR_PER = 4;               // column blocks per thread

struct RowDiv { uint32_t d, m; };       // division by the blocks of a row: m = floor(2^32 / d), one correction

__device__ __forceinline__ uint32_t divide(RowDiv r, uint32_t x, uint32_t* rem) {
  uint32_t q = __umulhi(x, r.m), e = x - q * r.d;
  if (e >= r.d) { ++q; e -= r.d; }
  *rem = e;
  return q;
}

// pieces of a row's last block: n = 1 .. 7 values
template <typename T, int N> struct alignas(sizeof(T)) PackN { T v[N]; };
template <typename T, int N> __device__ __forceinline__ void load_n(float* o, const T* p) {
  const PackN<T, N> u = *reinterpret_cast<const PackN<T, N>*>(p);
#pragma unroll
  for (int j = 0; j < N; ++j) o[j] = (float)u.v[j];
}
template <typename T, int N> __device__ __forceinline__ void store_n(T* p, const float* v) {
  PackN<T, N> u;
#pragma unroll
  for (int j = 0; j < N; ++j) u.v[j] = (T)v[j];
  *reinterpret_cast<PackN<T, N>*>(p) = u;
}
// registers are indexed by constants only: the pieces sit at fixed places (4 at 0, 2 at 4, 1 at 6) and `place` says which
// columns these are
template <typename T> __device__ __forceinline__ void load_tail(float* o, const T* p, int n) {
  if (n & 4) { load_n<T, 4>(o, p); p += 4; }
  if (n & 2) { load_n<T, 2>(o + 4, p); p += 2; }
  if (n & 1) load_n<T, 1>(o + 6, p);
}
template <typename T> __device__ __forceinline__ void store_tail(T* p, const float* v, int n) {
  if (n & 4) { store_n<T, 4>(p, v); p += 4; }
  if (n & 2) { store_n<T, 2>(p, v + 4); p += 2; }
  if (n & 1) store_n<T, 1>(p, v + 6);
}
// keep bits of the columns in the places of load_tail
__device__ __forceinline__ uint32_t tail_bits(uint32_t m, int n) {
  uint32_t o = 0;
  if (n & 4) { o |= m & 15; m >>= 4; }
  if (n & 2) { o |= (m & 3) << 4; m >>= 2; }
  if (n & 1) o |= (m & 1) << 6;
  return o;
}

enum { FWD = 0, FWD_RELU = 1, BWD = 2, BWD_RELU = 3 };

template <int KIND> __device__ __forceinline__ void apply(float* v, const float* y, uint32_t keep, float up) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (KIND == BWD_RELU) { v[j] = y[j] == 0.f ? 0.f : v[j] * up; continue; }
    float a = v[j];
    if (KIND == FWD_RELU) a = a < 0.f ? 0.f : a;
    v[j] = (keep >> j) & 1 ? a * up : 0.f;
  }
}

// in: x, or dy; y: the forward's output (BWD_RELU)
template <typename T, int KIND>
__global__ __launch_bounds__(DR_THREADS) void k_dropout(const T* __restrict__ in, long long ld_in, const T* __restrict__ y,
                                                        long long ld_y, T* __restrict__ out, long long ld_out,
                                                        long long n_blocks, int cols, RowDiv rd, KeepArgs ka) {
  const long long base = (long long)blockIdx.x * (DR_THREADS * DR_PER);
  const long long row_b = base / rd.d;                                  // uniform: once per workgroup
  const uint32_t off = (uint32_t)(base - row_b * rd.d);
  const KeepKey key = keep_key(ka);
  const int tail = cols & 7;
#pragma unroll
  for (int u = 0; u < DR_PER; ++u) {
    const uint32_t i = u * DR_THREADS + threadIdx.x;
    if (base + i >= n_blocks) return;
    uint32_t cb;
    const long long row = row_b + divide(rd, off + i, &cb);
    const T* pi = in + row * ld_in + 8ll * cb;
    const T* py = KIND == BWD_RELU ? y + row * ld_y + 8ll * cb : nullptr;
    T* po = out + row * ld_out + 8ll * cb;
    float v[8] = {}, z[8] = {};
    uint32_t keep = 0xff;
    if (KIND != BWD_RELU && ka.threshold != 0) keep = keep8(ka, key, (uint64_t)row, cb);
    if (tail == 0 || cb + 1 < rd.d) {
      load8(v, pi);
      if (KIND == BWD_RELU) load8(z, py);
      apply<KIND>(v, z, keep, ka.up);
      store8(po, v);
    } else {
      load_tail(v, pi, tail);
      if (KIND == BWD_RELU) load_tail(z, py, tail);
      apply<KIND>(v, z, tail_bits(keep, tail), ka.up);
      store_tail(po, v, tail);
    }
  }
}

template <typename T>
int launch(int kind, const void* in, long long ld_in, const void* y, long long ld_y, void* out, long long ld_out,
           long long rows, int cols, const KeepArgs& ka, hipStream_t st) {
  const uint32_t nb = (uint32_t)((cols + 7ll) / 8);
  // a launch takes fewer than 2^32 threads along a dimension; rows of whole blocks would come to that at 274 GB of 16-bit values
  constexpr long long per = DR_THREADS * DR_PER, most = 0xffffffffll / DR_THREADS * per;
  if (rows > most / nb) { hm_set_error("hm_dropout: %lld x %d values are too many for one call", rows, cols); return -1; }
  const long long n_blocks = rows * nb, grid = (n_blocks + per - 1) / per;
  const RowDiv rd = {nb, nb == 1 ? 0xffffffffu : (uint32_t)((1ull << 32) / nb)};
  const T *i = static_cast<const T*>(in), *v = static_cast<const T*>(y);
  T* o = static_cast<T*>(out);
#define HM_GO(KIND) hipLaunchKernelGGL((k_dropout<T, KIND>), dim3((unsigned)grid), dim3(DR_THREADS), 0, st, i, ld_in, v, ld_y, o, \
                                       ld_out, n_blocks, cols, rd, ka)
  if (kind == FWD) HM_GO(FWD);
  else if (kind == FWD_RELU) HM_GO(FWD_RELU);
  else if (kind == BWD) HM_GO(BWD);
  else HM_GO(BWD_RELU);
#undef HM_GO
  HM_CHECK_HIP(hipGetLastError());
  return 0;
}

int dropout(const char* name, int kind, const void* in, long long ld_in, const void* y, long long ld_y, void* out,
            long long ld_out, long long rows, int cols, int type, double p, unsigned long long seed,
            const unsigned long long* d_seed, unsigned tag, unsigned long long row0, void* stream) {
  KeepArgs ka;
  if (rows < 0 || cols < 0) { hm_set_error("%s: negative size (%lld x %d)", name, rows, cols); return -1; }
  if (!keep_args(&ka, p, seed, d_seed, tag, row0)) { hm_set_error("%s: p must be in [0, 1], got %g", name, p); return -1; }
  if (type < HM_TYPE_F32 || type > HM_TYPE_BF16) { hm_set_error("%s: unknown element type %d", name, type); return -1; }
  if (rows == 0 || cols == 0) return 0;
  if (in == nullptr || out == nullptr || (kind == BWD_RELU && y == nullptr)) { hm_set_error("%s: null argument", name); return -1; }
  if (rows > 1 && (ld_in < cols || ld_out < cols || (kind == BWD_RELU && ld_y < cols))) {
    hm_set_error("%s: a row stride is less than the %d columns", name, cols); return -1; }
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (type == HM_TYPE_F32) return launch<float>(kind, in, ld_in, y, ld_y, out, ld_out, rows, cols, ka, st);
  if (type == HM_TYPE_F16) return launch<f16>(kind, in, ld_in, y, ld_y, out, ld_out, rows, cols, ka, st);
  return launch<bf16>(kind, in, ld_in, y, ld_y, out, ld_out, rows, cols, ka, st);
}

}  // namespace

extern "C" int hm_dropout(const void* d_x, long long ld_x, void* d_y, long long ld_y, long long rows, int cols, int type,
                          int relu, double p, unsigned long long seed, const unsigned long long* d_seed, unsigned tag,
                          unsigned long long row0, void* stream) {
  return dropout("hm_dropout", relu ? FWD_RELU : FWD, d_x, ld_x, nullptr, 0, d_y, ld_y, rows, cols, type, p, seed, d_seed,
                 tag, row0, stream);
}

extern "C" int hm_dropout_backward(const void* d_dy, long long ld_dy, const void* d_y, long long ld_y, void* d_dx,
                                   long long ld_dx, long long rows, int cols, int type, int relu, double p,
                                   unsigned long long seed, const unsigned long long* d_seed, unsigned tag,
                                   unsigned long long row0, void* stream) {
  return dropout("hm_dropout_backward", relu ? BWD_RELU : BWD, d_dy, ld_dy, d_y, ld_y, d_dx, ld_dx, rows, cols, type, p, seed,
                 d_seed, tag, row0, stream);
}
