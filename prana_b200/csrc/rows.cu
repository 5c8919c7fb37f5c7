// rows.cu -- cache rows by index: write (with int8 quantisation), read back,
// and move the accepted branch of a drafted tree up behind its context.
//
// A cache layer is K and V [positions][n_kv][hd], f16 or int8 with one f32
// scale per (position, head): value = q * scale, scale = amax / 127.  One scale
// per head row (and not per 32 values, as the weights have) is what the
// attention kernel wants: a score is scale * (integer dot), a weighted value
// (p * scale) * integer, both with the scale of the position a thread owns.
#include "internal.h"
#include "mbar.cuh"

namespace prana {

constexpr int RW_THREADS = 256;

__device__ __forceinline__ float src_value(const float* p) { return *p; }
__device__ __forceinline__ float src_value(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void dst_value(float* p, float x) { *p = x; }
__device__ __forceinline__ void dst_value(__half* p, float x) { *p = __float2half_rn(x); }

// E values from or to E consecutive elements, one access of 4 to 16 bytes
template <int E>
__device__ __forceinline__ void load_values(const float* p, float* x) {
  static_assert(E == 4, "16 bytes");
  const float4 v = __ldcs(reinterpret_cast<const float4*>(p));
  x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
}
template <int E>
__device__ __forceinline__ void load_values(const __half* p, float* x) {
  uint32_t w[E / 2];
  if constexpr (E == 8) {
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p));
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else {
    const uint2 v = __ldcs(reinterpret_cast<const uint2*>(p));
    w[0] = v.x; w[1] = v.y;
  }
#pragma unroll
  for (int i = 0; i < E / 2; i++) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <int E>
__device__ __forceinline__ void load_values(const int8_t* p, float* x) {
  uint32_t w[E / 4];
  if constexpr (E == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
#pragma unroll
  for (int i = 0; i < E; i++) x[i] = (float)(int8_t)(w[i / 4] >> (8 * (i % 4)));
}
template <int E>
__device__ __forceinline__ void store_values(float* p, const float* x) {
  static_assert(E == 4, "16 bytes");
  __stcs(reinterpret_cast<float4*>(p), make_float4(x[0], x[1], x[2], x[3]));
}
template <int E>
__device__ __forceinline__ void store_values(__half* p, const float* x) {
  uint32_t w[E / 2];
#pragma unroll
  for (int i = 0; i < E / 2; i++) {
    const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  if constexpr (E == 8) __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
  else __stcs(reinterpret_cast<uint2*>(p), make_uint2(w[0], w[1]));
}

// Write and read: a few lanes a (row, head) of K (blockIdx.y 0) or V (1), whose
// E-value pieces they take in turn, PIECES each, all of them loaded before the
// first is used.  E fills 16 bytes of the wide side (source or destination).
// Reading is bound by the bytes: 40961 rows of 8 x 128 to f32 in 66 us, 6.4 TB/s
// (a value a lane, a warp a head row: 160 us).  Quantising is bound by the
// instructions per value: from f16 54 us, 4.7 TB/s (184 us).
constexpr int RW_LANES = 8;
// A head row's two divisions and its addresses cost as much as the rounding of
// ten values: an f16 source, half the bytes, has four lanes a head row (40961 rows
// of 8 x 128: 59 us with eight, 54 with four); f32 eight (2048 rows: 6.8 against 8.7).
template <typename T>
constexpr int WR_LANES = sizeof(T) == 2 ? 4 : 8;

// round_clamp127(x * inv) of four values as bytes, from twice the quotients (a
// power of two rounds alike): to the nearest with halves away from zero is
// (n + 1) >> 1 of n = trunc(2 t) >= 0, and n >> 1 of n < 0; a NaN truncates to
// 0.  |n| <= 254 by the scale itself, and 2 inv is in f32's range, unless the scale
// is tiny: SMALL doubles the quotient and clamps.  The shifts are done on two 16-bit
// halves at once.
template <bool SMALL>
__device__ __forceinline__ uint32_t quant_bytes(const float* x, float inv) {
  uint32_t m[4];
  const float f = SMALL ? inv : 2.0f * inv;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const float t = __fmul_rn(x[e], f);
    int n = __float2int_rz(SMALL ? 2.0f * t : t);
    if (SMALL) n = min(max(n, -254), 254);
    m[e] = (uint32_t)(n + 1 + (n >> 31));
  }
  return __byte_perm(__byte_perm(m[0], m[1], 0x5410) >> 1, __byte_perm(m[2], m[3], 0x5410) >> 1, 0x6420);
}

template <typename T, bool Q8, int E, int PIECES>
__global__ void __launch_bounds__(RW_THREADS) kv_rows_write_wide(const KvRowsDev c, const int* rows, const T* k,
                                                                const T* v, size_t src_stride, int n, unsigned* err) {
  constexpr int LANES = WR_LANES<T>;
  pdl_wait();
  pdl_trigger();
  const int item = blockIdx.x * (RW_THREADS / LANES) + threadIdx.x / LANES, sub = threadIdx.x % LANES;
  const unsigned mates = ((1u << LANES) - 1u) << (threadIdx.x & 31 & ~(LANES - 1));  // this (row, head)'s lanes
  if (item >= n * c.n_kv) return;
  const int i = item / c.n_kv, h = item - i * c.n_kv;
  const bool is_v = blockIdx.y != 0;
  const int row = rows[i];
  if (row < 0) return;
  if (row >= c.positions) {
    if (sub == 0) atomicOr(err, ERR_RANGE);
    return;
  }
  const T* x = (is_v ? v : k) + (size_t)i * src_stride + (size_t)h * c.hd;
  const size_t at = (size_t)row * c.row_stride + (size_t)h * c.head_stride;
  float f[PIECES][E], amax = 0.0f;
#pragma unroll
  for (int p = 0; p < PIECES; p++) {
    const int d = (p * LANES + sub) * E;
    if (d < c.hd) {
      load_values<E>(x + d, f[p]);
    } else {
#pragma unroll
      for (int e = 0; e < E; e++) f[p][e] = 0.0f;
    }
  }
  if constexpr (!Q8) {
    __half* o = static_cast<__half*>(is_v ? c.v : c.k) + at;
#pragma unroll
    for (int p = 0; p < PIECES; p++) {
      const int d = (p * LANES + sub) * E;
      if (d < c.hd) store_values<E>(o + d, f[p]);
    }
  } else {
#pragma unroll
    for (int p = 0; p < PIECES; p++)
#pragma unroll
      for (int e = 0; e < E; e++) amax = fmaxf(amax, fabsf(f[p][e]));
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(mates, amax, o));
    const float scale = amax > 0.0f ? __fdiv_rn(amax, 127.0f) : 1.0f;
    const float inv = __fdiv_rn(1.0f, scale);
    int8_t* o = static_cast<int8_t*>(is_v ? c.v : c.k) + at;
#pragma unroll
    for (int p = 0; p < PIECES; p++) {
      const int d = (p * LANES + sub) * E;
      uint32_t w[E / 4];
#pragma unroll
      for (int e = 0; e < E; e += 4)
        w[e / 4] = scale < 1e-36f ? quant_bytes<true>(&f[p][e], inv) : quant_bytes<false>(&f[p][e], inv);
      if (d < c.hd) {
        if constexpr (E == 8) *reinterpret_cast<uint2*>(o + d) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t*>(o + d) = w[0];
      }
    }
    if (sub == 0) (is_v ? c.v_scale : c.k_scale)[(size_t)row * c.scale_row + (size_t)h * c.scale_head] = scale;
  }
}

template <typename T, bool Q8, int E, int PIECES>
__global__ void __launch_bounds__(RW_THREADS) kv_rows_read_wide(const KvRowsDev c, const int* rows, T* k, T* v, int n,
                                                               unsigned* err) {
  pdl_wait();
  pdl_trigger();
  const int item = blockIdx.x * (RW_THREADS / RW_LANES) + threadIdx.x / RW_LANES, sub = threadIdx.x % RW_LANES;
  if (item >= n * c.n_kv) return;
  const int i = item / c.n_kv, h = item - i * c.n_kv;
  const bool is_v = blockIdx.y != 0;
  const int row = rows[i];
  const bool in = row >= 0 && row < c.positions;
  if (row >= c.positions && sub == 0) atomicOr(err, ERR_RANGE);
  T* o = (is_v ? v : k) + ((size_t)i * c.n_kv + h) * c.hd;
  const size_t at = in ? (size_t)row * c.row_stride + (size_t)h * c.head_stride : 0;
  float f[PIECES][E], scale = 1.0f;
  if (Q8 && in) scale = (is_v ? c.v_scale : c.k_scale)[(size_t)row * c.scale_row + (size_t)h * c.scale_head];
#pragma unroll
  for (int p = 0; p < PIECES; p++) {
    const int d = (p * RW_LANES + sub) * E;
#pragma unroll
    for (int e = 0; e < E; e++) f[p][e] = 0.0f;
    if (in && d < c.hd) {
      if constexpr (Q8) load_values<E>(static_cast<const int8_t*>(is_v ? c.v : c.k) + at + d, f[p]);
      else load_values<E>(static_cast<const __half*>(is_v ? c.v : c.k) + at + d, f[p]);
    }
  }
#pragma unroll
  for (int p = 0; p < PIECES; p++) {
    const int d = (p * RW_LANES + sub) * E;
    if (Q8 && in) {
#pragma unroll
      for (int e = 0; e < E; e++) f[p][e] = __fmul_rn(f[p][e], scale);
    }
    if (d < c.hd) store_values<E>(o + d, f[p]);
  }
}

// Head sizes that are no whole number of pieces, and rows that do not start on
// one: a warp a (row, head), a value a lane.
template <typename T>
__global__ void __launch_bounds__(RW_THREADS) kv_rows_write_kernel(const KvRowsDev c, const int* rows, const T* k,
                                                                  const T* v, size_t src_stride, int n,
                                                                  unsigned* err) {
  pdl_wait();
  pdl_trigger();
  const int item = blockIdx.x * (RW_THREADS / 32) + (threadIdx.x >> 5);
  if (item >= n * c.n_kv) return;
  const int i = item / c.n_kv, h = item % c.n_kv, lane = threadIdx.x & 31, which = blockIdx.y;
  const int row = rows[i];
  if (row < 0) return;
  if (row >= c.positions) {
    if (lane == 0) atomicOr(err, ERR_RANGE);
    return;
  }
  const T* x = (which ? v : k) + (size_t)i * src_stride + (size_t)h * c.hd;
  const size_t at = (size_t)row * c.row_stride + (size_t)h * c.head_stride;
  if (!c.q8) {
    __half* o = static_cast<__half*>(which ? c.v : c.k) + at;
    for (int d = lane; d < c.hd; d += 32) o[d] = __float2half_rn(src_value(x + d));
    return;
  }
  float amax = 0.0f;
  for (int d = lane; d < c.hd; d += 32) amax = fmaxf(amax, fabsf(src_value(x + d)));
  amax = warp_max(amax);
  const float scale = amax > 0.0f ? __fdiv_rn(amax, 127.0f) : 1.0f;
  const float inv = __fdiv_rn(1.0f, scale);
  int8_t* o = static_cast<int8_t*>(which ? c.v : c.k) + at;
  for (int d = lane; d < c.hd; d += 32) o[d] = (int8_t)round_clamp127(__fmul_rn(src_value(x + d), inv));
  if (lane == 0) (which ? c.v_scale : c.k_scale)[(size_t)row * c.scale_row + (size_t)h * c.scale_head] = scale;
}

template <typename T>
__global__ void __launch_bounds__(RW_THREADS) kv_rows_read_kernel(const KvRowsDev c, const int* rows, T* k, T* v, int n,
                                                                 unsigned* err) {
  pdl_wait();
  pdl_trigger();
  const int item = blockIdx.x * (RW_THREADS / 32) + (threadIdx.x >> 5);
  if (item >= n * c.n_kv) return;
  const int i = item / c.n_kv, h = item % c.n_kv, lane = threadIdx.x & 31, which = blockIdx.y;
  const int row = rows[i];
  T* o = (which ? v : k) + ((size_t)i * c.n_kv + h) * c.hd;
  if (row < 0 || row >= c.positions) {
    for (int d = lane; d < c.hd; d += 32) dst_value(o + d, 0.0f);
    if (row >= 0 && lane == 0) atomicOr(err, ERR_RANGE);
    return;
  }
  const size_t at = (size_t)row * c.row_stride + (size_t)h * c.head_stride;
  if (!c.q8) {
    const __half* x = static_cast<const __half*>(which ? c.v : c.k) + at;
    for (int d = lane; d < c.hd; d += 32) dst_value(o + d, __half2float(x[d]));
    return;
  }
  const int8_t* x = static_cast<const int8_t*>(which ? c.v : c.k) + at;
  const float scale = (which ? c.v_scale : c.k_scale)[(size_t)row * c.scale_row + (size_t)h * c.scale_head];
  for (int d = lane; d < c.hd; d += 32) dst_value(o + d, __fmul_rn((float)x[d], scale));
}

// Block (sequence, head, K | V): every row of the branch into shared memory,
// then to its new place, so that rows may move over one another.
template <typename W>
__global__ void __launch_bounds__(RW_THREADS) kv_rows_move_kernel(const KvRowsDev c, const int* starts, const int* lens,
                                                                 const int* path, const int* counts, int path_stride,
                                                                 unsigned* err) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ __align__(16) uint8_t stage[];
  __shared__ float scales[TREE_MAX_NODES];
  const int b = blockIdx.x, h = blockIdx.y, which = blockIdx.z;
  const int count = counts[b];
  const long long base = (long long)starts[b] + lens[b];
  if (count < 0 || count > path_stride || starts[b] < 0 || lens[b] < 0 || base + count > c.positions) {
    if (threadIdx.x == 0) atomicOr(err, ERR_RANGE);
    return;
  }
  const int words = c.hd * (c.q8 ? 1 : 2) / (int)sizeof(W);  // of one head row
  const size_t esz = c.q8 ? 1 : 2;
  uint8_t* x = static_cast<uint8_t*>(which ? c.v : c.k);
  float* sc = which ? c.v_scale : c.k_scale;
  W* st = reinterpret_cast<W*>(stage);
  auto at = [&](long long row) { return reinterpret_cast<W*>(x + (row * c.row_stride + (size_t)h * c.head_stride) * esz); };
  auto source = [&](int i) {  // row of the branch's i-th node; -1: not a row of the cache
    const int p = path[(size_t)b * path_stride + i];
    return p < 0 || base + p >= c.positions ? -1ll : base + p;
  };
  for (int e = threadIdx.x; e < count * words; e += RW_THREADS) {
    const long long s = source(e / words);
    if (s >= 0) st[e] = at(s)[e % words];
  }
  if (c.q8)
    for (int i = threadIdx.x; i < count; i += RW_THREADS) {
      const long long s = source(i);
      if (s >= 0) scales[i] = sc[s * c.scale_row + (size_t)h * c.scale_head];
    }
  __syncthreads();
  for (int e = threadIdx.x; e < count * words; e += RW_THREADS) {
    const long long s = source(e / words);
    if (s >= 0) at(base + e / words)[e % words] = st[e];
    else atomicOr(err, ERR_RANGE);
  }
  if (c.q8)
    for (int i = threadIdx.x; i < count; i += RW_THREADS)
      if (source(i) >= 0) sc[(base + i) * c.scale_row + (size_t)h * c.scale_head] = scales[i];
}

// Every kernel here waits for the one before it and lets the next one in at once.
template <typename F>
static cudaError_t rw_launch(F fn, dim3 grid, size_t smem, cudaStream_t st, void** args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(RW_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelExC(&cfg, (const void*)fn, args);
}

// Do all head rows start on a multiple of `bytes`?
static bool cache_aligned(const KvRowsDev& c, size_t bytes) {
  const size_t esz = c.q8 ? 1 : 2;
  return ((reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v) | c.row_stride * esz | c.head_stride * esz) &
          (bytes - 1)) == 0;
}
// pieces a lane takes of a head of hd <= 256 values, as a power of two
static int rw_pieces(int hd, int e, int lanes) {
  int n = 1;
  while (n * e * lanes < hd) n *= 2;
  return n;
}

template <typename T>
static cudaError_t write_go(const KvRowsDev& c, const int* rows, const T* k, const T* v, size_t src_stride, int n,
                            unsigned* err, cudaStream_t st) {
  constexpr int E = 16 / sizeof(T);
  const long long items = (long long)n * c.n_kv;
  KvRowsDev cc = c;
  void* args[] = {&cc, &rows, &k, &v, &src_stride, &n, &err};
  const bool wide = c.hd % E == 0 && cache_aligned(c, c.q8 ? E : E * 2) &&
                    ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | src_stride * sizeof(T)) & 15) == 0;
  if (!wide)
    return rw_launch(kv_rows_write_kernel<T>, dim3((unsigned)((items + RW_THREADS / 32 - 1) / (RW_THREADS / 32)), 2), 0, st, args);
  const dim3 grid((unsigned)((items + RW_THREADS / WR_LANES<T> - 1) / (RW_THREADS / WR_LANES<T>)), 2);
#define GO(P) (c.q8 ? rw_launch(kv_rows_write_wide<T, true, E, P>, grid, 0, st, args) \
                    : rw_launch(kv_rows_write_wide<T, false, E, P>, grid, 0, st, args))
  switch (rw_pieces(c.hd, E, WR_LANES<T>)) {
    case 1: return GO(1);
    case 2: return GO(2);
    case 4: return GO(4);
    default: return GO(8);
  }
#undef GO
}

cudaError_t launch_kv_rows_write(const KvRowsDev& c, const int* rows, const void* k, const void* v, bool f16,
                                 size_t src_stride, int n, unsigned* err, cudaStream_t st) {
  if (f16) return write_go(c, rows, static_cast<const __half*>(k), static_cast<const __half*>(v), src_stride, n, err, st);
  return write_go(c, rows, static_cast<const float*>(k), static_cast<const float*>(v), src_stride, n, err, st);
}

template <typename T>
static cudaError_t read_go(const KvRowsDev& c, const int* rows, T* k, T* v, int n, unsigned* err, cudaStream_t st) {
  constexpr int E = 16 / sizeof(T);
  const long long items = (long long)n * c.n_kv;
  KvRowsDev cc = c;
  void* args[] = {&cc, &rows, &k, &v, &n, &err};
  const bool wide = c.hd % E == 0 && cache_aligned(c, c.q8 ? E : E * 2) &&
                    ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
  if (!wide)
    return rw_launch(kv_rows_read_kernel<T>, dim3((unsigned)((items + RW_THREADS / 32 - 1) / (RW_THREADS / 32)), 2), 0, st, args);
  const dim3 grid((unsigned)((items + RW_THREADS / RW_LANES - 1) / (RW_THREADS / RW_LANES)), 2);
#define GO(P) (c.q8 ? rw_launch(kv_rows_read_wide<T, true, E, P>, grid, 0, st, args) \
                    : rw_launch(kv_rows_read_wide<T, false, E, P>, grid, 0, st, args))
  switch (rw_pieces(c.hd, E, RW_LANES)) {
    case 1: return GO(1);
    case 2: return GO(2);
    case 4: return GO(4);
    default: return GO(8);
  }
#undef GO
}

cudaError_t launch_kv_rows_read(const KvRowsDev& c, const int* rows, void* k, void* v, bool f16, int n, unsigned* err,
                                cudaStream_t st) {
  if (f16) return read_go(c, rows, static_cast<__half*>(k), static_cast<__half*>(v), n, err, st);
  return read_go(c, rows, static_cast<float*>(k), static_cast<float*>(v), n, err, st);
}

cudaError_t launch_kv_rows_move(const KvRowsDev& c, const int* starts, const int* lens, const int* path,
                                const int* counts, int n_seq, int path_stride, unsigned* err, cudaStream_t st) {
  const size_t row = (size_t)c.hd * (c.q8 ? 1 : 2);
  const dim3 grid((unsigned)n_seq, (unsigned)c.n_kv, 2);
  const size_t smem = (size_t)path_stride * row;
  KvRowsDev cc = c;
  void* args[] = {&cc, &starts, &lens, &path, &counts, &path_stride, &err};
  // 16-byte words when every head row starts on one and is made of them
  if (row % 16 == 0 && cache_aligned(c, 16)) return rw_launch(kv_rows_move_kernel<uint4>, grid, smem, st, args);
  if (c.q8) return rw_launch(kv_rows_move_kernel<uint8_t>, grid, smem, st, args);
  return rw_launch(kv_rows_move_kernel<uint16_t>, grid, smem, st, args);
}

}  // namespace prana
