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

// One warp per (row, head) of K (blockIdx.y 0) or V (1), any head size and stride.
template <typename T>
__global__ void __launch_bounds__(RW_THREADS) kv_rows_write_kernel(const KvRowsDev c, const int* rows, const T* k,
                                                                  const T* v, size_t src_stride, int n,
                                                                  unsigned* err) {
  const long long item = (long long)blockIdx.x * (RW_THREADS / 32) + (threadIdx.x >> 5);
  if (item >= (long long)n * c.n_kv) return;
  const int i = (int)(item / c.n_kv), h = (int)(item % c.n_kv), lane = threadIdx.x & 31, which = blockIdx.y;
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

__device__ __forceinline__ void dst_value(float* p, float x) { *p = x; }
__device__ __forceinline__ void dst_value(__half* p, float x) { *p = __float2half_rn(x); }

template <typename T>
__global__ void __launch_bounds__(RW_THREADS) kv_rows_read_kernel(const KvRowsDev c, const int* rows, T* k, T* v, int n,
                                                                 unsigned* err) {
  const long long item = (long long)blockIdx.x * (RW_THREADS / 32) + (threadIdx.x >> 5);
  if (item >= (long long)n * c.n_kv) return;
  const int i = (int)(item / c.n_kv), h = (int)(item % c.n_kv), lane = threadIdx.x & 31, which = blockIdx.y;
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

cudaError_t launch_kv_rows_write(const KvRowsDev& c, const int* rows, const void* k, const void* v, bool f16,
                                 size_t src_stride, int n, unsigned* err, cudaStream_t st) {
  const long long items = (long long)n * c.n_kv;
  const dim3 grid((unsigned)((items + RW_THREADS / 32 - 1) / (RW_THREADS / 32)), 2);
  if (f16)
    kv_rows_write_kernel<__half><<<grid, RW_THREADS, 0, st>>>(c, rows, static_cast<const __half*>(k),
                                                              static_cast<const __half*>(v), src_stride, n, err);
  else
    kv_rows_write_kernel<float><<<grid, RW_THREADS, 0, st>>>(c, rows, static_cast<const float*>(k),
                                                             static_cast<const float*>(v), src_stride, n, err);
  return cudaGetLastError();
}

cudaError_t launch_kv_rows_read(const KvRowsDev& c, const int* rows, void* k, void* v, bool f16, int n, unsigned* err,
                                cudaStream_t st) {
  const long long items = (long long)n * c.n_kv;
  const dim3 grid((unsigned)((items + RW_THREADS / 32 - 1) / (RW_THREADS / 32)), 2);
  if (f16)
    kv_rows_read_kernel<__half><<<grid, RW_THREADS, 0, st>>>(c, rows, static_cast<__half*>(k), static_cast<__half*>(v), n,
                                                             err);
  else
    kv_rows_read_kernel<float><<<grid, RW_THREADS, 0, st>>>(c, rows, static_cast<float*>(k), static_cast<float*>(v), n,
                                                            err);
  return cudaGetLastError();
}

cudaError_t launch_kv_rows_move(const KvRowsDev& c, const int* starts, const int* lens, const int* path,
                                const int* counts, int n_seq, int path_stride, unsigned* err, cudaStream_t st) {
  const size_t esz = c.q8 ? 1 : 2, row = (size_t)c.hd * esz;
  const dim3 grid((unsigned)n_seq, (unsigned)c.n_kv, 2);
  const size_t smem = (size_t)path_stride * row;
  // 16-byte words when every head row starts on one and is made of them
  const bool wide = ((reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v) | c.row_stride * esz |
                      c.head_stride * esz | row) & 15) == 0;
  if (wide)
    kv_rows_move_kernel<uint4><<<grid, RW_THREADS, smem, st>>>(c, starts, lens, path, counts, path_stride, err);
  else if (c.q8)
    kv_rows_move_kernel<uint8_t><<<grid, RW_THREADS, smem, st>>>(c, starts, lens, path, counts, path_stride, err);
  else
    kv_rows_move_kernel<uint16_t><<<grid, RW_THREADS, smem, st>>>(c, starts, lens, path, counts, path_stride, err);
  return cudaGetLastError();
}

}  // namespace prana
