// tree.cu -- attention of drafted tokens over a cache of rows.
//
// Sequence b owns the rows from starts[b]: len context rows every node sees,
// then one row per drafted node.  Node i (query row offsets[b] + i), head h:
//   s_j = q . k_j / sqrt(hd) over the context and the nodes in its mask,
//   out = sum_j exp(s_j - max) v_j / sum_j exp(s_j - max)   (zeros: nothing seen)
// A place that a node does not see takes no part, whatever it holds.
#include "internal.h"
#include "mbar.cuh"

namespace prana {

// Sequence b's rows and nodes; n = 0 (and the error word) when they do not fit
// the cache, the query rows or max_nodes.
struct TreeSeq {
  int start, len, n, off;
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs& a, int b) {
  TreeSeq s{a.starts[b], a.lens[b], 0, a.offsets[b]};
  const int n = a.offsets[b + 1] - s.off;
  const bool ok = s.start >= 0 && s.len >= 0 && s.off >= 0 && n >= 0 && n <= a.max_nodes &&
                  (long long)s.off + n <= a.n_nodes && (long long)s.start + s.len + n <= a.c.positions;
  if (ok) s.n = n;
  return s;
}
__device__ __forceinline__ bool tree_seq_bad(const TreeArgs& a, int b, const TreeSeq& s) {
  return s.n != a.offsets[b + 1] - s.off;
}
// The nodes that node i of a sequence of n sees, as bits
__device__ __forceinline__ unsigned long long tree_mask(const TreeArgs& a, const TreeSeq& s, int i) {
  const unsigned long long all = s.n >= 64 ? ~0ull : (1ull << s.n) - 1;
  const unsigned long long m = a.masks ? a.masks[s.off + i] : (i >= 63 ? ~0ull : (2ull << i) - 1);
  return m & all;
}

// Any head size and stride: one block per (node, head, sequence), 128
// positions at a time; scores take a thread per position, P.V a thread per dim.
constexpr int TR_THREADS = 128;

template <bool Q8>
__global__ void __launch_bounds__(TR_THREADS) tree_simple_kernel(const TreeArgs a) {
  __shared__ float q_s[256], p_s[TR_THREADS], red[TR_THREADS / 32];
  const int b = blockIdx.x, head = blockIdx.y, i = blockIdx.z, tid = threadIdx.x, lane = tid & 31, wi = tid >> 5;
  const TreeSeq s = tree_seq(a, b);
  if (i == 0 && head == 0 && tid == 0 && tree_seq_bad(a, b, s)) atomicOr(a.err, ERR_RANGE);
  if (i >= s.n) return;
  const int kvh = head / (a.n_heads / a.c.n_kv), hd = a.c.hd;
  const size_t row_q = (size_t)(s.off + i) * a.n_heads * hd + (size_t)head * hd;
  for (int d = tid; d < hd; d += TR_THREADS) q_s[d] = a.q[row_q + d];
  const unsigned long long mask = tree_mask(a, s, i);
  const float scale = 1.0f / sqrtf((float)hd);
  float m = -INFINITY, l = 0.0f, o[2] = {0.0f, 0.0f};
  const int total = s.len + s.n;
  auto value = [&](const void* x, size_t at) {
    return Q8 ? (float)static_cast<const int8_t*>(x)[at] : __half2float(static_cast<const __half*>(x)[at]);
  };
  for (int t0 = 0; t0 < total; t0 += TR_THREADS) {
    __syncthreads();
    const int t = t0 + tid;
    auto seen = [&](int u) { return u < s.len || (u < total && (mask >> (u - s.len) & 1)); };
    float sc = -INFINITY;
    if (seen(t)) {
      const size_t row = (size_t)(s.start + t), at = row * a.c.row_stride + (size_t)kvh * a.c.head_stride;
      float dot = 0.0f;
      for (int d = 0; d < hd; d++) dot = fmaf(q_s[d], value(a.c.k, at + d), dot);
      if (Q8) dot *= a.c.k_scale[row * a.c.scale_row + (size_t)kvh * a.c.scale_head];
      sc = dot * scale;
    }
    float mx = warp_max(sc);
    if (lane == 0) red[wi] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float m_new = fmaxf(m, mx), ref = m_new == -INFINITY ? 0.0f : m_new;
    const float alpha = expf(m - ref);
    p_s[tid] = seen(t) ? expf(sc - ref) : 0.0f;
    m = m_new;
    __syncthreads();
    float sum = 0.0f;
    for (int u = 0; u < TR_THREADS; u++) sum += p_s[u];
    l = fmaf(l, alpha, sum);
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int d = tid + e * TR_THREADS;
      if (d >= hd) break;
      float acc = 0.0f;
      for (int u = 0; u < TR_THREADS && t0 + u < total; u++) {
        if (!seen(t0 + u)) continue;
        const size_t row = (size_t)(s.start + t0 + u);
        float x = value(a.c.v, row * a.c.row_stride + (size_t)kvh * a.c.head_stride + d);
        if (Q8) x *= a.c.v_scale[row * a.c.scale_row + (size_t)kvh * a.c.scale_head];
        acc = fmaf(p_s[u], x, acc);
      }
      o[e] = fmaf(o[e], alpha, acc);
    }
  }
#pragma unroll
  for (int e = 0; e < 2; e++)
    if (tid + e * TR_THREADS < hd) a.out[row_q + tid + e * TR_THREADS] = l == 0.0f ? 0.0f : o[e] / l;
}

size_t tree_workspace_bytes(int, int, int, int, int, int) { return 256; }

cudaError_t launch_attn_tree(const TreeArgs& a, cudaStream_t st) {
  const dim3 grid((unsigned)a.n_seq, (unsigned)a.n_heads, (unsigned)a.max_nodes);
  if (a.c.q8) tree_simple_kernel<true><<<grid, TR_THREADS, 0, st>>>(a);
  else tree_simple_kernel<false><<<grid, TR_THREADS, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace prana
