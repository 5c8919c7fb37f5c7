// tree.cu -- attention of drafted tokens over a cache of rows.
//
// Sequence b owns the rows from starts[b]: len context rows every node sees,
// then one row per drafted node.  Node i (query row offsets[b] + i), head h:
//   s_j = q . k_j / sqrt(hd) over the context and the nodes in its mask,
//   out = sum_j exp(s_j - max) v_j / sum_j exp(s_j - max)   (zeros: nothing seen)
// A place that a node does not see takes no part, whatever it holds.
#include <atomic>
#include <climits>
#include <type_traits>

#include "internal.h"
#include "mbar.cuh"
#include "tc.cuh"

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
// positions at a time; scores take a thread per position, P.V a thread per dim.  o is
// kept divided by the sum, so that values near f32's largest do not pass it.
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
    const float before = l * alpha;
    l = before + sum;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
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
        acc = fmaf(p_s[u] * inv, x, acc);
      }
      o[e] = fmaf(o[e], before * inv, acc);
    }
  }
#pragma unroll
  for (int e = 0; e < 2; e++)
    if (tid + e * TR_THREADS < hd) a.out[row_q + tid + e * TR_THREADS] = o[e];
}

// ---------------------------------------------------------------- tcgen05
// Head sizes up to 128 whose rows a tensor map can describe.  The (node, head)
// pairs that share a kv head are columns; a unit of work is (sequence, kv head,
// chunk of columns), its tiles are 128 positions each, and the tiles of all
// units, in order, are dealt to the CTAs (one per SM) in equal contiguous
// shares, so ragged batches stay balanced.  A unit inside one share is finished
// there; otherwise its shares leave (max, sum, o) partials, which the CTA that is
// done last adds up, or tree_merge_kernel where there are 64 columns.
//
// Exactness.  An f16 cache: q and p enter as f16 head + remainder pairs (22
// bits), K and V as they are, sums in f32.  An int8 cache: q enters as three signed
// base-256 digits (23 bits), p as two pairs (30), and kind::i8 products take K and V as
// they lie in memory, with no conversion; every product and sum is an exact
// integer (a digit's sum over a tile stays within 2^21).  The K scale multiplies
// the score in f32.  The V scale, 2^e * m, goes with the probability: e is added to
// the score (in powers of two), so that p * 2^e, what the place adds to the
// output, is measured against a reference of the same kind, and m scales the
// digits.  The sum of the probabilities takes p * 2^e * 2^-e.  With e from TT_E_MIN to
// TT_E_MAX no weight that matters is lost on that way, a scale of 0 included (m = 0,
// e = TT_E_MIN: only where such places outweigh the rest 2^80 times, what is left of the
// rest is cut to 0).  A place whose scale lies beyond (or is no number) makes the sum NaN, and a
// column whose sum is NaN in the end, tree_column computes from the definition (8 us
// for every 32 places).
//   The reference of a column is its largest score when it was last set; it
// is set at the first tile, at tiles with drafted places, and when a later score
// passes it by more than TT_ROOM powers of two, which the digits and the f16 range
// have to spare (p = 1 keeps 23 bits).  Until then a tile needs no maximum, no
// exchange and no rescaling, and O of an int8 cache gathers in TMEM.
//   The digits' unit is 2^-23 of p = 1, and a long context may hold many places below
// half of that.  So the references of an int8 cache come down as well: they are set
// again after a tile that began them or raised one by TT_FAR (whose own digits use
// TT_SPARE of the room, which no later tile needs), and after every RUN tiles; where
// the largest score is then TT_LOW lower, to TT_ABOVE above it.  l goes to the
// columns' sums at the same times, since a thread's own sum would round small
// weights away.  (One score 18 above 16384 others, 64 columns: the error is 3e-6 of the
// large value with references that only rise, 4e-7 so.  24 trees of 60 nodes 423 and
// 450 us, 16 sequences' decode 31.8 and 32.3; a reference at each tile's largest score: 520
// us and 33.)
//
// Roles (20 warps): 16 loads K and V tiles by TMA into a ring of slots, 17 issues
// S = K . q^T (M = 128 positions), 18 issues O^T = V^T . p^T (M = dims; V is read
// MN-major as it lies, p is written position by position), 19 finds the next
// segment (and prepares its columns, up to 16), and four groups of four warps do
// the softmax, a thread per position for S and a thread per dim for O, 16 columns
// at most.  The groups form teams with a tile each: up to 16 columns four teams of
// one group, with 32 two teams of two, with 64 one team of four, whose columns
// share one product.  (A
// product of few columns costs the 4 KB of its K or V rows, 40 cycles at 32
// columns and 100 at 192: four of 48 took twice one of 192.)  The cache is so read
// once for 64 columns.
//
// What bounds it, one B200.  Decode: the cache's bytes where it is long (64
// sequences of 32000: f16 1153 us, 7.3 TB/s, int8 618 us, 7.0 TB/s with a head's
// positions adjacent and 6.0 with 128-byte rows 1 KB apart), a share's start, its
// units' ends and the joining where it is not (16 of up to 4095 int8 positions: 32
// us, 2.8 TB/s; its SMs issue 28% of their cycles).  Wide trees: the softmax (24 trees
// of 60 nodes over up to 6000: int8 450 us, f16 440; 64 columns keep 65% of the issue
// slots and 20% of the tensor cores busy).
constexpr int TT_GROUPS = 4, TT_SOFT = TT_GROUPS * 128, TT_THREADS = TT_SOFT + 128;
constexpr int TT_TMA_WARP = 16, TT_S_WARP = 17, TT_O_WARP = 18, TT_NEXT_WARP = 19;
constexpr int TT_TILE = 128;
constexpr int TT_MAX_SLOTS = 10;
constexpr float TT_DIGITS = 8355711.0f;  // 0x7f7f7f: the largest value of three balanced digits
constexpr float TT_ROOM = 6.0f;
// V scales of 8.3e-25 to 1e6: the smallest weight beside the largest is 2^-100 by
// these, and 2^-26 by the scores, in f32's range; and a sum stays below 2^(80 + 6) a place
constexpr int TT_E_MIN = -80, TT_E_MAX = 20;
// Units of the p operand for p = 1 (with m < 2): 2^6 * 2 of them stay below 2^15 *
// 0x7f7f, the largest value of its digits, 2^6 * 2^9 below f16's largest.
// With references that only rose, a room of 2^4 set them more often (24 trees of 60 nodes 447
// us against 421), and 2^8 took accuracy (an error of 1.5e-6 against 6e-7) for 1%.
template <bool Q8>
constexpr float TT_UNITS = Q8 ? 1069500000.0f / 128.0f : 512.0f;
// How far below its reference a column's largest score brings it down, and to what above the score
constexpr float TT_LOW = 8.0f, TT_ABOVE = 4.0f;
constexpr float TT_FAR = 12.0f;    // a rise after which the next tile sets the references again
constexpr float TT_SPARE = 5.0f;   // a power of two is left for the rounding of the scores
constexpr float TT_DEPTH = 24.0f;  // further below a column's largest score no reference goes: f32 sums do not show it
constexpr float LOG2E = 1.4426950408889634f;

// What a CTA leaves for tree_merge_kernel: the unit that began in it and went on
// in the next n - 1 CTAs (n = 0: none).
struct TreePart {
  int n, cols, vh0, kvh, b, pad[3];
};
struct TreeTcArgs {
  CUtensorMap tm_k, tm_v;
  TreeArgs t;
  int boxes;        // TMA boxes of a tile's K (or V): 1, or 2 for an f16 head above 64
  int slots;        // ring slots
  unsigned* tickets;  // [CTAs], zero between calls: the shares of the unit that began in a CTA that are done
  TreePart* parts;  // [CTAs]
  float2* part_ml;  // [2 * CTAs][columns] (max, sum)
  float* part_o;    // [2 * CTAs][columns][hd]
};

// NQ columns of a group, CG groups in a team
template <bool Q8, int NQ, int CG>
struct TtShape {
  static constexpr int CH = NQ * CG;                               // columns of a CTA
  static constexpr int TG = TT_GROUPS / CG;                        // teams: tiles in work at once
  // MMA columns of S and O: digit by digit, or heads and remainders
  static constexpr int N = Q8 ? (NQ == 8 ? 32 : 3 * CH) : 2 * CH, NO = Q8 ? 4 * CH : 2 * CH;
  static constexpr int CS = (N + 31) / 32 * 32, CO = (NO + 31) / 32 * 32;  // TMEM columns between accumulators
  static constexpr int TMEM = TG * (CS + CO) <= 128 ? 128 : TG * (CS + CO) <= 256 ? 256 : 512;
  static constexpr int QSZ = N * (Q8 ? 128 : 256);                  // bytes of the q operand
  static constexpr int PSZ = (4 * CH + 63) / 64 * TT_TILE * 64;     // of a team's p operand: blocks of 64 bytes a position
  static constexpr int RING = (CG < 4 ? 160 : 128) * 1024;
  static constexpr int OFF_P = RING, OFF_Q = OFF_P + TG * PSZ;
  static constexpr size_t BYTES = 1024 + OFF_Q + QSZ;
  // Who adds a unit's partials up: the CTA that is done last, which saves a launch
  // and its two waits (4 us of a call); 64 columns are more than one SM reads in
  // that time (600 KB of a 4096 context), and a kernel follows.
  static constexpr bool TICKET = CH <= 32;
  // Tiles of a team until an int8 cache's references are set in any case (O, which gathers
  // until then, has 2^21 a tile at most).  An f16 cache's are not: its p reaches down to 2^-33 of
  // the reference.  And its O gathers one tile, since the tensor core cuts sums off where
  // it does not round them (66000 positions: an error of 4.8e-6 with 31 tiles, 2.0e-6
  // with four, 6.5e-7 with one, at no cost in time).
  static constexpr int RUN = CG == 4 ? 16 : 8;
  static_assert(TG * (CS + CO) <= 512, "TMEM");
  // Warps that prepare the next segment's columns.  Up to 16 columns one warp does, while
  // the segment before ends (all softmax warps at its end: 24 sequences' decode 48.3
  // us against 45.9).  More are a chain of 8 or 16 trips to memory for that warp, which
  // nothing hides: the softmax warps do them, one trip each (24 trees of 60 nodes 421
  // us against 538).
  static constexpr int STAGERS = CG == 1 ? 1 : TT_SOFT / 32;
  // A segment's start and end, in tiles.  2 / 4 / 8 of them: 24 sequences of up to
  // 6000 int8 positions 47.9 / 45.9 / 45.1 us, 16 of 4095 f16 39.2 / 38.2 / 40.1; 24 trees
  // of 60 nodes over 6000 f16 positions 419 / 406 / 376, eight over 1000 int8 61.3 /
  // 60.7 / 66.5, where a long start leaves shares with little else.
  static constexpr int LEAD = 4;
  // tiles until V is in the same slot again; a group that waits for its V knows that
  // of its last tile has landed, and so all before
  static constexpr int turn(int slots) { return slots & 1 ? slots : slots / 2; }
  static_assert(turn(RING / 32768) >= TG && turn(RING / 16384 < TT_MAX_SLOTS ? RING / 16384 : TT_MAX_SLOTS) >= TG, "V's phases");
  static_assert(TG == 1 || PSZ >= CG * NQ * 128 * 4, "the groups' o pass through the p operand");
};

// instruction descriptors: M = 128; i8 (s32 accumulators) or f16 (f32); `mn`: both operands MN-major
template <bool Q8>
constexpr uint32_t tt_idesc(int n, bool mn) {
  const uint32_t kind = Q8 ? (2u << 4) | (1u << 7) | (1u << 10) : 1u << 4;
  return kind | (mn ? 3u << 15 : 0u) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
// MN-major operand in 64-byte swizzled atoms: blocks of 64 bytes along MN (a
// block's 128 rows are 8 KB), 8-row K groups 512 bytes apart
__device__ __forceinline__ uint64_t sw64_desc_mn(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)(8192 >> 4) << 16 | (uint64_t)(512 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)4 << 61;
}
// byte offset of 16-byte piece c of row r of such an operand
__device__ __forceinline__ int sw64(int r, int c) { return (c >> 2) * 8192 + r * 64 + (((c & 3) ^ ((r >> 1) & 3)) << 4); }

__device__ __forceinline__ float redux_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Two columns.  (The packed f32x2 instructions were slower here: they take no
// constants as operands, and the moves that bring those into register pairs cost
// more than the packing saves.)
struct F2 {
  float x, y;
  __device__ __forceinline__ F2() {}
  __device__ __forceinline__ F2(float a, float b) : x(a), y(b) {}
  __device__ __forceinline__ explicit F2(float a) : x(a), y(a) {}
  __device__ __forceinline__ float lo() const { return x; }
  __device__ __forceinline__ float hi() const { return y; }
};
__device__ __forceinline__ F2 operator+(F2 a, F2 b) { return F2(a.x + b.x, a.y + b.y); }
__device__ __forceinline__ F2 operator*(F2 a, F2 b) { return F2(a.x * b.x, a.y * b.y); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) { return F2(fmaf(a.x, b.x, c.x), fmaf(a.y, b.y, c.y)); }
// two integers in [-2^22, 2^22) as floats, without the conversion unit
__device__ __forceinline__ F2 small_ints(uint32_t a, uint32_t b) {
  return F2(__uint_as_float(a + 0x4B400000u), __uint_as_float(b + 0x4B400000u)) + F2(-12582912.0f);
}
template <int W>
__device__ __forceinline__ void tt_ld(uint32_t taddr, uint32_t* r) {
  if constexpr (W == 8) tc_ld8(taddr, r);
  else tc_ld16(taddr, r);
}
// Columns c, c + 1 of W loaded from an accumulator: the three digits' sums put together, or head + remainder
template <bool Q8, int W>
__device__ __forceinline__ F2 joined(const uint32_t* v, int c) {
  const uint32_t *v1 = v + W, *v2 = v + 2 * W;
  if constexpr (Q8) {
    const F2 k(256.0f);
    return fma2(fma2(small_ints(v[c], v[c + 1]), k, small_ints(v1[c], v1[c + 1])), k, small_ints(v2[c], v2[c + 1]));
  } else {
    return F2(__uint_as_float(v[c]), __uint_as_float(v[c + 1])) + F2(__uint_as_float(v1[c]), __uint_as_float(v1[c + 1]));
  }
}
// A bounded wait.  Once any role of the CTA has given up, every wait returns at
// once: the loops run on to their ends, so that named barriers stay matched.  A
// try may suspend, for 20 us at most, since a spinning warp takes issue slots from
// the rest; it takes 350 cycles even for a phase long over, a test 150, so that
// comes first (three of them are slower again).  The loop stays rolled: there are
// many waits, and unrolled ones cost the roles 20% in instruction fetch.
constexpr uint32_t TT_POLLS = 1u << 17;
__device__ __forceinline__ bool tt_wait(uint64_t* bar, uint32_t phase, volatile int* abort) {
  if (mbar_test_wait(bar, phase)) return true;
#pragma unroll 1
  for (uint32_t i = 0; i < TT_POLLS; i++) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(phase), "r"(20000u)
        : "memory");
    if (ok) return true;
    if (*abort) return false;
  }
  *abort = 1;
  return false;
}
__device__ __forceinline__ void group_sync(int g) { asm volatile("bar.sync %0, 128;" ::"r"(1 + g) : "memory"); }
// the OR of `pred` over the 128 * N threads of a team (barriers 7 and up)
template <int N>
__device__ __forceinline__ bool team_any(int team, bool pred) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.or.pred q, %2, %3, p;\n selp.u32 %0, 1, 0, q;\n}"
      : "=r"(r)
      : "r"((uint32_t)pred), "r"(7 + team), "n"(128 * N)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void first_sync() { asm volatile("bar.sync 6, 544;" ::: "memory"); }  // the groups and the next segments' warp
__device__ __forceinline__ void groups_sync() { asm volatile("bar.sync 5, 512;" ::: "memory"); }
__device__ __forceinline__ bool groups_any(bool pred) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.or.pred q, 5, 512, p;\n selp.u32 %0, 1, 0, q;\n}"
      : "=r"(r)
      : "r"((uint32_t)pred)
      : "memory");
  return r != 0;
}

__device__ __forceinline__ int tree_tiles(const TreeSeq& s) { return (s.len + s.n + TT_TILE - 1) / TT_TILE; }
__device__ __forceinline__ int tree_chunks(const TreeSeq& s, int group, int ch) { return (s.n * group + ch - 1) / ch; }
// A unit counts as its tiles and `lead` more in front, which stand for what
// beginning and ending it costs; a share that ends among those has none of it.
__device__ __forceinline__ unsigned long long tree_work(const TreeSeq& s, int n_kv, int group, int ch, int lead) {
  return s.n ? (unsigned long long)(tree_tiles(s) + lead) * tree_chunks(s, group, ch) * n_kv : 0ull;
}

// A CTA's walk over its share: segments of consecutive tiles of one unit.
struct TreeWalk {
  const TreeArgs* a;
  TreeSeq s;
  int b, kvh, chunk, tile, tiles, chunks, group, ch, lead;
  int left;  // of the share, this segment included
  int took;  // of the share, by this segment
  int seg;   // tiles of this segment
  // place `at` of sequence seq's work, n on from there; false: no tile among them
  __device__ __forceinline__ bool start(const TreeArgs* args, int ch_, int lead_, int seq, const TreeSeq& sq,
                                        unsigned long long at, int n) {
    a = args;
    ch = ch_;
    lead = lead_;
    group = a->n_heads / a->c.n_kv;
    b = seq;
    left = n;
    s = sq;
    tiles = tree_tiles(s);
    chunks = tree_chunks(s, group, ch);
    const int size = tiles + lead;
    unsigned long long u;
    if (at <= 0xffffffffull) {
      u = (unsigned)at / (unsigned)size;
      kvh = (int)((unsigned)u / (unsigned)chunks);
    } else {
      u = at / size;
      kvh = (int)(u / chunks);
    }
    const int place = (int)(at - u * size);
    chunk = (int)(u - (unsigned long long)kvh * chunks);
    took = min(left, size - place);
    tile = max(0, place - lead);
    seg = max(0, place + took - lead) - tile;
    return seg > 0;
  }
  __device__ __forceinline__ bool next() {  // false: the share is done
    left -= took;
    if (left <= lead) return false;
    tile = 0;
    if (++chunk == chunks) {
      chunk = 0;
      if (++kvh == a->c.n_kv) {
        kvh = 0;
        s = tree_seq(*a, ++b);
        while (!s.n && b + 1 < a->n_seq) s = tree_seq(*a, ++b);
        tiles = max(1, tree_tiles(s));
        chunks = max(1, tree_chunks(s, group, ch));
      }
    }
    took = min(left, tiles + lead);
    seg = took - lead;
    return true;
  }
  __device__ __forceinline__ bool more() const { return left - took > lead; }
};

// What the softmax groups need of a segment; places count from its first tile.
struct TreeSegment {
  int row, len, total, off;  // cache row of place 0; places all nodes see; places; first query row
  int b;                     // sequence
  int kvh, tiles;
  int before, rest;          // the unit's tiles before and after this segment
  int vh0, cols;             // the chunk's first column of the unit, and its columns
  int more;                  // another segment follows
};

// Column c of a unit whose n partials lie in the CTAs from i0: every STEP-th from
// `from` on, weighed by the maximum of all, onto x (the dims lane + 32 e); returns
// the sum of all.  The order is that of the tiles, whoever does it.
template <int STEP>
__device__ __forceinline__ float tree_add(const TreeTcArgs& ta, int ch, int c, int i0, int n, int from, int lane, int hd,
                                          float (&x)[4]) {
  auto slot = [&](int i) { return (2 * (size_t)(i0 + i) + (i == 0 ? 1 : 0)) * ch + c; };
  auto ml = [&](int i) { return i < n ? __ldcg(&ta.part_ml[slot(i)]) : make_float2(-INFINITY, 0.0f); };
  float2 f0 = ml(lane);
  float m = f0.x, sum = 0.0f;
  for (int i = lane + 32; i < n; i += 32) m = fmaxf(m, ml(i).x);
  m = warp_max(m);
  for (int ib = 0; ib < n; ib += 32) {
    if (ib) f0 = ml(ib + lane);
    const float wt = f0.x == -INFINITY ? 0.0f : ex2(f0.x - m);
    sum = fmaf(f0.y, wt, sum);
#pragma unroll 8
    for (int i = from; i < min(32, n - ib); i += STEP) {
      const float f = __shfl_sync(0xffffffffu, wt, i);
      const float* po = ta.part_o + slot(ib + i) * hd;
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (e * 32 + lane < hd) x[e] = fmaf(__ldcg(po + e * 32 + lane), f, x[e]);
    }
  }
  return warp_sum(sum);
}
// One column of an int8 cache from the definition, by a warp: for the few whose
// places' V scales the digits do not take.  A place a lane for the scores, four dims
// a lane for o, which is kept divided by the sum, so that values up to f32's
// largest do not pass it.  (Rows start on 16 bytes and are made of them.)
__device__ __noinline__ void tree_column(const TreeArgs& a, const TreeSeq& s, int kvh, int vh, int lane) {
  const int group = a.n_heads / a.c.n_kv, node = vh / group, head = kvh * group + vh % group, hd = a.c.hd;
  const size_t at = ((size_t)(s.off + node) * a.n_heads + head) * hd;
  const float* q = a.q + at;
  const unsigned long long mask = tree_mask(a, s, node);
  const float scale = 1.0f / sqrtf((float)hd);
  const int8_t *k8 = static_cast<const int8_t*>(a.c.k), *v8 = static_cast<const int8_t*>(a.c.v);
  const size_t head_at = (size_t)kvh * a.c.head_stride, scale_at = (size_t)kvh * a.c.scale_head;
  float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int t0 = 0; t0 < s.len + s.n; t0 += 32) {
    const int t = t0 + lane;
    const bool seen = t < s.len || (t < s.len + s.n && (mask >> (t - s.len) & 1));
    float sc = -INFINITY, vs = 0.0f;
    if (seen) {
      const size_t row = (size_t)(s.start + t);
      vs = a.c.v_scale[row * a.c.scale_row + scale_at];
      const uint4* k = reinterpret_cast<const uint4*>(k8 + row * a.c.row_stride + head_at);
      float dot = 0.0f;
      for (int d = 0; d < hd; d += 16) {
        const uint4 w = k[d / 16];
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 16; e++) dot = fmaf(q[d + e], (float)(int8_t)(ws[e / 4] >> (8 * (e % 4))), dot);
      }
      sc = dot * a.c.k_scale[row * a.c.scale_row + scale_at] * scale;
    }
    const float top = fmaxf(m, warp_max(sc)), ref = top == -INFINITY ? 0.0f : top;
    float p = seen ? expf(sc - ref) : 0.0f;
    const float before = l * expf(m - ref);
    m = top;
    l = before + warp_sum(p);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    p *= inv;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const unsigned all = __ballot_sync(0xffffffffu, seen);
#pragma unroll 1
    for (int u0 = 0; u0 < 32; u0 += 8) {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const size_t row = (size_t)(s.start + t0 + u0 + i);
        const bool take = lane * 4 < hd && (all >> (u0 + i) & 1);
        w[i] = take ? *reinterpret_cast<const uint32_t*>(v8 + row * a.c.row_stride + head_at + lane * 4) : 0u;
      }
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float pu = __shfl_sync(0xffffffffu, p, u0 + i), vu = __shfl_sync(0xffffffffu, vs, u0 + i);
#pragma unroll
        for (int e = 0; e < 4; e++) acc[e] = fmaf(pu, (float)(int8_t)(w[i] >> (8 * e)) * vu, acc[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = fmaf(o[e], before * inv, acc[e]);
    if (__all_sync(0xffffffffu, o[0] != o[0] && o[1] != o[1] && o[2] != o[2] && o[3] != o[3])) break;  // NaN from here on
  }
  if (lane * 4 < hd) {
#pragma unroll
    for (int e = 0; e < 4; e++) a.out[at + lane * 4 + e] = o[e];
  }
}
// A ticket of a count over CTAs: what this CTA wrote (the others' writes ordered
// before by the caller's barrier) is released, and the last to draw acquires it all.
__device__ __forceinline__ unsigned ticket_acq_rel(unsigned* counter) {
  unsigned old;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(old) : "l"(counter) : "memory");
  return old;
}

__device__ __forceinline__ TreeSegment tree_segment(const TreeWalk& w) {
  const int skip = w.tile * TT_TILE, vh0 = w.chunk * w.ch;
  return TreeSegment{w.s.start + skip, w.s.len - skip, w.s.len + w.s.n - skip, w.s.off, w.b, w.kvh, w.seg, w.tile,
                     w.tiles - w.tile - w.seg, vh0, min(w.ch, w.s.n * w.group - vh0), w.more()};
}

template <bool Q8, int NQ, int CG>
__global__ void __launch_bounds__(TT_THREADS, 1) tree_tc_kernel(const __grid_constant__ TreeTcArgs ta) {
  using S = TtShape<Q8, NQ, CG>;
  constexpr int CH = S::CH, TG = S::TG, N = S::N, CS = S::CS, CO = S::CO;
  const TreeArgs& a = ta.t;
  extern __shared__ __align__(16) uint8_t smem_dyn[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~(uintptr_t)1023);
  uint8_t* q_t = base + S::OFF_Q;
  // A waiter names a phase by its parity, so none may fall two phases behind: each
  // barrier's next phase needs the waiter's own step past the last.  (K and V use
  // a slot in turn when their number is odd, for two waiters: each has its own
  // `full`.)
  __shared__ __align__(8) uint64_t full[2][TT_MAX_SLOTS], empty[TT_MAX_SLOTS];  // full: of K, of V
  __shared__ __align__(8) uint64_t s_full[4], s_free[4], p_full[4], o_full[4], q_ready, q_free, seg_seen, seg_ready, parts0, done_s, done_o;
  __shared__ uint32_t tmem_s;
  __shared__ int s_abort;
  // a segment and its columns, in one of two sets: the nodes a column's node sees,
  // its place in the sequence's q and out rows, its score factor; and the nodes
  // some column sees
  __shared__ TreeSegment seg_tab[2];
  __shared__ int2 seg_part[2];  // the CTA where its unit began, and how many the unit went to
  __shared__ unsigned long long col_mask[2][CH], any_mask[2];
  __shared__ int col_off[2][CH];
  __shared__ __align__(16) float col_mul[2][CH];
  __shared__ __align__(16) float x_max[4][4][NQ];
  // per warp: minus a column's reference, minus its last rise, what that does to l and o
  __shared__ __align__(16) float x_m[16][NQ], x_d[16][NQ], x_al[16][NQ];
  __shared__ float4 x_col[16][NQ];             // per warp: a column's reference, its largest score, the sum so far and what that rounded away
  __shared__ int x_on[4];                      // does a team's O go onto what its accumulator holds?
  __shared__ float2 x_fin[4][NQ];              // (max, sum) of a finished segment
  __shared__ int s_nan;                        // a sum of a unit that is finished here is NaN
  __shared__ unsigned long long x_bad[4];   // drafted rows of V that are not finite
  __shared__ unsigned long long w_sum[TT_THREADS / 32], s_all;
  __shared__ int s_any;       // has the share a tile?
  __shared__ int s_merge[2];  // partials for this CTA to add up (0: not its turn), the first's CTA
  __shared__ TreeWalk s_walk;  // where the share begins
  volatile int* abort = &s_abort;

  const int tid = threadIdx.x, lane = tid & 31, wi = tid >> 5;
  const int hd = a.c.hd, n_kv = a.c.n_kv, group = a.n_heads / n_kv;
  const int slots = ta.slots, boxes = ta.boxes;
  const uint32_t slot_bytes = (uint32_t)boxes * 16384u;
  const int period = slots & 1 ? slots : slots / 2;  // tiles between two uses of a slot by K (or by V)

  if (tid < 32) {
    auto init = [&](uint64_t* bars, int n, unsigned count) {
      if (lane < n) mbar_init(bars + lane, count);
    };
    init(full[0], TT_MAX_SLOTS, 1);
    init(full[1], TT_MAX_SLOTS, 1);
    init(empty, TT_MAX_SLOTS, 1);
    init(s_full, TG, 1);
    init(s_free, TG, 128 * CG);
    init(p_full, TG, 128 * CG);
    init(o_full, TG, 1);
    if (lane == 0) {
      s_abort = 0;
      s_any = 0;
      s_nan = 0;
      any_mask[0] = any_mask[1] = 0ull;
      mbar_init(&q_ready, 32 * S::STAGERS);
      mbar_init(&q_free, 1);
      mbar_init(&seg_seen, 1);
      mbar_init(&seg_ready, 1);
      mbar_init(&parts0, 1);
      mbar_init(&done_s, 1);
      mbar_init(&done_o, 1);
    }
    fence_barrier_init();
  }
  if (tid == 32 || tid == 64)
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(tid == 32 ? &ta.tm_k : &ta.tm_v)) : "memory");
  __syncthreads();
  pdl_wait();     // what comes next reads what earlier kernels wrote
  pdl_trigger();  // the merge kernel may take its place; it waits for this grid
  if (wi == TT_S_WARP) {  // after the wait: an earlier kernel may still have needed the TMEM
    tc_alloc(&tmem_s, S::TMEM);
    tc_relinquish();
  }

  // ---- this CTA's share of the tiles
  {
    const int n_seq = a.n_seq;
    // no more shares than tiles, so that every share between two others holds something
    auto share = [&](unsigned long long total, unsigned i) {
      const unsigned shares = total < gridDim.x ? (unsigned)total : gridDim.x;
      if (i >= shares) return total;
      return total <= 0xffffffull ? (unsigned long long)((unsigned)total * i / shares) : total * i / shares;
    };
    auto found = [&](const TreeSeq& sq, int b, unsigned long long at, unsigned long long n) {
      s_any = s_walk.start(&a, CH, S::LEAD, b, sq, at, (int)n);
      seg_tab[0] = tree_segment(s_walk);
    };
    const bool all = blockIdx.x == 0;  // CTA 0 looks for sequences that do not fit
    auto look = [&](int b, const TreeSeq& sq) {
      if (tree_seq_bad(a, b, sq)) atomicOr(a.err, ERR_RANGE);
    };
    auto scan = [&](unsigned long long x) {  // inclusive, over a warp
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      return x;
    };
    if (!S::TICKET && tid == 0) ta.parts[blockIdx.x].n = 0;
    if (n_seq <= 32) {  // one warp sees them all
      if (wi == 0) {
        TreeSeq sq{0, 0, 0, 0};
        if (lane < n_seq) sq = tree_seq(a, lane);
        const unsigned long long w = tree_work(sq, n_kv, group, CH, S::LEAD), inc = scan(w);
        const unsigned long long total = __shfl_sync(0xffffffffu, inc, 31);
        const unsigned long long t0 = share(total, blockIdx.x), t1 = share(total, blockIdx.x + 1);
        if (lane == 0) s_all = total;
        if (w && inc - w <= t0 && t0 < inc && t1 > t0) found(sq, lane, t0 - (inc - w), t1 - t0);
        if (all && lane < n_seq) look(lane, sq);
      }
    } else {
      auto seq = [&](int b) { return b < n_seq ? tree_seq(a, b) : TreeSeq{0, 0, 0, 0}; };
      unsigned long long sum = 0;
      for (int b = tid; b < n_seq; b += TT_THREADS) sum += tree_work(seq(b), n_kv, group, CH, S::LEAD);
      sum = scan(sum);
      if (lane == 31) w_sum[wi] = sum;
      __syncthreads();
      unsigned long long total = 0;
      for (int w = 0; w < TT_THREADS / 32; w++) total += w_sum[w];
      const unsigned long long t0 = share(total, blockIdx.x), t1 = share(total, blockIdx.x + 1);
      if (tid == 0) s_all = total;
      unsigned long long before = 0;
      for (int b0 = 0; b0 < n_seq && (all || (t1 > t0 && before <= t0)); b0 += TT_THREADS) {
        const int b = b0 + tid;
        const TreeSeq sq = seq(b);
        const unsigned long long w = tree_work(sq, n_kv, group, CH, S::LEAD), inc = scan(w);
        __syncthreads();
        if (lane == 31) w_sum[wi] = inc;
        __syncthreads();
        unsigned long long pre = before + inc - w;
        for (int x = 0; x < TT_THREADS / 32; x++) {
          if (x < wi) pre += w_sum[x];
          before += w_sum[x];
        }
        if (w && pre <= t0 && t0 < pre + w && t1 > t0) found(sq, b, t0 - pre, t1 - t0);
        if (all && b < n_seq) look(b, sq);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_s;
  // A segment's columns: q operand, masks, places.  Eight lanes a column, four
  // columns a warp at a time; this warp is number `at` of `warps`.
  auto stage = [&](const TreeSegment& sg, int set, int at, int warps) {
    const float scale2 = LOG2E / sqrtf((float)hd);
    const int sub = lane & 7;
    const TreeSeq sq{sg.row, sg.len, sg.total - sg.len, sg.off};
#pragma unroll 1
    for (int c = at * 4 + (lane >> 3); c < CH; c += warps * 4) {
      const int vh = sg.vh0 + c, node = vh / group, head = sg.kvh * group + vh - node * group;
      const bool in = c < sg.cols;
      const int off = (node * a.n_heads + head) * hd;
      const float* src = a.q + (size_t)sg.off * a.n_heads * hd + off;
      float x[16], amax = 0.0f;
      bool nan = false;
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const int d = (e >> 2) * 32 + sub * 4 + (e & 3);
        x[e] = in && d < hd ? src[d] : 0.0f;
        nan |= x[e] != x[e];
        amax = fmaxf(amax, fabsf(x[e]));
      }
      const unsigned long long mask = in ? tree_mask(a, sq, node) : 0ull;
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        nan |= __shfl_xor_sync(0xffffffffu, (int)nan, o) != 0;
      }
      float mul;
      if constexpr (Q8) {
        const float up = amax < 1e-25f ? 0x1p96f : 1.0f;  // keeps the quotient finite
        const float inv = amax > 0.0f ? TT_DIGITS / (amax * up) : 0.0f;
        mul = (amax / TT_DIGITS) * scale2;
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          uint32_t b[4];  // balanced digits, a byte each
#pragma unroll
          for (int z = 0; z < 4; z++)
            b[z] = (uint32_t)(__float2int_rn(fminf(fmaxf(x[e + z] * up * inv, -TT_DIGITS), TT_DIGITS)) + 0x808080) ^ 0x808080u;
#pragma unroll
          for (int z = 0; z < 3; z++) {
            const int row = z * CH + c, sh = 16 - 8 * z;
            *reinterpret_cast<uint32_t*>(q_t + row * 128 + (((e / 2 + (sub >> 2)) ^ (row & 7)) << 4) + (sub & 3) * 4) =
                (b[0] >> sh & 255u) | (b[1] >> sh & 255u) << 8 | (b[2] >> sh & 255u) << 16 | (b[3] >> sh & 255u) << 24;
          }
        }
      } else {
        // a power of two that brings the largest value to [2^13, 2^14)
        const int e2 = amax > 0.0f && amax < INFINITY ? min(120, 13 - ilogbf(amax)) : 0;
        const float up = __int_as_float((e2 + 127) << 23);
        mul = scale2 / up;
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          alignas(8) __half hh[4], hl[4];
#pragma unroll
          for (int z = 0; z < 4; z++) {
            const float v = x[e + z] * up;
            hh[z] = __float2half_rn(v);
            hl[z] = __float2half_rn(v - __half2float(hh[z]));
          }
#pragma unroll
          for (int z = 0; z < 2; z++) {
            const int row = z * CH + c, k = e * 8 + sub * 4;
            *reinterpret_cast<uint2*>(q_t + (k >> 6) * (N * 128) + row * 128 + ((((k & 63) >> 3) ^ (row & 7)) << 4) + (k & 7) * 2) =
                *reinterpret_cast<const uint2*>(z ? hl : hh);
          }
        }
      }
      if (sub == 0) {
        col_off[set][c] = off;
        col_mul[set][c] = nan ? __int_as_float(0x7fffffff) : mul;
        col_mask[set][c] = mask;
        if (!Q8 && mask) atomicOr(&any_mask[set], mask);
      }
    }
    if constexpr (Q8 && NQ == 8) {  // the operand's last eight rows
      if (at == 0)
        for (int i = lane; i < 64; i += 32) *reinterpret_cast<uint4*>(q_t + 24 * 128 + i * 16) = make_uint4(0u, 0u, 0u, 0u);
    }
    fence_async_smem();
  };

  // Team k % TG does the CTA's tile k, as its item k / TG.
  if (!s_any) {
    // nothing: fall through to the end
  } else if (wi == TT_TMA_WARP) {
    // ------------------------------------------------ TMA: K and V of every tile, slot after slot
    if (lane == 0) {
      TreeWalk w = s_walk;
      int slot = 0, used = 0;
      uint32_t phase = 1;  // a fresh barrier's previous phase counts as done
      bool go = true;
      do {
        for (int t = w.tile; go && t < w.tile + w.seg; t++)
          for (int kv = 0; kv < 2; kv++) {
            if (!tt_wait(&empty[slot], phase, abort)) {
              go = false;
              break;
            }
            mbar_arrive_expect_tx(&full[kv][slot], slot_bytes);
            for (int x = 0; x < boxes; x++)
              tma_load_3d(base + slot * slot_bytes + x * 16384, kv ? &ta.tm_v : &ta.tm_k, x * 64, w.kvh,
                          w.s.start + t * TT_TILE, &full[kv][slot]);
            used++;
            if (++slot == slots) {
              slot = 0;
              phase ^= 1;
            }
          }
      } while (go && w.next());
      // wind down: every copy issued has landed before the CTA may exit
      for (int i = max(0, used - slots); i < used; i++)
        if (!mbar_wait(&full[i & 1][i % slots], (uint32_t)((i >> 1) / period) & 1, *abort ? 1u << 16 : kMbarPolls)) *abort = 1;
    }
    __syncwarp();
  } else if (wi == TT_S_WARP || wi == TT_O_WARP) {
    // ------------------------------------------------ MMA: scores (K slots), outputs (V slots)
    if (lane == 0) {
      TreeWalk w = s_walk;
      const bool scores = wi == TT_S_WARP;
      const int ks_n = Q8 ? (hd + 31) / 32 : (hd + 15) / 16;
      constexpr uint32_t IDESC_S = tt_idesc<Q8>(N, false), IDESC_O = tt_idesc<Q8>(S::NO, true);
      int slot = scores ? 0 : 1, seg_left = w.seg;
      uint32_t phase = 0, segs = 0;
      int turn = 0;  // of `period` tiles, after which a slot's barrier is in its next phase
      bool fresh = true;  // a segment begins: its columns first
      for (int k = 0;; k++) {
        const int g = k % TG;
        const uint32_t n = (uint32_t)(k / TG);
        if (scores) {
          if (fresh && !tt_wait(&q_ready, segs & 1, abort)) break;
          if (n && !tt_wait(&s_free[g], (n - 1) & 1, abort)) break;
          if (!tt_wait(&full[0][slot], phase, abort)) break;
          tc_fence_after();
          const uint64_t kd = sw128_desc(smem_u32(base + slot * slot_bytes));
          const uint64_t qd = sw128_desc(smem_u32(q_t));
          // unrolled: a product whose descriptors and flags the compiler does not
          // know takes 125 cycles to issue, not 40
#pragma unroll
          for (int ks = 0; ks < (Q8 ? 4 : 8); ks++) {
            if (ks >= ks_n) break;
            if constexpr (Q8)
              tc_mma_i8_acc(tmem + g * CS, kd + ks * 2, qd + ks * 2, IDESC_S, ks > 0);
            else
              tc_mma_f16(tmem + g * CS, kd + (uint64_t)((ks >> 2) * 1024 + (ks & 3) * 2),
                         qd + (uint64_t)((ks >> 2) * (N * 8) + (ks & 3) * 2), IDESC_S, ks > 0);
          }
          tc_commit(&s_full[g]);
          fresh = --seg_left == 0;
          if (fresh) {
            tc_commit(&q_free);
            segs++;
          }
        } else {
          if (!tt_wait(&p_full[g], n & 1, abort)) break;
          if (!tt_wait(&full[1][slot], phase, abort)) break;
          tc_fence_after();
          // one 128-byte-wide block of M per box; a lone f16 box stands for both
          // halves (the upper half of O is not read)
          const uint64_t vd = sw128_desc_mn(smem_u32(base + slot * slot_bytes), boxes == 2 ? 16384u : 0u, 1024u);
          const uint64_t pd = sw64_desc_mn(smem_u32(base + S::OFF_P + g * S::PSZ));
          const uint32_t d = tmem + TG * CS + g * CO;
          const bool on = x_on[g] != 0;      // onto the tiles before this one
          constexpr int STEPS = Q8 ? 4 : 8;  // 32 or 16 positions each
#pragma unroll
          for (int ks = 0; ks < STEPS; ks++) {
            if constexpr (Q8)
              tc_mma_i8_acc(d, vd + ks * 256, pd + ks * 128, IDESC_O, ks > 0 || on);
            else
              tc_mma_f16(d, vd + ks * 128, pd + ks * 64, IDESC_O, ks > 0 || on);
          }
          tc_commit(&o_full[g]);
          fresh = --seg_left == 0;
        }
        tc_commit(&empty[slot]);
        slot += 2;  // K and V alternate
        if (slot >= slots) slot -= slots;
        if (++turn == period) {
          turn = 0;
          phase ^= 1;
        }
        if (fresh) {
          if (!w.next()) break;
          seg_left = w.seg;
        }
      }
      // wind down: every MMA issued has completed before TMEM is freed
      uint64_t* last = scores ? &done_s : &done_o;
      tc_commit(last);
      if (!mbar_wait(last, 0, *abort ? 1u << 16 : kMbarPolls)) *abort = 1;
    }
    __syncwarp();
  } else if (wi == TT_NEXT_WARP) {
    // ------------------------------------------------ the segments, one ahead
    auto part = [&](const TreeSegment& sg) {
      const unsigned shares = s_all < gridDim.x ? (unsigned)s_all : gridDim.x;
      const int all = sg.before + sg.tiles + sg.rest;
      auto cta = [&](unsigned long long place) {  // whose share holds it
        const unsigned long long x = (place + 1) * shares - 1;
        return x <= 0xffffffffull ? (int)((unsigned)x / (unsigned)s_all) : (int)(x / s_all);
      };
      // a unit that goes on ends this share, one that came from before began it
      const unsigned long long u0 = sg.before ? s_all * blockIdx.x / shares - sg.before : s_all * (blockIdx.x + 1) / shares - sg.tiles;
      const int i0 = cta(u0);
      return make_int2(i0, cta(u0 + all - 1) - i0 + 1);
    };
    stage(seg_tab[0], 0, TT_SOFT / 32, TT_SOFT / 32 + 1);
    first_sync();
    if (S::STAGERS == 1) mbar_arrive(&q_ready);
    if (lane == 0) {
      seg_part[0] = part(seg_tab[0]);
      mbar_arrive(&parts0);
    }
    TreeWalk w = s_walk;
    for (int seg = 1; w.next(); seg++) {
      const int set = seg & 1;
      // everybody is in the last segment, so the set's readers, two segments ago, are done
      tt_wait(&seg_seen, (uint32_t)(seg - 1) & 1, abort);
      if (S::STAGERS == 1) tt_wait(&q_free, (uint32_t)(seg - 1) & 1, abort);  // the last segment's products have read q
      if (__any_sync(0xffffffffu, *abort != 0)) break;
      const TreeSegment sg = tree_segment(w);
      if (lane == 0) {
        seg_tab[set] = sg;
        seg_part[set] = part(sg);
        if (S::STAGERS > 1) mbar_arrive(&seg_ready);
      }
      if constexpr (S::STAGERS == 1) {
        stage(sg, set, 0, 1);
        mbar_arrive(&q_ready);
      }
    }
  } else {
    // ------------------------------------------------ softmax groups
    const int g = wi >> 2, wq = wi & 3, r = tid & 127, tg = g / CG, cg = g % CG;
    const uint32_t lanes = (uint32_t)(wq * 32) << 16;
    const int c0 = cg * NQ;  // of the team's columns
    const uint32_t s_at = tmem + lanes + (uint32_t)(tg * CS + c0), o_at = tmem + lanes + (uint32_t)(TG * CS + tg * CO + c0);
    uint8_t* p_t = base + S::OFF_P + tg * S::PSZ;
    const bool has_dim = wq * 32 < hd;  // this warp's lanes of O are dims
    int item = 0;  // of this group, over all segments
    int k0 = 0;    // tiles of the CTA before this segment
    int seg_no = 0, more;
    do {
      const int set = seg_no & 1;
      if (seg_no) {
        tt_wait(&q_ready, (uint32_t)seg_no & 1, abort);  // its columns' tables
        // one decision for all, so that the named barriers stay matched; from here
        // on the last segment's p operands are free
        if (groups_any(*abort != 0)) break;
      }
      if (tid == 0) mbar_arrive(&seg_seen);
      const TreeSegment& sg = seg_tab[set];
      const int len = sg.len, total = sg.total, tiles = sg.tiles;
      const int first = (tg - k0) & (TG - 1);
      const bool trees = total - len > 1;
      const float *ks_at = nullptr, *vs_at = nullptr;
      float ks_next = 0.0f, vs_next = 0.0f;
      auto scales = [&](int t) {  // of tile t's place r, and on to the group's next tile
        const bool in = t * TT_TILE + r < total;
        ks_next = in ? *ks_at : 0.0f;
        vs_next = in ? *vs_at : 0.0f;
        ks_at += (size_t)(TG * TT_TILE) * a.c.scale_row;
        vs_at += (size_t)(TG * TT_TILE) * a.c.scale_row;
      };
      if (Q8 && first < tiles) {
        const size_t at = ((size_t)sg.row + first * TT_TILE + r) * a.c.scale_row + (size_t)sg.kvh * a.c.scale_head;
        ks_at = a.c.k_scale + at;
        vs_at = a.c.v_scale + at;
        scales(first);
      }
      if (seg_no == 0) {
        stage(sg, 0, wi, TT_SOFT / 32 + 1);
        first_sync();
        if (S::STAGERS > 1) mbar_arrive(&q_ready);
      }
      F2 l[NQ / 2], o[NQ / 2];
      if (lane < NQ) x_col[wi][lane] = make_float4(-INFINITY, -INFINITY, 0.0f, 0.0f);
      int left = 0;           // tiles until the references are due
      bool held = false;      // O holds tiles that are not in o
#pragma unroll
      for (int c = 0; c < NQ / 2; c++) l[c] = o[c] = F2(0.0f);
      if (!Q8 && r == 0) x_bad[g] = 0ull;

      // l, summed over the warp, joins the columns' sums
      auto sums = [&]() {
        float v[NQ];
#pragma unroll
        for (int c = 0; c < NQ / 2; c++) {
          v[2 * c] = l[c].lo();
          v[2 * c + 1] = l[c].hi();
          l[c] = F2(0.0f);
        }
        auto halve = [&](auto columns, int bit) {  // a lane keeps half of its columns, and the other's of the same
          constexpr int n = decltype(columns)::value;
          const bool upper = lane & bit;
#pragma unroll
          for (int i = 0; i < n; i++) {
            const float other = __shfl_xor_sync(0xffffffffu, upper ? v[i] : v[i + n], bit);
            v[i] = (upper ? v[i + n] : v[i]) + other;
          }
        };
        if constexpr (NQ == 16) halve(std::integral_constant<int, 8>(), 16);
        halve(std::integral_constant<int, 4>(), 128 / NQ);
        halve(std::integral_constant<int, 2>(), 64 / NQ);
        halve(std::integral_constant<int, 1>(), 32 / NQ);
        if constexpr (NQ == 8) v[0] += __shfl_xor_sync(0xffffffffu, v[0], 2);
        v[0] += __shfl_xor_sync(0xffffffffu, v[0], 1);
        __syncwarp();
        if (lane % (32 / NQ) == 0) {
          float4& at = x_col[wi][lane / (32 / NQ)];
          if (Q8) {  // and what that rounds away
            const float sum = at.z + v[0], part = sum - at.z;
            at.w += (at.z - (sum - part)) + (v[0] - part);
            at.z = sum;
          } else {
            at.z += v[0];
          }
        }
      };
      // O into the registers
      auto fold = [&]() {
        tt_wait(&o_full[tg], (uint32_t)(item - 1) & 1, abort);
        tc_fence_after();
        if (has_dim) {
          const F2 unit(1.0f / TT_UNITS<Q8>);
#pragma unroll
          for (int cb = 0; cb < NQ; cb += 8) {
            uint32_t v[32];
            tc_ld8(o_at + cb, v);
            tc_ld8(o_at + CH + cb, v + 8);
            if constexpr (Q8) {
              tc_ld8(o_at + 2 * CH + cb, v + 16);
              tc_ld8(o_at + 3 * CH + cb, v + 24);
            }
            tc_wait_ld();
#pragma unroll
            for (int c = 0; c < 8; c += 2) {
              F2& x = o[(cb + c) / 2];
              if constexpr (Q8) {
                const F2 k(256.0f), k7(128.0f);
                auto digit = [&](int z) { return F2((float)(int)v[8 * z + c], (float)(int)v[8 * z + c + 1]); };
                x = fma2(fma2(fma2(fma2(digit(0), k, digit(1)), k7, digit(2)), k, digit(3)), unit, x);
              } else {
                x = fma2(joined<false, 8>(v, c), unit, x);
              }
            }
          }
        }
        tc_fence_before();
      };

      for (int t = first; t < tiles; t += TG, item++) {
        // (not where drafted places are: what one node sees must not change the order of another's sum)
        if (Q8 && left == 0 && t != first && (!trees || (t + 1) * TT_TILE <= len)) sums();
        const int pos = t * TT_TILE + r, j = pos - len;
        const bool edge = (t + 1) * TT_TILE > len;  // drafted places or none at all among the tile's
        const bool there = pos < total;
        // an f16 edge tile: which 8-value pieces of this drafted V row are not finite
        uint32_t odd = 0;
        if constexpr (!Q8) {
          if (edge && there && j >= 0 && (any_mask[set] >> j & 1)) {
            const uint4* v = reinterpret_cast<const uint4*>(static_cast<const __half*>(a.c.v) +
                                                            (size_t)(sg.row + pos) * a.c.row_stride +
                                                            (size_t)sg.kvh * a.c.head_stride);
            for (int c = 0; c < hd / 8; c++) {
              const uint4 x = v[c];
              const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
              bool bad = false;
#pragma unroll
              for (int e = 0; e < 4; e++)
                bad |= (xs[e] & 0x7c00u) == 0x7c00u || (xs[e] & 0x7c000000u) == 0x7c000000u;
              odd |= (uint32_t)bad << c;
            }
          }
        }
        // this place's scales: K's, and V's as 2^ve * vm
        float ks = ks_next, vm = 0.0f;
        int ve = 0;
        if constexpr (Q8) {
          const float vs = vs_next;
          if (t + TG < tiles) scales(t + TG);
          const uint32_t b = __float_as_uint(vs);
          ve = (int)(b >> 23 & 255u) - 127;
          const bool in = (unsigned)(ve - TT_E_MIN) < TT_E_MAX - TT_E_MIN;
          vm = in ? __uint_as_float((b & 0x807fffffu) | 0x3f800000u) : 0.0f;  // with its sign: the digits have theirs
          if (!in) ve = TT_E_MIN;
          if (!in && vs != 0.0f) ks = __int_as_float(0x7fffffff);
        }
        // ---- scores (with V's exponent), in powers of two, against the references
        tt_wait(&s_full[tg], (uint32_t)item & 1, abort);
        tc_fence_after();
        constexpr int W = NQ;  // columns of one load: each wait for TMEM costs its whole latency
        F2 s[NQ / 2];
        const F2 ks2(ks), ve2((float)ve);
#pragma unroll
        for (int cb = 0; cb < NQ; cb += W) {
          uint32_t v[3 * W];
          tt_ld<W>(s_at + cb, v);
          tt_ld<W>(s_at + CH + cb, v + W);
          if constexpr (Q8) tt_ld<W>(s_at + 2 * CH + cb, v + 2 * W);
          tc_wait_ld();
#pragma unroll
          for (int c = 0; c < W; c += 4) {
            const float4 m = *reinterpret_cast<const float4*>(&col_mul[set][c0 + cb + c]);
            F2& s0 = s[(cb + c) / 2];
            F2& s1 = s[(cb + c) / 2 + 1];
            if constexpr (Q8) {
              s0 = fma2(joined<Q8, W>(v, c), F2(m.x, m.y) * ks2, ve2);
              s1 = fma2(joined<Q8, W>(v, c + 2), F2(m.z, m.w) * ks2, ve2);
            } else {
              s0 = joined<Q8, W>(v, c) * F2(m.x, m.y);
              s1 = joined<Q8, W>(v, c + 2) * F2(m.z, m.w);
            }
          }
        }
        tc_fence_before();
        mbar_arrive(&s_free[tg]);
        if (edge) {
#pragma unroll
          for (int c = 0; c < NQ; c += 2) {
            const bool s0 = j < 0 || (there && (col_mask[set][c0 + c] >> j & 1));
            const bool s1 = j < 0 || (there && (col_mask[set][c0 + c + 1] >> j & 1));
            s[c / 2] = F2(s0 ? s[c / 2].lo() : -INFINITY, s1 ? s[c / 2].hi() : -INFINITY);
          }
        }
        // tiles with drafted places set the references anew each: whether another
        // node's score passes its reference must not touch this one's sums
        const bool due = left == 0;  // (an f16 cache: at the first tile)
        bool fresh = due || (edge && trees);
        if (t != first) {
          float top = -INFINITY;
#pragma unroll
          for (int c = 0; c < NQ; c += 4) {
            const float4 m = *reinterpret_cast<const float4*>(&x_m[wi][c]);
            s[c / 2] = s[c / 2] + F2(m.x, m.y);
            s[c / 2 + 1] = s[c / 2 + 1] + F2(m.z, m.w);
            top = fmaxf(fmaxf(top, fmaxf(s[c / 2].lo(), s[c / 2].hi())), fmaxf(s[c / 2 + 1].lo(), s[c / 2 + 1].hi()));
          }
          if (!fresh) fresh = team_any<CG>(tg, top > TT_ROOM);
        }
        if (held && (fresh || !Q8)) {
          fold();
          held = false;
        }
        if (fresh) {
          // ---- the references
#pragma unroll
          for (int c = 0; c < NQ; c += 4) {
            float4 m;
            m.x = redux_max(s[c / 2].lo());
            m.y = redux_max(s[c / 2].hi());
            m.z = redux_max(s[c / 2 + 1].lo());
            m.w = redux_max(s[c / 2 + 1].hi());
            if (lane == 0) *reinterpret_cast<float4*>(&x_max[g][wq][c]) = m;
          }
          group_sync(g);
          bool soon = false;
          if (lane < NQ) {
            // against the old reference, or against 0 where there is none
            const float m = fmaxf(fmaxf(x_max[g][0][lane], x_max[g][1][lane]), fmaxf(x_max[g][2][lane], x_max[g][3][lane]));
            float4 at = x_col[wi][lane];
            const bool none = at.x == -INFINITY;
            float up = none ? (m == -INFINITY ? 0.0f : m) : fmaxf(m, 0.0f);
            const float top = none ? m : at.x + m;  // the tile's largest score
            soon = none || top - at.y > TT_FAR;
            if (Q8 && !none) {
              // whole powers of two, so that rescaling rounds nothing
              if (m < -TT_LOW && m != -INFINITY) up = fmaxf(m + TT_ABOVE, at.y - TT_DEPTH - at.x);
              up = ceilf(up);
            }
            if (Q8 && soon && fabsf(top) < 65536.0f) up -= TT_SPARE;
            const float al = none ? 1.0f : ex2(-up);
            if (!none) at.x += up;
            else if (m != -INFINITY) at.x = up;
            at.y = fmaxf(at.y, top);
            at.z *= al;
            at.w *= al;
            x_col[wi][lane] = at;
            x_al[wi][lane] = al;
            x_m[wi][lane] = at.x == -INFINITY ? 0.0f : -at.x;
            x_d[wi][lane] = -up;
          }
          // the tables are written, and x_max may be again
          if constexpr (Q8) {
            soon = team_any<CG>(tg, soon);
            left = soon ? 1 : due ? S::RUN : left;
          } else {
            group_sync(g);
            left = 1;
          }
#pragma unroll
          for (int c = 0; c < NQ; c += 4) {
            const float4 m = *reinterpret_cast<const float4*>(&x_d[wi][c]), al = *reinterpret_cast<const float4*>(&x_al[wi][c]);
            s[c / 2] = s[c / 2] + F2(m.x, m.y);
            s[c / 2 + 1] = s[c / 2 + 1] + F2(m.z, m.w);
            l[c / 2] = l[c / 2] * F2(al.x, al.y);
            l[c / 2 + 1] = l[c / 2 + 1] * F2(al.z, al.w);
            o[c / 2] = o[c / 2] * F2(al.x, al.y);
            o[c / 2 + 1] = o[c / 2 + 1] * F2(al.z, al.w);
          }
        }
        // ---- probabilities, in the operand's form, a row per position
        if constexpr (Q8) {
          const F2 cm(vm * TT_UNITS<true>), iv(__uint_as_float((uint32_t)(127 - ve) << 23));
          uint32_t dg[4][NQ / 4];
#pragma unroll
          for (int c = 0; c < NQ; c += 4) {
            const F2 p0(ex2(s[c / 2].lo()), ex2(s[c / 2].hi())), p1(ex2(s[c / 2 + 1].lo()), ex2(s[c / 2 + 1].hi()));
            l[c / 2] = fma2(p0, iv, l[c / 2]);
            l[c / 2 + 1] = fma2(p1, iv, l[c / 2 + 1]);
            // x = 2^15 h + l, both by adding 3 * 2^22 (and 128, which makes the lower byte's
            // balanced digit that byte less 128): two digits each, all exact
            const F2 x0 = p0 * cm, x1 = p1 * cm, one(12582912.0f + 128.0f), low(-32768.0f);
            const F2 h0 = fma2(x0, F2(1.0f / 32768.0f), one), h1 = fma2(x1, F2(1.0f / 32768.0f), one);
            const F2 minus(-12582912.0f - 128.0f);
            const F2 l0 = fma2(h0 + minus, low, x0) + one, l1 = fma2(h1 + minus, low, x1) + one;
            auto word = [](float x) { return __float_as_uint(x); };
            const uint32_t a01 = __byte_perm(word(l0.lo()), word(l0.hi()), 0x5140), a23 = __byte_perm(word(l1.lo()), word(l1.hi()), 0x5140);
            const uint32_t b01 = __byte_perm(word(h0.lo()), word(h0.hi()), 0x5140), b23 = __byte_perm(word(h1.lo()), word(h1.hi()), 0x5140);
            dg[3][c / 4] = __byte_perm(a01, a23, 0x5410) ^ 0x80808080u;
            dg[2][c / 4] = __byte_perm(a01, a23, 0x7632);
            dg[1][c / 4] = __byte_perm(b01, b23, 0x5410) ^ 0x80808080u;
            dg[0][c / 4] = __byte_perm(b01, b23, 0x7632);
          }
          if (item) tt_wait(&o_full[tg], (uint32_t)(item - 1) & 1, abort);  // the p operand has been read
          if constexpr (NQ == 16) {
#pragma unroll
            for (int z = 0; z < 4; z++)
              *reinterpret_cast<uint4*>(p_t + sw64(r, z * CG + cg)) = make_uint4(dg[z][0], dg[z][1], dg[z][2], dg[z][3]);
          } else {
            *reinterpret_cast<uint4*>(p_t + sw64(r, 0)) = make_uint4(dg[0][0], dg[0][1], dg[1][0], dg[1][1]);
            *reinterpret_cast<uint4*>(p_t + sw64(r, 1)) = make_uint4(dg[2][0], dg[2][1], dg[3][0], dg[3][1]);
          }
        } else {
          if (item) tt_wait(&o_full[tg], (uint32_t)(item - 1) & 1, abort);  // the p operand has been read
#pragma unroll
          for (int cb = 0; cb < NQ; cb += 8) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const int c = cb + e * 2;
              const F2 p(ex2(s[c / 2].lo()), ex2(s[c / 2].hi()));
              l[c / 2] = l[c / 2] + p;
              const F2 x = p * F2(TT_UNITS<false>);  // far from f16's smallest values
              const F2 h(__uint_as_float(__float_as_uint(x.lo()) & 0xffffe000u), __uint_as_float(__float_as_uint(x.hi()) & 0xffffe000u));
              const F2 rest = fma2(h, F2(-1.0f), x);
              const __half2 hh = __floats2half2_rn(h.lo(), h.hi()), dd = __floats2half2_rn(rest.lo(), rest.hi());
              hi[e] = *reinterpret_cast<const uint32_t*>(&hh);
              lo[e] = *reinterpret_cast<const uint32_t*>(&dd);
            }
            *reinterpret_cast<uint4*>(p_t + sw64(r, (c0 + cb) / 8)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4*>(p_t + sw64(r, (CH + c0 + cb) / 8)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          }
          // V of places nobody sees, and values that are not finite in drafted rows, become zeros
          if (edge) {
            const int v_slot = (2 * (k0 + t) + 1) % slots;  // K and V alternate over the CTA's tiles
            const bool row_gone = j >= 0 && !(there && (any_mask[set] >> j & 1));
            if (row_gone || odd) {
              tt_wait(&full[1][v_slot], (uint32_t)((k0 + t) / period) & 1, abort);
              uint8_t* vt = base + v_slot * slot_bytes + r * 128;
              for (int c = 0; c < 8 * boxes; c++)
                if (row_gone || (odd >> c & 1)) {
                  uint4* at = reinterpret_cast<uint4*>(vt + (c >> 3) * 16384 + (((c & 7) ^ (r & 7)) << 4));
                  if (row_gone) {
                    *at = make_uint4(0u, 0u, 0u, 0u);
                  } else {
                    uint4 x = *at;
                    uint32_t* xs = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                      if ((xs[e] & 0x7c00u) == 0x7c00u) xs[e] &= 0xffff0000u;
                      if ((xs[e] & 0x7c000000u) == 0x7c000000u) xs[e] &= 0xffffu;
                    }
                    *at = x;
                  }
                }
              if (odd) atomicOr(&x_bad[g], 1ull << j);
            }
          }
        }
        if (r == 0 && cg == 0) x_on[tg] = held;
        held = true;
        if (Q8) left--;
        fence_async_smem();
        mbar_arrive(&p_full[tg]);
      }
      if (S::STAGERS > 1 && sg.more) {
        // the next segment's columns, so that its scores are under way while this one ends
        tt_wait(&seg_ready, (uint32_t)seg_no & 1, abort);
        tt_wait(&q_free, (uint32_t)seg_no & 1, abort);  // this segment's products have read the operand
        if (!__any_sync(0xffffffffu, *abort != 0)) stage(seg_tab[set ^ 1], set ^ 1, wi, TT_SOFT / 32);
        mbar_arrive(&q_ready);
      }
      if (held) fold();
      if constexpr (!Q8) {  // drafted rows of V that are not finite: nodes that see them get NaN
        group_sync(g);
        unsigned long long bad = x_bad[g];
        while (bad) {
          const int j = __ffsll((long long)bad) - 1;
          bad &= bad - 1;
          float v = 0.0f;
          if (r < hd)
            v = __half2float(static_cast<const __half*>(a.c.v)[(size_t)(sg.row + len + j) * a.c.row_stride +
                                                              (size_t)sg.kvh * a.c.head_stride + r]);
          if (!(fabsf(v) < INFINITY)) {
            const float nan = __int_as_float(0x7fffffff);
#pragma unroll
            for (int c = 0; c < NQ; c += 2)
              o[c / 2] = F2(col_mask[set][c0 + c] >> j & 1 ? nan : o[c / 2].lo(),
                            col_mask[set][c0 + c + 1] >> j & 1 ? nan : o[c / 2].hi());
          }
        }
      }

      // ---- the segment's (max, sum, o): the groups of a column range meet through their idle p operands
      sums();
      if constexpr (TG > 1) {
        float* po = reinterpret_cast<float*>(p_t) + cg * NQ * 128;
#pragma unroll
        for (int c = 0; c < NQ; c++) po[c * 128 + r] = c & 1 ? o[c / 2].hi() : o[c / 2].lo();
      }
      group_sync(g);
      if (wq == 0 && lane < NQ) {
        const float sum = (x_col[wi][lane].z + x_col[wi + 1][lane].z) + (x_col[wi + 2][lane].z + x_col[wi + 3][lane].z) +
                          (Q8 ? (x_col[wi][lane].w + x_col[wi + 1][lane].w) + (x_col[wi + 2][lane].w + x_col[wi + 3][lane].w) : 0.0f);
        x_fin[g][lane] = make_float2(x_col[wi][lane].x, sum);
        if (Q8 && sum != sum && !sg.before && !sg.rest) s_nan = 1;
      }
      groups_sync();
      {
        const bool first_part = sg.before == 0, whole = first_part && !sg.rest;
        const size_t slot = 2 * (size_t)blockIdx.x + (first_part ? 1 : 0);
        const int cols = sg.cols;
        float* out_seq = a.out + (size_t)sg.off * a.n_heads * hd;
        auto put = [&](int c, float m, float sum, float x) {  // column c: final, or a partial
          if (whole) {
            if (r < hd) out_seq[col_off[set][c0 + c] + r] = sum == 0.0f ? 0.0f : x / sum;
          } else {
            if (r == 0) ta.part_ml[slot * CH + c0 + c] = make_float2(m, sum);
            if (r < hd) ta.part_o[(slot * CH + c0 + c) * hd + r] = x;
          }
        };
        if constexpr (TG == 1) {
#pragma unroll
          for (int c = 0; c < NQ; c++)
            if (c0 + c < cols) put(c, x_fin[g][c].x, x_fin[g][c].y, c & 1 ? o[c / 2].hi() : o[c / 2].lo());
        } else {
#pragma unroll
          for (int i = 0; i < NQ / TG; i++) {  // the teams share the columns
            const int c = i * TG + tg;
            if (c0 + c >= cols) break;
            float m = -INFINITY, sum = 0.0f, x = 0.0f;
#pragma unroll
            for (int q = 0; q < TG; q++) m = fmaxf(m, x_fin[q * CG + cg][c].x);
#pragma unroll
            for (int q = 0; q < TG; q++) {
              const float2 f = x_fin[q * CG + cg][c];
              const float wt = f.x == -INFINITY ? 0.0f : ex2(f.x - m);
              sum = fmaf(f.y, wt, sum);
              x = fmaf(reinterpret_cast<const float*>(base + S::OFF_P + q * S::PSZ)[(c0 + c) * 128 + r], wt, x);
            }
            put(c, m, sum, x);
          }
        }
        if (!whole) {
          if (S::TICKET) groups_sync();
          if (tid == 0) {
            const bool known = seg_no || tt_wait(&parts0, 0, abort);
            const int i0 = seg_part[set].x, n = seg_part[set].y;
            if constexpr (S::TICKET) {
              const bool last = known && ticket_acq_rel(ta.tickets + i0) == (unsigned)n - 1;
              if (last) ta.tickets[i0] = 0u;
              s_merge[0] = last ? n : 0;
              s_merge[1] = i0;
            } else if (first_part && known) {
              ta.parts[blockIdx.x] = TreePart{n, cols, sg.vh0, sg.kvh, sg.b, {0, 0, 0}};
            }
          }
          if constexpr (S::TICKET) {
            groups_sync();
            if (s_merge[0]) {
              // the last of them: one warp a column (or two, with half the partials each)
              const int n = s_merge[0], i0 = s_merge[1];
              constexpr int WPC = CH == 8 ? 2 : 1;
              float* half = reinterpret_cast<float*>(base + S::OFF_P);  // [16][128], the p operands are idle
              for (int cb = 0; cb < cols; cb += 16 / WPC) {
                const int c = cb + wi / WPC;
                float sum = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if (c < cols) sum = tree_add<WPC>(ta, CH, c, i0, n, wi % WPC, lane, hd, x);
                if constexpr (WPC == 2) {
                  if (wi & 1) {
#pragma unroll
                    for (int e = 0; e < 4; e++) half[wi * 128 + e * 32 + lane] = x[e];
                  }
                  group_sync(g);
                  if (!(wi & 1)) {
#pragma unroll
                    for (int e = 0; e < 4; e++) x[e] += half[(wi + 1) * 128 + e * 32 + lane];
                  }
                }
                if (Q8 && sum != sum) {
                  if (wi % WPC == 0) tree_column(a, tree_seq(a, sg.b), sg.kvh, sg.vh0 + c, lane);
                } else if (c < cols && wi % WPC == 0) {
#pragma unroll
                  for (int e = 0; e < 4; e++)
                    if (e * 32 + lane < hd) out_seq[col_off[set][c] + e * 32 + lane] = sum == 0.0f ? 0.0f : x[e] / sum;
                }
              }
            }
          }
        }
      }
      more = sg.more;
      if (!Q8 && tid == 0) any_mask[set] = 0ull;
      if (Q8 && s_nan) {
        groups_sync();  // all have seen that, and the NaNs are written
        for (int c = wi; c < sg.cols; c += TT_SOFT / 32) {
          float sum = 0.0f;
          for (int q = 0; q < TG; q++) sum += x_fin[q * CG + c / NQ][c % NQ].y;
          if (sum != sum) tree_column(a, tree_seq(a, sg.b), sg.kvh, sg.vh0 + c, lane);
        }
        s_nan = 0;  // every warp meets before the next segment's end
      }
      k0 += tiles;
      seg_no++;
    } while (more);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (tid == 0 && *abort) atomicOr(a.err, ERR_TIMEOUT);
  if (wi == TT_S_WARP) tc_dealloc(tmem, S::TMEM);
}

// The units that several CTAs shared, each found at the CTA it began in: one
// warp per column.
__global__ void __launch_bounds__(128) tree_merge_kernel(const __grid_constant__ TreeTcArgs ta, int ch) {
  const TreeArgs& a = ta.t;
  const int group = a.n_heads / a.c.n_kv, hd = a.c.hd, lane = threadIdx.x & 31;
  const int i0 = blockIdx.x, c = blockIdx.y * 4 + (threadIdx.x >> 5);
  pdl_wait();
  pdl_trigger();
  const TreePart u = ta.parts[i0];
  if (c >= ch || !u.n || c >= u.cols) return;
  float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const float sum = tree_add<1>(ta, ch, c, i0, u.n, 0, lane, hd, x);
  const TreeSeq s = tree_seq(a, u.b);
  const int vh = u.vh0 + c, node = vh / group, head = u.kvh * group + vh % group;
  if (a.c.q8 && sum != sum) {
    tree_column(a, s, u.kvh, vh, lane);
    return;
  }
  float* out = a.out + ((size_t)(s.off + node) * a.n_heads + head) * hd;
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (e * 32 + lane < hd) out[e * 32 + lane] = sum == 0.0f ? 0.0f : x[e] / sum;
}

static size_t al256(size_t x) { return (x + 255) & ~(size_t)255; }
// Columns of a CTA: as many as there are, up to 64, so that the cache is read
// once.  33 to 64 of a few units are taken as two chunks of 32: with two tiles
// or so for each SM, two teams and no merge kernel count for more than reading
// twice (16 nodes x 4 heads, 8 kv heads, f16: one sequence of 4096 positions 25.8 us
// against 28.4, two of 3000 25.3 against 29.0, four 37.5 against 31.9; one of 30000, a
// length that is not known here, 60 against 54).
static int tt_columns(int max_nodes, int group, int units) {
  const int vh = max_nodes * group;
  return vh <= 8 ? 8 : vh <= 16 ? 16 : vh <= 32 || (vh <= 64 && units <= 16) ? 32 : 64;
}

size_t tree_workspace_bytes(int max_nodes, int n_heads, int n_kv, int hd, int sm_count) {
  const size_t cols = (size_t)2 * sm_count * tt_columns(max_nodes, n_heads / n_kv, INT_MAX);
  return al256(sm_count * sizeof(unsigned)) + al256(sm_count * sizeof(TreePart)) + al256(cols * 8) + al256(cols * hd * 4);
}

template <typename F>
static cudaError_t tt_launch(F fn, dim3 grid, int threads, size_t smem, cudaStream_t st, void** args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelExC(&cfg, (const void*)fn, args);
}

template <bool Q8, int NQ, int CG>
static cudaError_t tt_go(TreeTcArgs& ta, cudaStream_t st) {
  using S = TtShape<Q8, NQ, CG>;
  auto k = tree_tc_kernel<Q8, NQ, CG>;
  static std::atomic<unsigned long long> ready{0};  // devices this kernel has its shared memory on
  const unsigned long long dev = 1ull << (ta.t.device & 63);
  cudaError_t e = cudaSuccess;
  if (!(ready.load(std::memory_order_relaxed) & dev)) {
    e = cudaFuncSetAttribute((const void*)k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::BYTES);
    if (e != cudaSuccess) return e;
    ready.fetch_or(dev, std::memory_order_relaxed);
  }
  ta.slots = S::RING / (ta.boxes * 16384);
  if (ta.slots > TT_MAX_SLOTS) ta.slots = TT_MAX_SLOTS;
  void* args[] = {&ta};
  e = tt_launch(k, dim3(ta.t.sm_count), TT_THREADS, S::BYTES, st, args);
  if (e != cudaSuccess || S::TICKET) return e;
  int ch = S::CH;
  void* margs[] = {&ta, &ch};
  return tt_launch(tree_merge_kernel, dim3(ta.t.sm_count, S::CH / 4), 128, 0, st, margs);
}

cudaError_t launch_attn_tree(const TreeArgs& a, cudaStream_t st) {
  TreeTcArgs ta;
  const KvRowsDev& c = a.c;
  const int box = c.q8 ? 128 : 64, group = a.n_heads / c.n_kv;
  const bool maps = c.hd <= 128 &&
                    encode_rows_map(&ta.tm_k, c.k, c.q8, c.positions, c.n_kv, c.hd, c.row_stride, c.head_stride, box) &&
                    encode_rows_map(&ta.tm_v, c.v, c.q8, c.positions, c.n_kv, c.hd, c.row_stride, c.head_stride, box);
  if (!maps) {
    const dim3 grid((unsigned)a.n_seq, (unsigned)a.n_heads, (unsigned)a.max_nodes);
    if (c.q8) tree_simple_kernel<true><<<grid, TR_THREADS, 0, st>>>(a);
    else tree_simple_kernel<false><<<grid, TR_THREADS, 0, st>>>(a);
    return cudaGetLastError();
  }
  ta.t = a;
  ta.boxes = !c.q8 && c.hd > 64 ? 2 : 1;
  const int cols = tt_columns(a.max_nodes, group, a.n_seq > 16 ? INT_MAX : a.n_seq * c.n_kv);
  const size_t n = (size_t)2 * a.sm_count * cols;
  uint8_t* w = static_cast<uint8_t*>(a.work);
  ta.tickets = a.tickets ? a.tickets : reinterpret_cast<unsigned*>(w);
  w += al256(a.sm_count * sizeof(unsigned));
  ta.parts = reinterpret_cast<TreePart*>(w);
  w += al256(a.sm_count * sizeof(TreePart));
  ta.part_ml = reinterpret_cast<float2*>(w);
  ta.part_o = reinterpret_cast<float*>(w + al256(n * 8));
  switch (cols) {
    case 8: return c.q8 ? tt_go<true, 8, 1>(ta, st) : tt_go<false, 8, 1>(ta, st);
    case 16: return c.q8 ? tt_go<true, 16, 1>(ta, st) : tt_go<false, 16, 1>(ta, st);
    case 32: return c.q8 ? tt_go<true, 16, 2>(ta, st) : tt_go<false, 16, 2>(ta, st);
    default: return c.q8 ? tt_go<true, 16, 4>(ta, st) : tt_go<false, 16, 4>(ta, st);
  }
}

}  // namespace prana
