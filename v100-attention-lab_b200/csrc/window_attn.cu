// Causal attention over a sliding window and the first few tokens (sinks).
//
// Query row i of T sits at position p = S - T + i of S keys and sees key j when
//
//     j <= p,  j < length,  and  (p - j < window  or  j < sinks)
//
//     o_i = sum_j softmax_j(scale q_i . k_j) v_j,   o_i = 0 where nothing is seen
//     (rows at or behind the sequence's length see nothing)
//
// computed with the running maximum and sum of the softmax, one pass over the
// visible key tiles.  Tensor cores bound it at 4 D operations per visible pair;
// the exponentials (16 per clock and SM) take as long as the products do.
//
// Split.  A work item is two tiles of 128 query rows that share their keys: two
// heads of one key head where heads share keys in even groups, else two
// neighbouring tiles of one head.  So every K/V tile fetched feeds two
// products, and while one tile's softmax runs the tensor core works on the
// other's.  One CTA per SM takes item after item; its loads and first scores
// of the next item run under the last one's epilogue.  Warps: 2 x 4 softmax
// (a thread per query row), one that fetches tiles by TMA, two that issue the
// MMAs (one for each query tile).  TMEM holds two score buffers of 64 keys and
// the output of both query tiles; the probabilities overwrite their scores'
// columns and are the second product's TMEM operand, so they never touch shared
// memory.
//
// Measured, 16384 tokens, 32 query and 8 key heads of 128, window 4096, fp16: 842 us
// on the GPU alone (a few launches of a replayed graph), 970 to 990 a call under
// lasting load, where the clock gives way; with heads of 64 684 and 759.  2 x 4096
// tokens, 16 heads of 128, window 1024: 80 and 90.
//
// What was tried, GPU alone, each against the build of its day: two threads per row,
// to have more warps to switch between, together with a quarter of the
// exponentials as polynomials on the FMA pipe, 922, and 851 without either; the polynomials
// with one thread per row 868.  64-key tiles with two score buffers came in one
// step with the cheap MMA issue below (1119 -> 1006): what the tile's size does by
// itself is not known.  A spilled register costs dearly: with this much shared
// memory taken, local memory is L2.
//
// The probabilities are rounded once to the operands' type, as the 16-bit product
// has to have them.  Where keys of like weight make up the output that adds as
// much as the output's own rounding (the sum of the two against 64 bits, for
// normally distributed scores: 1.3 to 1.4 times the latter); fp16 adds its grid
// (see kSlack) for keys far below the largest.  Scores, maxima, sums and outputs are fp32.
//
// Masks.  Only tiles that some mask cuts are masked element by element.  In
// those a key hidden from a row has probability 0, and 0 times a value that is
// not finite would still poison the row.  Such an output cannot be missed: it is
// not finite itself.  Items with one are done again in a careful pass, which
// looks the values of cut tiles over and sums those that hold a non-finite one
// on the CUDA cores, over visible keys alone.
#include "../../include/gdn_b200.h"
#include "host_util.h"
#include "tc.cuh"
#include "tmap.h"

#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstring>
#include <type_traits>

namespace gdn {
namespace wa {
namespace {

constexpr int kTile = 128;          // query rows per tile
constexpr int kKeys = 64;           // keys per tile
constexpr int kSoftmaxWarps = 8;    // 4 per query tile
constexpr int kTmaWarp = 8, kMmaWarp = 9;  // and kMmaWarp + 1: a query tile's products each
constexpr int kThreads = 11 * 32;
constexpr int kBarGroup = 1, kBarAll = 3;  // named barriers: 1 and 2 a query tile's group, 3 all warps
constexpr int kMaxItems = 8192;     // of one CTA
constexpr uint32_t kTmCols = 512;
constexpr uint32_t kTmS = 0, kTmO = 256;  // + 128 x tile (+ 64 x buffer of the scores)

struct Params {
  CUtensorMap tm_q, tm_k, tm_v;
  const int* lengths;
  void* o;
  int* status;
  long long so_b, so_t, so_h;
  int qb, qh, kb, kh, vb, vh;  // 0 where an input is expanded over the batch or the heads (one element of the map), else 1
  int T, S, HK, G;
  int window, sinks;
  int nx, ny, items;  // row tiles (or pairs) and heads (or pairs) of an item grid, items in all
  int pair_heads;    // an item's two tiles are two heads (else two row tiles of one head)
  int single;        // an item is one tile, its second one empty
  float scale_log2;  // scale * log2(e)
  float shift;       // log2 of the scale of a probability at the reference
};

template <int D>
struct Lay {
  static constexpr uint32_t boxes = D / 64;               // 64-column boxes of a tile
  static constexpr uint32_t qtile = boxes * 16384, kvtile = boxes * 8192;  // bytes
  static constexpr uint32_t stages = 4;                   // of the ring; a stage holds V of one key tile and K of the
  static constexpr uint32_t stage = 2 * kvtile;           // one two on: what the MMA warp takes in one step
  static constexpr uint32_t q = 0;                        // two query tiles
  static constexpr uint32_t kv = 2 * qtile;
  static constexpr uint32_t out = kv + stages * stage;    // [8 warps][32 rows][32 columns] of outputs
  static constexpr uint32_t bars = out + 16384;
  static constexpr uint32_t misc = bars + 8 * (2 * stages + 20);
  static constexpr uint32_t redo = misc + 64;             // one bit per item of this CTA
  static constexpr uint32_t bytes = redo + kMaxItems / 8;
  static constexpr uint32_t alloc = bytes + 1024;
};

// Barriers behind the ring's full[stages], empty[stages]; two each, one per query
// tile, or four, one per tile and score buffer.
// Upper half of the operands' shared-memory descriptors: 1024 bytes between groups
// of 8 rows, descriptor version 1, 128-byte swizzle.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (uint32_t(kSw128) << 29);
enum { B_Q = 0, B_QE = 2, B_S = 4, B_P = 8, B_V = 12, B_O = 14, B_OE = 16, B_COUNT = 18 };

// Four K = 16 steps of a product, issued by one elected lane of the converged
// warp.  The descriptors' upper halves are constants and their lower halves
// advance by constants, so that a step costs a few instructions: with two busy
// softmax warps beside it the issuing warp is what the products wait for first.
__device__ __forceinline__ void mma4_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                        uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e, t;\n\t.reg .b64 a, b;\n\t.reg .b32 x, y;\n\t"
      "setp.ne.b32 p, %6, 0;\n\tsetp.eq.b32 t, 0, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
      "mov.b64 a, {%1, %2};\n\tmov.b64 b, {%3, %4};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n\t"
      "add.u32 x, %1, 2;\n\tadd.u32 y, %3, 2;\n\tmov.b64 a, {x, %2};\n\tmov.b64 b, {y, %4};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, t;\n\t"
      "add.u32 x, %1, 4;\n\tadd.u32 y, %3, 4;\n\tmov.b64 a, {x, %2};\n\tmov.b64 b, {y, %4};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, t;\n\t"
      "add.u32 x, %1, 6;\n\tadd.u32 y, %3, 6;\n\tmov.b64 a, {x, %2};\n\tmov.b64 b, {y, %4};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, t;\n\t}\n" ::"r"(d_tmem),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// A from TMEM (8 columns a step), B with its steps 2048 bytes apart.
__device__ __forceinline__ void mma4_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e, t;\n\t.reg .b64 b;\n\t.reg .b32 x, y;\n\t"
      "setp.ne.b32 p, %5, 0;\n\tsetp.eq.b32 t, 0, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t"
      "add.u32 x, %1, 8;\n\tadd.u32 y, %2, 128;\n\tmov.b64 b, {y, %3};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %4, t;\n\t"
      "add.u32 x, %1, 16;\n\tadd.u32 y, %2, 256;\n\tmov.b64 b, {y, %3};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %4, t;\n\t"
      "add.u32 x, %1, 24;\n\tadd.u32 y, %2, 384;\n\tmov.b64 b, {y, %3};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %4, t;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), 
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// How far (log2) a row's probabilities may pass 1 before its reference follows
// the maximum, and the scale that they get before they are rounded, which the sum
// shares, so that it cancels.
// fp16 has a grid of 2^-24 and ends at 2^16: with the reference at 2^11 a
// probability is exact to 2^-36, or to its own half step (at 1, with a slack of 8,
// keys 15 nats below a dominant sink were 8 half steps off and those 18 below it
// lost); a factor of 2 is left for the exponent's rounding at scores of millions.
// A smaller slack has O scaled more often: a call of 1 x 16384 tokens, 32/8 heads of
// 128, window 4096, takes 985 to 996 us at 8 and at 4 alike, 1013 at 3, 1071 at 2.
// bf16 keeps its accuracy at any scale: it takes the slack and the number of keys
// back, so that sums of values near the end of fp32's range stay in it, as their
// average does (values below some 2^-100 lose bits instead).
template <typename T> constexpr float kSlack = Cvt<T>::kIsBf16 ? 8.f : 4.f;
float shift_of(int dtype, long long keys) {
  return dtype == GDN_DTYPE_F16 ? 11.f : -kSlack<__nv_bfloat16> - float(std::ceil(std::log2(double(keys))));
}

// Two fp32 operations in one instruction.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 f2_get(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 f2_add(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

// The larger of three; NaN if one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <typename T> struct Pair;
template <> struct Pair<__half> {
  static __device__ __forceinline__ __half2 zero() { return __floats2half2_rn(0.f, 0.f); }
  using V = __half2;
};
template <> struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ __nv_bfloat162 zero() { return __floats2bfloat162_rn(0.f, 0.f); }
  using V = __nv_bfloat162;
};

// One of a work item's two query tiles: which rows it has and which keys they see.
struct Rows {
  int p0, p1;  // positions of its first row and of its last one that exists (p1 < p0: no rows)
  int len, window;

  // whether it has a row that sees anything (then its first row sees itself)
  __device__ __forceinline__ bool used() const { return p1 >= p0 && p0 < len; }
};

// The key tiles, by their order in an item, that one query tile sees: some of the
// sinks' first, then a run of the window's.
struct Seen {
  int sinks, from, to;
  __device__ __forceinline__ bool operator()(int u) const { return u >= 0 && u <= to && (u < sinks || u >= from); }
  __device__ __forceinline__ int first() const { return sinks > 0 ? 0 : from; }
  __device__ __forceinline__ int last() const { return to; }
};

// A work item and its key tiles, in order: those of the sinks, then those of the window.
// (All scalars: an array indexed by the tile would live in local memory, and
// with this much shared memory taken, that means L2.)
struct Item {
  int b, hy, hk, row0;  // hy: the (first) query head
  int len, count;
  int sink_tiles;  // key tiles that hold sinks
  int n_sink, w0;  // order: tiles 0 .. n_sink - 1, then w0, w0 + 1 ...

  __device__ __forceinline__ int key0(int u) const { return (u < n_sink ? u : w0 + (u - n_sink)) * kKeys; }
  // (The first row that a query tile has sees itself, so there always is a run of the window's.)
  __device__ __forceinline__ Seen seen(const Rows& r) const {
    if (!r.used()) return Seen{0, 0, -1};
    const int lo = r.p0 - r.window + 1;
    const int from = (lo > 0 ? lo / kKeys : 0) - w0 + n_sink, to = (r.p1 < len ? r.p1 : len - 1) / kKeys - w0 + n_sink;
    return Seen{sink_tiles < from ? sink_tiles : from, from, to};
  }
  __device__ __forceinline__ int row(const Params& P, int x) const { return row0 + (P.pair_heads ? 0 : x * kTile); }
  __device__ __forceinline__ int head(const Params& P, int x) const { return hy + (P.pair_heads ? x : 0); }
  __device__ __forceinline__ Rows rows(const Params& P, int x) const {
    const int r = row(P, x);
    const int p0 = P.S - P.T + r;
    return Rows{p0, x && P.single ? p0 - 1 : P.S - P.T + (r + kTile < P.T ? r + kTile : P.T) - 1, len, P.window};
  }
};

__device__ __forceinline__ Item make_item(const Params& P, int i) {
  Item it;
  // Row tiles from the last to the first: early rows see fewer keys, and short
  // items at the end fill the last round.
  const int nb = P.items / P.nx, x = i / nb, y = i - x * nb;
  it.row0 = (P.nx - 1 - x) * (P.pair_heads || P.single ? kTile : 2 * kTile);
  it.b = y / P.ny;
  it.hy = (y - it.b * P.ny) * (P.pair_heads ? 2 : 1);
  it.hk = it.hy / P.G;
  it.len = P.S;
  if (P.lengths) {
    it.len = __shfl_sync(0xffffffffu, P.lengths[it.b], 0);
    it.len = it.len < 0 ? 0 : (it.len > P.S ? P.S : it.len);
  }
  const Rows r0 = it.rows(P, 0), r1 = it.rows(P, 1);
  int end = r1.p1 > r0.p1 ? r1.p1 : r0.p1;
  if (end > it.len - 1) end = it.len - 1;
  it.sink_tiles = P.sinks > 0 ? (P.sinks - 1) / kKeys + 1 : 0;
  it.n_sink = it.w0 = it.count = 0;
  if (r0.p0 >= it.len) return it;
  const int lo = r0.p0 - P.window + 1;
  it.w0 = lo > 0 ? lo / kKeys : 0;
  it.n_sink = it.sink_tiles < it.w0 ? it.sink_tiles : it.w0;  // w0: the sinks' tiles run into the window's
  it.count = it.n_sink + (end / kKeys - it.w0 + 1);
  return it;
}

// One column of this thread's TMEM lane (warp-collective).
__device__ __forceinline__ uint32_t tmem_ld1w(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(r)
               : "r"(taddr)
               : "memory");
  return r;
}

// O (+)= P V of one key tile over this row's visible keys alone, on the CUDA
// cores: for tiles whose values are not all finite.  P is read back from TMEM.
template <typename T, int D>
__device__ __noinline__ void sum_visible(uint32_t tm_p, uint32_t tm_o, const uint8_t* vt, bool first, int k0,
                                         int last, int behind, int sinks) {
  for (int c0 = 0; c0 < D; c0 += 32) {
    float o[32];
    uint32_t ou[32];
    if (first) {
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = 0.f;
    } else {
      tmem_ld32w(tm_o + c0, o);
    }
    for (int j = 0; j < kKeys; ++j) {
      const float2 pp = Cvt<T>::unpack(tmem_ld1w(tm_p + (j >> 1)));
      const float pj = (j & 1) ? pp.y : pp.x;
      const int kj = k0 + j;
      if (kj <= last && (kj > behind || kj < sinks)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 w =
              *reinterpret_cast<const uint4*>(vt + (c0 >> 6) * 8192 + sw128_off(j, ((c0 & 63) >> 3) + i));
          const float2 a = Cvt<T>::unpack(w.x), b = Cvt<T>::unpack(w.y), c = Cvt<T>::unpack(w.z),
                       d = Cvt<T>::unpack(w.w);
          o[8 * i] = fmaf(pj, a.x, o[8 * i]);
          o[8 * i + 1] = fmaf(pj, a.y, o[8 * i + 1]);
          o[8 * i + 2] = fmaf(pj, b.x, o[8 * i + 2]);
          o[8 * i + 3] = fmaf(pj, b.y, o[8 * i + 3]);
          o[8 * i + 4] = fmaf(pj, c.x, o[8 * i + 4]);
          o[8 * i + 5] = fmaf(pj, c.y, o[8 * i + 5]);
          o[8 * i + 6] = fmaf(pj, d.x, o[8 * i + 6]);
          o[8 * i + 7] = fmaf(pj, d.y, o[8 * i + 7]);
        }
      }
      __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) ou[i] = __float_as_uint(o[i]);
    tmem_st32(tm_o + c0, ou);
    tmem_wait_st();
  }
}

// Masked scores of 32 keys: this row's visible keys are those up to hi, from lo on or below sk.
__device__ __forceinline__ void mask_row(float* s, int hi, int lo, int sk) {
  // bits of the columns < n
  auto below = [](int n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); };
  const uint32_t see = below(hi + 1) & (~below(lo) | below(sk));
#pragma unroll
  for (int c = 0; c < 32; ++c)
    if (!(see & (1u << c))) s[c] = -INFINITY;
}

// Whether a value of this thread's key row of the tile is not finite (times 0 it is NaN).
template <typename T, int D>
__device__ __noinline__ bool row_not_finite(const uint8_t* vt, int r) {
  using V2 = typename Pair<T>::V;
  V2 acc = Pair<T>::zero();
  for (int c = 0; c < D / 8; ++c) {
    const uint4 w = *reinterpret_cast<const uint4*>(vt + (c >> 3) * 8192 + sw128_off(r, c & 7));
    acc = __hfma2(*reinterpret_cast<const V2*>(&w.x), Pair<T>::zero(), acc);
    acc = __hfma2(*reinterpret_cast<const V2*>(&w.y), Pair<T>::zero(), acc);
    acc = __hfma2(*reinterpret_cast<const V2*>(&w.z), Pair<T>::zero(), acc);
    acc = __hfma2(*reinterpret_cast<const V2*>(&w.w), Pair<T>::zero(), acc);
  }
  const float z = __low2float(acc) + __high2float(acc);
  return z != z;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) window_attn_kernel(const __grid_constant__ Params P) {
  using L = Lay<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + L::bars);
  uint64_t* empty = full + L::stages;
  uint64_t* bars = empty + L::stages;
  uint32_t* tmem_base_p = reinterpret_cast<uint32_t*>(sm + L::misc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + L::misc + 4);
  volatile int* skip_pv = reinterpret_cast<volatile int*>(sm + L::misc + 8);  // per score buffer: its product is already in O
  volatile int* any_redo = reinterpret_cast<volatile int*>(sm + L::misc + 24);
  uint32_t* redo = reinterpret_cast<uint32_t*>(sm + L::redo);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // known to be uniform: roles may use uniform registers
  const uint32_t sb = smem_u32(sm);

  if (tid == 0) {
    for (uint32_t i = 0; i < L::stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 2);  // both query tiles' products
    }
    for (int i = 0; i < B_COUNT; ++i) {
      const bool softmax = (i >= B_P && i < B_P + 4) || i >= B_OE;  // arrived at by a group's warps
      mbar_init(&bars[i], softmax ? kSoftmaxWarps / 2 : 1);
    }
    *abort_flag = 0;
    *any_redo = 0;
    for (int i = 0; i < 4; ++i) skip_pv[i] = 0;
    fence_mbar_init();
  }
  for (int i = tid; i < kMaxItems / 32; i += kThreads) redo[i] = 0;
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_base_p, kTmCols);
    tmem_relinquish();
  }
  __syncthreads();
  tc_fence_after();
  // All 512 columns are this CTA's, so they start at 0: a constant.
  constexpr uint32_t tmem = 0;

  // A second, careful pass follows if the first one noted any item; all warps meet in between.
  auto again = [&](bool careful) {
    named_bar(kBarAll, kThreads);
    return !careful && *any_redo && !*abort_flag;
  };
  // Counts over all items and passes, for the barriers' phases:
  uint32_t nkv = 0;           // ring stages used
  uint32_t nq0 = 0, nq1 = 0;  // items that used query tile 0, 1 (a role of one tile: the first)
  uint32_t ns0 = 0, np0 = 0;  // key tiles of the role's query tile: scores, products
  bool ok = true;

  if (warp >= kSoftmaxWarps) {
    bool careful = false;
    do {
      if (warp == kTmaWarp) {
        // -------------------------------------------- producer: Q tiles, then the ring's stages, V of tile u and K of u + 2
        for (int j = 0, i = blockIdx.x; i < P.items && ok; ++j, i += gridDim.x) {
          if (careful && !(redo[j >> 5] >> (j & 31) & 1)) continue;
          const Item it = make_item(P, i);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            uint32_t& nq = x ? nq1 : nq0;
            if (!ok || !it.rows(P, x).used()) continue;
            if (nq > 0) ok = mbar_wait_warp(&bars[B_QE + x], (nq - 1) & 1, abort_flag);
            if (!ok) continue;
            if (lane == 0) {
              mbar_arrive_expect_tx(&bars[B_Q + x], L::qtile);
              for (uint32_t c = 0; c < L::boxes; ++c)
                tma_load_4d(sm + L::q + x * L::qtile + c * 16384, &P.tm_q, &bars[B_Q + x], c * 64, it.row(P, x),
                            it.head(P, x) * P.qh, it.b * P.qb);
            }
            __syncwarp();
            ++nq;
          }
          for (int u = -2; it.count > 0 && u < it.count && ok; ++u) {
            const uint32_t s = nkv % L::stages;
            if (nkv >= L::stages) ok = mbar_wait_warp(&empty[s], (nkv / L::stages - 1) & 1, abort_flag);
            if (!ok) break;
            if (lane == 0) {
              uint8_t* dst = sm + L::kv + s * L::stage;
              const bool v = u >= 0, k = u + 2 < it.count;
              mbar_arrive_expect_tx(&full[s], (v + k) * L::kvtile);
              for (uint32_t c = 0; c < L::boxes; ++c) {
                if (v) tma_load_4d(dst + c * 8192, &P.tm_v, &full[s], c * 64, it.key0(u), it.hk * P.vh, it.b * P.vb);
                if (k)
                  tma_load_4d(dst + L::kvtile + c * 8192, &P.tm_k, &full[s], c * 64, it.key0(u + 2), it.hk * P.kh,
                              it.b * P.kb);
              }
            }
            __syncwarp();
            ++nkv;
          }
        }
      } else if (warp == kMmaWarp || warp == kMmaWarp + 1) {
        // -------------------------------------------- MMA issue (the whole warp; elect.sync inside)
        constexpr uint32_t kBf16 = Cvt<T>::kIsBf16;
        constexpr uint32_t id_s = idesc_f16(128, kKeys, kBf16, 0, 0), id_o = idesc_f16(128, D, kBf16, 0, 1);
        const int x = warp - kMmaWarp;
        const uint32_t tm_s = tmem + kTmS + x * 128, tm_o = tmem + kTmO + x * 128;
        const uint32_t q_lo = ((sb + L::q + x * L::qtile) >> 4) | (1u << 16);
        for (int j = 0, i = blockIdx.x; i < P.items && ok; ++j, i += gridDim.x) {
          if (careful && !(redo[j >> 5] >> (j & 31) & 1)) continue;
          const Item it = make_item(P, i);
          if (it.count == 0) continue;
          const Rows rows = it.rows(P, x);
          const Seen seen = it.seen(rows);
          const int first = seen.first(), last = seen.last();
          // Scores run two key tiles ahead of the products, so that a softmax group
          // finds its next tile's ready.
          for (int u = -2; u < it.count && ok; ++u) {
            const uint32_t s = nkv % L::stages;
            ok = mbar_wait_warp(&full[s], (nkv / L::stages) & 1, abort_flag);
            ++nkv;
            if (ok && seen(u)) {
              const uint32_t v_lo = ((sb + L::kv + s * L::stage) >> 4) | (512u << 16);  // 8192 bytes between its boxes
              const bool fresh = u == first;  // this item's first product: O is written, not added to
              const uint32_t buf = np0 & 1;
              ok = mbar_wait_warp(&bars[B_P + 2 * x + buf], (np0 >> 1) & 1, abort_flag);
              // the last item's output must have left O
              if (ok && fresh && nq0 > 0) ok = mbar_wait_warp(&bars[B_OE + x], (nq0 - 1) & 1, abort_flag);
              if (!ok) break;
              ++np0;
              tc_fence_after();
              if (!careful || !skip_pv[2 * x + buf]) mma4_ts(tm_o, tm_s + buf * 64, v_lo, kDescHi, id_o, !fresh);
              mma_commit_warp(&bars[B_V + x]);
              if (u == last) mma_commit_warp(&bars[B_O + x]);
            }
            // A score buffer is written again two tiles on: in issue order after the
            // product that read its probabilities.
            if (ok && seen(u + 2)) {
              const uint32_t k_lo = ((sb + L::kv + s * L::stage + L::kvtile) >> 4) | (1u << 16);
              if (u + 2 == first) ok = mbar_wait_warp(&bars[B_Q + x], nq0 & 1, abort_flag);
              if (!ok) break;
              const uint32_t buf = ns0 & 1;
              ++ns0;
#pragma unroll
              for (uint32_t c = 0; c < L::boxes; ++c)
                mma4_ss(tm_s + buf * 64, q_lo + c * 1024, kDescHi, k_lo + c * 512, kDescHi, id_s, c);
              mma_commit_warp(&bars[B_S + 2 * x + buf]);
              if (u + 2 == last) mma_commit_warp(&bars[B_QE + x]);
            }
            if (ok) mma_commit_warp(&empty[s]);
          }
          nq0 += rows.used();
        }
      }
    } while (careful = again(careful), careful);
  } else {
    // ------------------------------------------------ softmax: thread = one query row of tile x
    // After an abort a warp runs on without waiting or computing, so that the
    // group's barriers still meet.
    const int x = warp >> 2, quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_base = uint32_t(quarter * 32) << 16;
    const uint32_t tm_s0 = tmem + lane_base + kTmS + x * 128, tm_o = tmem + lane_base + kTmO + x * 128;
    const float sl2 = P.scale_log2;
    // Two copies of the loop: the careful one's calls would cost the other its registers.
    auto softmax_pass = [&](auto kind) {
      constexpr bool careful = decltype(kind)::value;
#pragma unroll 1
      for (int i = blockIdx.x; i < P.items; i += gridDim.x) {
        const int j = (i - int(blockIdx.x)) / int(gridDim.x);
        if (careful && !(redo[j >> 5] >> (j & 31) & 1)) continue;
        // What the loop below keeps of the item, in few registers (a spilled one
        // would come from L2): its key tiles in this tile's own order are n_sink
        // ones from key 0, then those from key `from` on; those with k0 <= all_to
        // and either k0 > all_from or k0 + kKeys <= sinks are whole.
        int tiles, n_sink, from, len, p, all_to, all_from;
        const uint32_t base = nkv + 2;  // ring stage of the item's first V
        {
          const Item it = make_item(P, i);
          const Rows rows = it.rows(P, x);
          if (it.count > 0) nkv += it.count + 2;
          if (!rows.used()) {
            if (rows.p1 >= rows.p0 && it.row(P, x) + r < P.T) {
              T* op = static_cast<T*>(P.o) + P.so_b * it.b + P.so_t * (long long)(it.row(P, x) + r) + P.so_h * it.head(P, x);
              for (int c = 0; c < D / 8; ++c) reinterpret_cast<uint4*>(op)[c] = make_uint4(0, 0, 0, 0);
            }
            continue;
          }
          const Seen seen = it.seen(rows);
          n_sink = seen.sinks;
          from = it.key0(seen.from);
          tiles = n_sink + seen.to - seen.from + 1;
          len = it.len;
          p = rows.p0 + r;
          all_to = (rows.p0 < len - 1 ? rows.p0 : len - 1) - (kKeys - 1);
          all_from = rows.p1 - P.window;
        }
        float m = -INFINITY, l = 0.f;  // running reference maximum (raw scores); sum
#pragma unroll 1
        for (int t = 0; t < tiles; ++t) {
          const int k0 = t < n_sink ? t * kKeys : from + (t - n_sink) * kKeys;
          const bool cut = k0 > all_to || (k0 <= all_from && k0 + kKeys > P.sinks);
          const uint32_t buf = ns0 & 1, before = (ns0 - 1) & 1;
          const uint32_t tm_s = tm_s0 + buf * 64;
          if (ok) ok = mbar_wait_warp(&bars[B_S + 2 * x + buf], (ns0 >> 1) & 1, abort_flag);
          float s[64];
          float mt = 0.f;
          if (ok) {
            tc_fence_after();
            tmem_ld32x2w(tm_s, s, tm_s + 32, s + 32);
            if (cut) {
              const int hi = p < len ? p : -1;
              mask_row(s, hi - k0, p - P.window + 1 - k0, P.sinks - k0);
              mask_row(s + 32, hi - k0 - 32, p - P.window + 1 - k0 - 32, P.sinks - k0 - 32);  // rows behind the sequence see none
            }
            // a NaN among the scores becomes the maximum, and so the row's output
            float mx[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e] = max3(s[e], s[4 + e], s[8 + e]);
#pragma unroll
            for (int c = 12; c < 60; c += 8)
#pragma unroll
              for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], s[c + e], s[c + 4 + e]);
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], s[60 + e], s[60 + e]);
            mt = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]);
          }
          ++ns0;
          if (ok) {
            // The reference follows the maximum only when a probability would
            // pass the slack: most tiles then leave O as it is.
            const bool up = !((mt - m) * sl2 <= kSlack<T>) && mt != -INFINITY;
            if (__any_sync(0xffffffffu, up)) {
              const float corr = !up ? 1.f : (m == -INFINITY ? 0.f : fast_exp2((m - mt) * sl2));
              if (up) m = mt == INFINITY ? NAN : mt;  // infinity less infinity
              l *= corr;
              if (t > 0) {
                // the product before has to be in O
                ok = mbar_wait_warp(&bars[B_V + x], before, abort_flag);
                if (ok) {
                  tc_fence_after();
#pragma unroll 1
                  for (int c = 0; c < D; c += 16) {
                    float o[16];
                    tmem_ld16w(tm_o + c, o);
                    uint32_t ou[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) ou[e] = __float_as_uint(o[e] * corr);
                    tmem_st16(tm_o + c, ou);
                  }
                }
              }
            }
            const float ms = m == -INFINITY ? 0.f : m * sl2;
            const F2 sl = f2(sl2, sl2), nm = f2(P.shift - ms, P.shift - ms);
            F2 sum0 = f2(0.f, 0.f), sum1 = sum0;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t pk[16];
#pragma unroll
              for (int c = 0; c < 16; ++c) {
                float2 e = f2_get(f2_fma(f2(s[32 * h + 2 * c], s[32 * h + 2 * c + 1]), sl, nm));
                e = make_float2(fast_exp2(e.x), fast_exp2(e.y));
                if (c & 1)
                  sum1 = f2_add(sum1, f2(e.x, e.y));
                else
                  sum0 = f2_add(sum0, f2(e.x, e.y));
                pk[c] = Cvt<T>::pack(e.x, e.y);
              }
              tmem_st16(tm_s + 16 * h, pk);
            }
            const float2 sum = f2_get(f2_add(sum0, sum1));
            l += sum.x + sum.y;
            tmem_wait_st();
          }
          if (careful) {
            bool slow = false;
            if (cut) {
              const Item it = make_item(P, i);
              const uint32_t n = base + (t < n_sink ? t : it.seen(it.rows(P, x)).from + (t - n_sink));
              const uint8_t* vt = sm + L::kv + n % L::stages * L::stage;
              if (ok) ok = mbar_wait_warp(&full[n % L::stages], (n / L::stages) & 1, abort_flag);
              if (ok && t > 0) ok = mbar_wait_warp(&bars[B_V + x], before, abort_flag);
              tc_fence_before();
              slow = bar_any(kBarGroup + x, 128, ok && r < kKeys && row_not_finite<T, D>(vt, r));
              if (slow && ok) {
                tc_fence_after();
                sum_visible<T, D>(tm_s, tm_o, vt, t == 0, k0, p < len ? p : -1, p - P.window, P.sinks);
              }
            }
            if (ok && r == 0) skip_pv[2 * x + buf] = slow;
            __threadfence_block();
          }
          if (ok) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars[B_P + 2 * x + buf]);
          }
        }
        // -------------------------------------------- o = O / l
        if (ok) ok = mbar_wait_warp(&bars[B_O + x], nq0 & 1, abort_flag);
        if (ok) {
          tc_fence_after();
          const Item it = make_item(P, i);
          const bool live = p < len;
          const float inv = 1.f / l;
          float odd = 0.f;  // NaN if some output is not finite
          // Rows leave through shared memory, so that a store covers whole sectors.
          uint8_t* stage = sm + L::out + warp * 2048;
          const int row = it.row(P, x) + quarter * 32;  // this warp's first
          T* op = static_cast<T*>(P.o) + P.so_b * it.b + P.so_h * it.head(P, x) + P.so_t * (long long)row;
#pragma unroll 1
          for (int part = 0; part < D / 32; ++part) {
            float o[32];
            tmem_ld32w(tm_o + 32 * part, o);
            if (part == D / 32 - 1) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&bars[B_OE + x]);
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint4 w;
              uint32_t* wp = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float a = o[8 * c + 2 * e] * inv, b2 = o[8 * c + 2 * e + 1] * inv;
                odd = fmaf(a, 0.f, odd);
                odd = fmaf(b2, 0.f, odd);
                wp[e] = live ? Cvt<T>::pack(a, b2) : 0u;
              }
              *reinterpret_cast<uint4*>(stage + sw64_off(lane, c)) = w;
            }
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int rr = 8 * c + (lane >> 2);
              const uint4 w = *reinterpret_cast<const uint4*>(stage + sw64_off(rr, lane & 3));
              if (row + rr < P.T) reinterpret_cast<uint4*>(op + P.so_t * (long long)rr + 32 * part)[lane & 3] = w;
            }
            __syncwarp();
          }
          if (!careful && row + lane < P.T && live && odd != odd) {
            atomicOr(&redo[j >> 5], 1u << (j & 31));
            *any_redo = 1;
          }
        }
        ++nq0;
      }
    };
    softmax_pass(std::false_type{});
    if (again(false)) {
      softmax_pass(std::true_type{});
      again(true);
    }
  }
  // On an abort the loads and products still in flight end before the CTA leaves.
  if (warp == kTmaWarp && *abort_flag) {
    volatile int never = 0;
    if (nq0 > 0) mbar_wait(&bars[B_Q], (nq0 - 1) & 1, &never);
    if (nq1 > 0) mbar_wait(&bars[B_Q + 1], (nq1 - 1) & 1, &never);
    for (uint32_t n = nkv > L::stages ? nkv - L::stages : 0; n < nkv; ++n)
      mbar_wait(&full[n % L::stages], (n / L::stages) & 1, &never);
  }
  if ((warp == kMmaWarp || warp == kMmaWarp + 1) && *abort_flag) {
    // a commit of its own: every product this warp has issued has ended when it arrives
    uint64_t* done = &bars[B_COUNT + warp - kMmaWarp];
    if (lane == 0) {
      mbar_init(done, 1);
      fence_mbar_init();
    }
    __syncwarp();
    mma_commit_warp(done);
    volatile int never = 0;
    mbar_wait(done, 0, &never);
    __syncwarp();
  }
  __syncthreads();
  if (tid == 0 && *abort_flag && P.status) atomicOr(P.status, 1 << GDN_ERR_TIMEOUT);
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmCols);
  }
}

// ------------------------------------------------------------------ host side
int validate(const gdn_window_attn_args* a) {
  if (a == nullptr || a->abi_version != GDN_B200_ABI_VERSION) return GDN_ERR_INVALID_ARGUMENT;
  if (a->B < 1 || a->T < 1 || a->S < a->T || a->H < 1 || a->HK < 1 || a->D < 1) return GDN_ERR_INVALID_ARGUMENT;
  if (a->H % a->HK != 0 || a->window < 1 || a->sinks < 0) return GDN_ERR_INVALID_ARGUMENT;
  if (!(a->scale > 0.f) || a->scale > 1.0e30f) return GDN_ERR_INVALID_ARGUMENT;
  if (a->dtype != GDN_DTYPE_F16 && a->dtype != GDN_DTYPE_BF16)
    return a->dtype == GDN_DTYPE_F32 ? GDN_ERR_UNSUPPORTED : GDN_ERR_INVALID_ARGUMENT;
  if (!a->q || !a->k || !a->v || !a->o) return GDN_ERR_INVALID_ARGUMENT;
  if (a->D != 64 && a->D != 128) return GDN_ERR_UNSUPPORTED;
  if (a->B > 65535 || a->H > 65535 || a->S > (1 << 30) || a->window > (1 << 30) || a->sinks > (1 << 30))
    return GDN_ERR_UNSUPPORTED;
  const void* ptr[4] = {a->q, a->k, a->v, a->o};
  const int64_t* st[4] = {a->q_stride, a->k_stride, a->v_stride, a->o_stride};
  for (int i = 0; i < 4; ++i) {
    if (reinterpret_cast<uintptr_t>(ptr[i]) % 16) return GDN_ERR_ALIGNMENT;
    const int n[3] = {a->B, i == 1 || i == 2 ? a->S : a->T, i == 1 || i == 2 ? a->HK : a->H};
    // stride 0: an input that is expanded over the batch or the heads
    for (int j = 0; j < 3; ++j)
      if (n[j] > 1 && (st[i][j] < 0 || st[i][j] % 8 != 0 || (st[i][j] == 0 && (i == 3 || j == 1)))) return GDN_ERR_ALIGNMENT;
  }
  if (reinterpret_cast<uintptr_t>(a->lengths) % 4) return GDN_ERR_ALIGNMENT;
  return GDN_OK;
}

bool make_map(CUtensorMap* m, const gdn_window_attn_args* a, const void* base, const int64_t* st, int rows, int heads,
              int box_rows) {
  const CUtensorMapDataType dt =
      a->dtype == GDN_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  // a dimension of stride 0 is one element
  const uint64_t dims[4] = {uint64_t(a->D), uint64_t(rows), st[2] != 0 ? uint64_t(heads) : 1, st[0] != 0 ? uint64_t(a->B) : 1};
  // and one of one element may come with any stride: it is never taken
  auto bytes = [&](int64_t s, int n) { return n > 1 && s != 0 ? uint64_t(s) * 2 : uint64_t(a->D) * 2; };
  const uint64_t strides[3] = {bytes(st[1], rows), bytes(st[2], heads), bytes(st[0], a->B)};
  const uint32_t box[4] = {64, uint32_t(box_rows), 1, 1};
  return make_tmap(m, dt, 4, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <typename T, int D>
int launch(const Params& p, dim3 grid, cudaStream_t s, int dev) {
  static bool configured[kMaxDevices] = {};
  auto kern = window_attn_kernel<T, D>;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(Lay<D>::alloc)) != cudaSuccess)
      return cuda_failed();
    configured[dev] = true;
  }
  kern<<<grid, kThreads, Lay<D>::alloc, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? GDN_OK : GDN_ERR_CUDA;
}

int run(const gdn_window_attn_args* a, void* stream) {
  const int rc = validate(a);
  if (rc != GDN_OK) return rc;
  int dev = 0;
  if (!device_is_sm100(&dev)) return GDN_ERR_NO_DEVICE;
  Params p;
  memset(&p, 0, sizeof(p));
  if (!make_map(&p.tm_q, a, a->q, a->q_stride, a->T, a->H, kTile) || !make_map(&p.tm_k, a, a->k, a->k_stride, a->S, a->HK, kKeys) ||
      !make_map(&p.tm_v, a, a->v, a->v_stride, a->S, a->HK, kKeys))
    return GDN_ERR_CUDA;
  p.lengths = a->lengths;
  p.o = a->o;
  p.status = a->status;
  p.so_b = a->o_stride[0], p.so_t = a->o_stride[1], p.so_h = a->o_stride[2];
  auto steps = [](int64_t stride) { return stride != 0 ? 1 : 0; };
  p.qb = steps(a->q_stride[0]), p.qh = steps(a->q_stride[2]);
  p.kb = steps(a->k_stride[0]), p.kh = steps(a->k_stride[2]);
  p.vb = steps(a->v_stride[0]), p.vh = steps(a->v_stride[2]);
  p.T = a->T, p.S = a->S, p.HK = a->HK, p.G = a->H / a->HK;
  // a window or sinks past the keys see no more than all of them
  p.window = a->window < a->S ? a->window : a->S;
  p.sinks = a->sinks < a->S ? a->sinks : a->S;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  const long long keys = (long long)p.window + p.sinks;  // that a row sees
  p.shift = shift_of(a->dtype, keys < a->S ? keys : a->S);
  int sms = 0;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms < 1) return cuda_failed();
  // Items of one tile where all of them run at once: a chunk of 3 x 501 rows, 12
  // heads of 64, takes 15.8 us (18.2 in items of two).  With more items than SMs
  // two tiles share the keys fetched, and one's softmax runs under the other's products.
  const int tiles = (a->T + kTile - 1) / kTile;
  p.single = (long long)tiles * a->H * a->B <= sms;
  p.pair_heads = !p.single && p.G % 2 == 0;
  p.nx = p.single || p.pair_heads ? tiles : (tiles + 1) / 2;
  p.ny = p.pair_heads ? a->H / 2 : a->H;
  const long long items = (long long)p.nx * p.ny * a->B;
  if (items > 0x7fff0000LL) return GDN_ERR_UNSUPPORTED;
  p.items = int(items);
  // one CTA per SM, more only where one could not note all its items
  long long ctas = (items + kMaxItems - 1) / kMaxItems;
  if (ctas < sms) ctas = items < sms ? items : sms;
  const dim3 grid{unsigned(ctas)};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf = a->dtype == GDN_DTYPE_BF16;
  if (a->D == 128)
    return bf ? launch<__nv_bfloat16, 128>(p, grid, s, dev) : launch<__half, 128>(p, grid, s, dev);
  return bf ? launch<__nv_bfloat16, 64>(p, grid, s, dev) : launch<__half, 64>(p, grid, s, dev);
}

}  // namespace
}  // namespace wa
}  // namespace gdn

extern "C" int gdn_window_attn_sm100(const gdn_window_attn_args* args, void* stream) {
  return gdn::wa::run(args, stream);
}
