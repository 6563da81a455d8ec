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
// Split.  A CTA owns two tiles of 128 query rows that share their keys: two
// heads of one key head where heads share keys in even groups, else two
// neighbouring tiles of one head.  So every K/V tile fetched feeds two
// products, and while one tile's softmax runs the tensor core works on the
// other's.  Warps: 2 x 4 softmax (one thread per query row), one that
// fetches K/V tiles by TMA, one that issues the MMAs.  TMEM holds both score
// tiles and both outputs; the probabilities overwrite their scores' columns
// and are the second product's TMEM operand, so they never touch shared memory.
//
// Masks.  Only tiles that some mask cuts are masked element by element.  In
// those a key hidden from a row has probability 0, and 0 times a non-finite
// value would still poison the row; so the values of a cut tile are looked
// over, and if one is not finite its product is summed on the CUDA cores over
// visible keys alone.
#include "../../include/gdn_b200.h"
#include "host_util.h"
#include "tc.cuh"
#include "tmap.h"

#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>

namespace gdn {
namespace wa {
namespace {

constexpr int kTile = 128;          // query rows and keys per tile
constexpr int kTmaWarp = 8, kMmaWarp = 9;
// Three warpgroups, so that registers can be moved between them: 168 each at
// launch, then 2 x 216 for the softmax warps and 72 for the others (504 in all).
constexpr int kThreads = 384;
constexpr uint32_t kTmCols = 512;
constexpr uint32_t kTmS = 0, kTmO = 256;  // + 128 x tile

struct Params {
  CUtensorMap tm_q, tm_k, tm_v;
  const int* lengths;
  void* o;
  int* status;
  long long so_b, so_t, so_h;
  int T, S, HK, G;
  int window, sinks;
  int pair_heads;    // the CTA's two tiles are two heads (else two row tiles of one head)
  float scale_log2;  // scale * log2(e)
};

template <int D>
struct Lay {
  static constexpr uint32_t boxes = D / 64;               // 64-column boxes of a tile
  static constexpr uint32_t tile = boxes * 16384;         // bytes of a 128-row tile
  static constexpr uint32_t stages = D == 128 ? 4 : 6;
  static constexpr uint32_t q = 0;                        // two query tiles
  static constexpr uint32_t kv = 2 * tile;                // ring of K and V tiles
  static constexpr uint32_t bars = kv + stages * tile;
  static constexpr uint32_t misc = bars + 8 * (2 * stages + 8);
  static constexpr uint32_t bytes = misc + 64;
  static constexpr uint32_t alloc = bytes + 1024;
};

// barriers behind the ring's full[stages], empty[stages]
enum { B_Q = 0, B_S = 2, B_P = 4, B_O = 6, B_COUNT = 8 };

__device__ __forceinline__ void mma_f16_ts_warp(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                                uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
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
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <int N> __device__ __forceinline__ void regs_more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_less() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <typename T> struct Pair;
template <> struct Pair<__half> {
  static __device__ __forceinline__ __half2 zero() { return __floats2half2_rn(0.f, 0.f); }
  using V = __half2;
};
template <> struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ __nv_bfloat162 zero() { return __floats2bfloat162_rn(0.f, 0.f); }
  using V = __nv_bfloat162;
};

// The CTA's key tiles, in order: those of the sinks, then those of the window.
struct Tiles {
  int n_sink, w0, count;
  int p0[2];       // position of each query tile's first row
  int p1[2];       // and of its last one that exists (p0 - 1: no rows)
  int len, window, sinks;

  __device__ __forceinline__ int key0(int u) const { return (u < n_sink ? u : w0 + (u - n_sink)) * kTile; }
  // whether some row of query tile x sees a key of the tile at k0
  __device__ __forceinline__ bool sees(int x, int k0) const {
    if (p1[x] < p0[x] || p0[x] >= len || k0 >= len || k0 > p1[x]) return false;
    return k0 < sinks || k0 + kTile > p0[x] - window + 1;
  }
  // whether every row of query tile x sees every key of the tile at k0
  __device__ __forceinline__ bool whole(int x, int k0) const {
    const int k1 = k0 + kTile - 1;
    return k1 <= p0[x] && k1 < len && (k1 < sinks || p1[x] - k0 < window);
  }
};

__device__ __forceinline__ Tiles make_tiles(const Params& P, int len) {
  Tiles t;
  t.len = len;
  t.window = P.window;
  t.sinks = P.sinks;
  const int row0 = blockIdx.x * (P.pair_heads ? kTile : 2 * kTile);
  for (int x = 0; x < 2; ++x) {
    const int r = row0 + (P.pair_heads ? 0 : x * kTile);
    t.p0[x] = P.S - P.T + r;
    const int last = r + kTile < P.T ? r + kTile : P.T;
    t.p1[x] = P.S - P.T + last - 1;
  }
  int end = t.p1[1] > t.p1[0] ? t.p1[1] : t.p1[0];
  if (end > len - 1) end = len - 1;
  if (t.p0[0] >= len || end < 0) {
    t.n_sink = t.w0 = t.count = 0;
    return t;
  }
  const int w1 = end / kTile;
  const int lo = t.p0[0] - P.window + 1;
  t.n_sink = P.sinks > 0 ? (P.sinks - 1) / kTile + 1 : 0;
  t.w0 = lo > 0 ? lo / kTile : 0;
  if (t.n_sink >= t.w0) t.n_sink = t.w0;  // the sinks' tiles run into the window's
  t.count = t.n_sink + (w1 - t.w0 + 1);
  return t;
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
__device__ __noinline__ void sum_visible(uint32_t tm_p, uint32_t tm_o, const uint8_t* vt, bool first, int k0, int last,
                                         int behind, int sinks) {
  for (int c0 = 0; c0 < D; c0 += 32) {
    float o[32];
    uint32_t ou[32];
    if (first) {
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = 0.f;
    } else {
      tmem_ld32w(tm_o + c0, o);
    }
    for (int j = 0; j < kTile; ++j) {
      const float2 pp = Cvt<T>::unpack(tmem_ld1w(tm_p + (j >> 1)));
      const float pj = (j & 1) ? pp.y : pp.x;
      const int kj = k0 + j;
      if (kj <= last && (kj > behind || kj < sinks)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 w =
              *reinterpret_cast<const uint4*>(vt + (c0 >> 6) * 16384 + sw128_off(j, ((c0 & 63) >> 3) + i));
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
  volatile int* skip_pv = reinterpret_cast<volatile int*>(sm + L::misc + 8);  // [2]: the product is already in O
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t sb = smem_u32(sm);

  const int b = blockIdx.z;
  const int hy = P.pair_heads ? 2 * blockIdx.y : blockIdx.y;
  const int hk = hy / P.G;
  const int row0 = blockIdx.x * (P.pair_heads ? kTile : 2 * kTile);
  int len = P.S;
  if (P.lengths) {
    len = P.lengths[b];
    len = len < 0 ? 0 : (len > P.S ? P.S : len);
  }
  const Tiles tl = make_tiles(P, len);

  if (tid == 0) {
    for (uint32_t i = 0; i < L::stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&bars[B_Q + x], 1);
      mbar_init(&bars[B_S + x], 1);
      mbar_init(&bars[B_P + x], 4);
      mbar_init(&bars[B_O + x], 1);
    }
    *abort_flag = 0;
    skip_pv[0] = skip_pv[1] = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_base_p, kTmCols);
    tmem_relinquish();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_base_p;

  if (warp >= 8) {
    regs_less<72>();
  if (warp == kTmaWarp) {
    // ------------------------------------------------ producer: Q tiles, then K0 V0 K1 V1 ...
    int loads = 0;
    bool ok = true;
    if (tl.count > 0) {
      if (lane == 0) {
        for (int x = 0; x < 2; ++x) {
          if (tl.p1[x] < tl.p0[x]) continue;
          mbar_arrive_expect_tx(&bars[B_Q + x], L::tile);
          for (uint32_t c = 0; c < L::boxes; ++c)
            tma_load_4d(sm + L::q + x * L::tile + c * 16384, &P.tm_q, &bars[B_Q + x], c * 64,
                        row0 + (P.pair_heads ? 0 : x * kTile), hy + (P.pair_heads ? x : 0), b);
        }
      }
      for (int u = 0; u < tl.count && ok; ++u) {
        const int k0 = tl.key0(u);
        for (int kv = 0; kv < 2; ++kv, ++loads) {
          const int s = loads % L::stages;
          if (loads >= int(L::stages) && !mbar_wait_warp(&empty[s], (loads / L::stages - 1) & 1, abort_flag)) {
            ok = false;
            break;
          }
          if (lane == 0) {
            mbar_arrive_expect_tx(&full[s], L::tile);
            for (uint32_t c = 0; c < L::boxes; ++c)
              tma_load_4d(sm + L::kv + s * L::tile + c * 16384, kv ? &P.tm_v : &P.tm_k, &full[s], c * 64, k0, hk, b);
          }
          __syncwarp();
        }
      }
      // On an abort the loads still in flight land before the CTA leaves.
      volatile int never = 0;
      for (int x = 0; x < 2; ++x)
        if (*abort_flag && tl.p1[x] >= tl.p0[x]) mbar_wait(&bars[B_Q + x], 0, &never);
      for (int i = loads > int(L::stages) ? loads - int(L::stages) : 0; i < loads && *abort_flag; ++i)
        mbar_wait(&full[i % L::stages], (i / L::stages) & 1, &never);
    }
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------ MMA issue (the whole warp; elect.sync inside)
    constexpr uint32_t kBf16 = Cvt<T>::kIsBf16;
    constexpr uint32_t id_s = idesc_f16(128, 128, kBf16, 0, 0), id_o = idesc_f16(128, D, kBf16, 0, 1);
    bool ok = true;
    uint32_t np[2] = {0, 0}, acc[2] = {0, 0};
    bool got_q[2] = {false, false};
    auto score = [&](int x, int u) {
      const uint32_t q = sb + L::q + x * L::tile, k = sb + L::kv + ((2 * u) % L::stages) * L::tile;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
        mma_f16_ss_warp(tmem + kTmS + x * 128, sdesc(q + (kk >> 2) * 16384 + (kk & 3) * 32, 16, 1024, kSw128),
                        sdesc(k + (kk >> 2) * 16384 + (kk & 3) * 32, 16, 1024, kSw128), id_s, kk > 0);
      mma_commit_warp(&bars[B_S + x]);
    };
    auto wait_kv = [&](int i) { return mbar_wait_warp(&full[i % L::stages], (i / L::stages) & 1, abort_flag); };
    for (int u = -1; u < tl.count && ok; ++u) {
      for (int x = 0; x < 2 && ok; ++x) {
        if (u >= 0 && tl.sees(x, tl.key0(u))) {
          ok = wait_kv(2 * u + 1) && mbar_wait_warp(&bars[B_P + x], np[x] & 1, abort_flag);
          if (!ok) break;
          ++np[x];
          tc_fence_after();
          if (!skip_pv[x]) {
            const uint32_t v = sb + L::kv + ((2 * u + 1) % L::stages) * L::tile;
#pragma unroll
            for (int kk = 0; kk < kTile / 16; ++kk)
              mma_f16_ts_warp(tmem + kTmO + x * 128, tmem + kTmS + x * 128 + kk * 8,
                              sdesc(v + kk * 2048, 16384, 1024, kSw128), id_o, acc[x] | (kk > 0));
          }
          acc[x] = 1;
        }
        // The scores follow their tile's last product on the same issue order,
        // so they overwrite its probabilities only after they were read.
        if (u + 1 < tl.count && tl.sees(x, tl.key0(u + 1))) {
          ok = wait_kv(2 * u + 2);
          if (ok && !got_q[x]) ok = got_q[x] = mbar_wait_warp(&bars[B_Q + x], 0, abort_flag);
          if (!ok) break;
          score(x, u + 1);
        }
      }
      if (ok) {
        if (u >= 0) mma_commit_warp(&empty[(2 * u + 1) % L::stages]);
        if (u + 1 < tl.count) mma_commit_warp(&empty[(2 * u + 2) % L::stages]);
      }
    }
    mma_commit_warp(&bars[B_O]);
    mma_commit_warp(&bars[B_O + 1]);
    volatile int never = 0;
    mbar_wait(&bars[B_O], 0, &never);
  }
  } else {
    regs_more<216>();
    // ------------------------------------------------ softmax: thread = one query row of tile x
    // After an abort a warp runs on without waiting or computing, so that the
    // group's barriers still meet.
    const int x = warp >> 2;
    const int r = tid & 127;
    const int p = tl.p0[x] + r;
    const uint32_t lane_base = uint32_t((warp & 3) * 32) << 16;
    const uint32_t tm_s = tmem + lane_base + kTmS + x * 128, tm_o = tmem + lane_base + kTmO + x * 128;
    const float sl2 = P.scale_log2;
    const int last = p < len ? p : -1;  // the last visible key; rows behind the sequence see none
    float m = -INFINITY, l = 0.f;       // running reference maximum (raw scores) and sum
    bool ok = true, first = true;
    uint32_t ns = 0;
    for (int u = 0; u < tl.count; ++u) {
      const int k0 = tl.key0(u);
      if (!tl.sees(x, k0)) continue;
      const bool cut = !tl.whole(x, k0);
      if (ok) ok = mbar_wait_warp(&bars[B_S + x], ns & 1, abort_flag);
      ++ns;
      if (ok) {
        tc_fence_after();
        float s[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32w(tm_s + c * 32, s + c * 32);
        if (cut) {
          const int hi = last - k0, lo = p - P.window + 1 - k0, sk = P.sinks - k0;
#pragma unroll
          for (int c = 0; c < 128; ++c)
            if (!(c <= hi && (c >= lo || c < sk))) s[c] = -INFINITY;
        }
        float mt = s[0];
#pragma unroll
        for (int c = 1; c < 128; ++c) mt = fmaxf(mt, s[c]);
        // The reference follows the maximum only when a probability would pass
        // 2^8: most tiles then leave O as it is.
        float corr = 1.f;
        if ((mt - m) * sl2 > 8.f || (m == -INFINITY && mt > m)) {
          corr = m == -INFINITY ? 0.f : fast_exp2((m - mt) * sl2);
          m = mt;
          l *= corr;
        }
        if (!first && __any_sync(0xffffffffu, corr != 1.f)) {
          for (int c = 0; c < D; c += 32) {
            float o[32];
            uint32_t ou[32];
            tmem_ld32w(tm_o + c, o);
#pragma unroll
            for (int i = 0; i < 32; ++i) ou[i] = __float_as_uint(o[i] * corr);
            tmem_st32(tm_o + c, ou);
          }
        }
        const float ms = m == -INFINITY ? 0.f : m * sl2;
        float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t pk[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const float e0 = fast_exp2(fmaf(s[64 * h + 2 * c], sl2, -ms));
            const float e1 = fast_exp2(fmaf(s[64 * h + 2 * c + 1], sl2, -ms));
            sum0 += e0;
            sum1 += e1;
            pk[c] = Cvt<T>::pack(e0, e1);
          }
          tmem_st32(tm_s + 32 * h, pk);
        }
        l += sum0 + sum1;
        tmem_wait_st();
      }
      bool slow = false;
      if (cut) {
        const int i = 2 * u + 1;
        const uint8_t* vt = sm + L::kv + (i % L::stages) * L::tile;
        if (ok) ok = mbar_wait_warp(&full[i % L::stages], (i / L::stages) & 1, abort_flag);
        bool bad = false;
        if (ok) {
          // one key per thread; a value that is not finite times 0 is NaN
          using V2 = typename Pair<T>::V;
          V2 acc = Pair<T>::zero();
          for (uint32_t c = 0; c < L::boxes * 8; ++c) {
            const uint4 w = *reinterpret_cast<const uint4*>(vt + (c >> 3) * 16384 + sw128_off(r, c & 7));
            acc = __hfma2(*reinterpret_cast<const V2*>(&w.x), Pair<T>::zero(), acc);
            acc = __hfma2(*reinterpret_cast<const V2*>(&w.y), Pair<T>::zero(), acc);
            acc = __hfma2(*reinterpret_cast<const V2*>(&w.z), Pair<T>::zero(), acc);
            acc = __hfma2(*reinterpret_cast<const V2*>(&w.w), Pair<T>::zero(), acc);
          }
          const float z = __low2float(acc) + __high2float(acc);
          bad = z != z;
        }
        slow = bar_any(1 + x, 128, bad);
        if (slow && ok) sum_visible<T, D>(tm_s, tm_o, vt, first, k0, last, p - P.window, P.sinks);
      }
      first = false;
      if (ok) {
        tc_fence_before();
        if (lane == 0) {
          if ((warp & 3) == 0) skip_pv[x] = slow;
          __threadfence_block();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[B_P + x]);
      }
    }
    // ------------------------------------------------ o = O / l
    if (ok && tl.count > 0) ok = mbar_wait_warp(&bars[B_O + x], 0, abort_flag);
    if (ok) {
      tc_fence_after();
      const int i = row0 + (P.pair_heads ? 0 : x * kTile) + r;
      const int h = hy + (P.pair_heads ? x : 0);
      const bool dead = first || last < 0;
      const float inv = dead ? 0.f : 1.f / l;
      T* op = static_cast<T*>(P.o) + P.so_b * b + P.so_t * (long long)i + P.so_h * h;
      for (int c = 0; c < D; c += 32) {
        float o[32];
        tmem_ld32w(tm_o + c, o);
        if (i < P.T) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint4 w;
            uint32_t* wp = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float a = o[8 * j + 2 * e] * inv, c2 = o[8 * j + 2 * e + 1] * inv;
              wp[e] = dead ? 0u : Cvt<T>::pack(a, c2);
            }
            reinterpret_cast<uint4*>(op + c)[j] = w;
          }
        }
      }
      tc_fence_before();
    }
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
    for (int j = 0; j < 3; ++j)
      if (n[j] > 1 && (st[i][j] <= 0 || st[i][j] % 8 != 0)) return GDN_ERR_ALIGNMENT;
  }
  if (reinterpret_cast<uintptr_t>(a->lengths) % 4) return GDN_ERR_ALIGNMENT;
  return GDN_OK;
}

bool make_map(CUtensorMap* m, const gdn_window_attn_args* a, const void* base, const int64_t* st, int rows, int heads) {
  const CUtensorMapDataType dt =
      a->dtype == GDN_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const uint64_t dims[4] = {uint64_t(a->D), uint64_t(rows), uint64_t(heads), uint64_t(a->B)};
  // a dimension of one element may come with any stride: it is never taken
  auto bytes = [&](int64_t s, int n) { return n > 1 ? uint64_t(s) * 2 : uint64_t(a->D) * 2; };
  const uint64_t strides[3] = {bytes(st[1], rows), bytes(st[2], heads), bytes(st[0], a->B)};
  const uint32_t box[4] = {64, kTile, 1, 1};
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
  if (!make_map(&p.tm_q, a, a->q, a->q_stride, a->T, a->H) || !make_map(&p.tm_k, a, a->k, a->k_stride, a->S, a->HK) ||
      !make_map(&p.tm_v, a, a->v, a->v_stride, a->S, a->HK))
    return GDN_ERR_CUDA;
  p.lengths = a->lengths;
  p.o = a->o;
  p.status = a->status;
  p.so_b = a->o_stride[0], p.so_t = a->o_stride[1], p.so_h = a->o_stride[2];
  p.T = a->T, p.S = a->S, p.HK = a->HK, p.G = a->H / a->HK;
  // a window or sinks past the keys see no more than all of them
  p.window = a->window < a->S ? a->window : a->S;
  p.sinks = a->sinks < a->S ? a->sinks : a->S;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.pair_heads = p.G % 2 == 0;
  const int rows = p.pair_heads ? kTile : 2 * kTile;
  const dim3 grid((a->T + rows - 1) / rows, p.pair_heads ? a->H / 2 : a->H, a->B);
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
