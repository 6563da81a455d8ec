// Gated linear recurrence over the sequence, one independent chain per channel:
//
//     h_t = a_t h_{t-1} + x_t,   o_t = h_t,   a_t = exp(g_t) or sigmoid(g_t)
//
// and its gradients.  With mu_t = a_t lambda_t (the gradient of h_{t-1}):
//
//     lambda_t = do_t + mu_{t+1},   mu_{T+1} = dh_T
//     dx_t = lambda_t,   dg_t = mu_t h_{t-1}  (times 1 - a_t for logits),   dh_0 = mu_1
//
// Both directions are scans of affine maps h -> A h + X, which compose:
// (A2, X2) after (A1, X1) is (A2 A1, A2 X1 + X2).  Memory bounds them: x and g
// are read once and o is written once (dx and dg besides, in the backward).
//
// Split.  A CTA owns 64 channels (32 lanes x 2) and walks tiles of 128 rows;
// consecutive tiles of a chain belong to the up to 16 CTAs of a cluster, which
// advances in strides of that many tiles.  Per stride every warp composes its
// rows, the CTA composes its warps in shared memory and sends its map to every
// CTA of the cluster (distributed shared memory); each then folds the maps
// before its own into the running state, replays its rows with the gates it
// kept in registers, and writes them.  The order of all sums is fixed, so
// results repeat bit for bit, and no CTA waits on global memory.
//
// Loads.  Tiles whose rows are 16-byte aligned come by TMA, issued by one
// thread a stride ahead, while the current stride's maps are exchanged (copies
// that each thread issued for itself took 40 % of the kernel's instructions;
// bulk copies row by row were slower still).  Other tensors (odd sizes or
// strides) take one channel per thread, each thread copying its own rows.
// Rows beyond the sequence get x = 0 and a gate of exactly 1, which keeps the
// arithmetic free of conditions.
//
// The backward walks the strides from the end.  It needs h_{t-1}; instead of
// the rounded outputs it takes the fp32 state at each tile's start, which the
// forward leaves behind, and recomputes the tile from x.
#include "../../include/gdn_b200.h"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>
#include <mutex>

#include "host_util.h"
#include "tc.cuh"
#include "tmap.h"

namespace gdn {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxCluster = 16;

struct GscanParams {
  CUtensorMap tm_x, tm_g, tm_d;  // (D, T, H, B) maps of x, g, d_o, for the tiles that TMA fetches
  const void* x;
  const void* g;
  const void* d_o;  // backward: gradient of o, or NULL (zero)
  const float* h0;
  const float* dht;
  void* o;
  void* dx;
  void* dg;
  float* ht;
  float* dh0;
  float* states;  // [B, NT, C] state before each tile, or NULL (forward only)
  long long xs[3], gs[3], os[3], dos[3], dxs[3], dgs[3];
  int B, T, C, H, D;  // C = H * D channels (H = 1, D = C where all tensors are flat)
  int NT, S;       // tiles of the sequence, CTAs per cluster
  int logits;      // g holds logits: a = sigmoid(g)
  int* status;
};

// ---------------------------------------------------------------- vectors
template <int BYTES> struct Raw;
template <> struct Raw<2> { using T = unsigned short; };
template <> struct Raw<4> { using T = uint32_t; };
template <> struct Raw<8> { using T = uint2; };
template <> struct Raw<16> { using T = uint4; };

template <typename T, int V>
struct Vec {
  using R = typename Raw<sizeof(T) * V>::T;
  union U {
    R r;
    T e[V];
    __device__ U() {}
  };
  static __device__ __forceinline__ R load(const T* p) { return __ldcs(reinterpret_cast<const R*>(p)); }
  // Asynchronous copy into this thread's shared-memory slot; 2-byte vectors
  // (odd 16-bit tensors) are too small for one and are copied at once.
  static __device__ __forceinline__ void fetch(R* slot, const T* p) {
    if constexpr (sizeof(R) >= 4)
      asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(uint32_t(__cvta_generic_to_shared(slot))), "l"(p),
                   "n"(int(sizeof(R)))
                   : "memory");
    else
      *slot = __ldcs(reinterpret_cast<const R*>(p));
  }
  static __device__ __forceinline__ R fill(float v) {
    U u;
#pragma unroll
    for (int i = 0; i < V; ++i) u.e[i] = T(v);
    return u.r;
  }
  static __device__ __forceinline__ void unpack(R r, float* f) {
    U u;
    u.r = r;
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = float(u.e[i]);
  }
  static __device__ __forceinline__ void store(T* p, const float* f) {
    U u;
#pragma unroll
    for (int i = 0; i < V; ++i) u.e[i] = T(f[i]);
    *reinterpret_cast<R*>(p) = u.r;
  }
};

// A tile has 128 rows of 16-bit x or 64 of fp32 x, in the forward (whose tile
// states the backward reads) and the backward alike.  The forward gives them
// to few warps with many rows each: fewer maps to compose, and registers hold
// one value per element.  The backward holds two, so twice the warps.
// Measured for the forward (2 x 4096 tokens, 1 x 65536, 8 x 2048; 2048 channels): 4 warps of
// 32 rows 25.3, 166, 37 us; 8 of 16 rows 24.4, 171, 44; 8 of 8 rows (64-row
// tiles) 25.6, 212, 45.  Four channels per thread instead of two: 25.4, 203, 44.
template <typename XT, bool BWD>
struct Shape {
  static constexpr int W = BWD ? 8 : 4;                                  // warps
  static constexpr int TC = sizeof(XT) == 4 ? 64 : 128;                  // rows of a tile
  static constexpr int R = TC / W;                                       // rows per warp
  static constexpr int T = W * 32;                                       // threads
};
constexpr int kVec = 2;  // channels per thread where TMA fetches the tiles

// Gates.  The hardware's base-2 exponential and reciprocal (2^-22 and 1 ulp) on
// plain products, whose rounding adds |g| eps.  A gate's relative error counts once
// for every row that the state remembers: with a gate that forgets within some
// hundred rows it stays below 1e-4 of the state.  Near 1 it would add up to
// thousands of times 8e-8 (the error measured there), and a constant gate's
// always the same way.  So there the gate is 1 plus a small term that has its own
// relative accuracy: one rounding, 2^-25 below 1, the least that an fp32 gate has.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNear = 0x1p-9f;  // log decays nearer to 0 get their gate as 1 + g + g^2 / 2

template <bool LOGITS>
__device__ __forceinline__ float decay(float g) {
  if constexpr (LOGITS) {
    const float e = ex2(-kLog2e * g), r = rcp(1.f + e);
    return g > 4.f ? fmaf(-e, r, 1.f) : r;  // above 4, 1 - a is below 0.018
  } else {
    const float near = fmaf(g, fmaf(g, 0.5f, 1.f), 1.f);  // g^3 / 6 is below 2^-29.5
    return fabsf(g) < kNear ? near : ex2(kLog2e * g);
  }
}
// The gates of a thread's channels.  Of two log decays at once the products take one
// instruction: with it the small term costs 1 % of the forward (2 x 4096 tokens: 25.3
// -> 25.7 us), without it 3 %.  Logits (1 x 65536 tokens: 166 -> 171 us) do not gain by it (179).
template <bool LOGITS, int V>
__device__ __forceinline__ void decays(const float* g, float* a) {
  if constexpr (!LOGITS && V == 2) {
    uint64_t gg, log2e, half, one;
    float2 z, near;
    asm("mov.b64 %0, {%1, %2};" : "=l"(gg) : "f"(g[0]), "f"(g[1]));
    asm("mov.b64 %0, {%1, %1};" : "=l"(log2e) : "f"(kLog2e));
    asm("mov.b64 %0, {%1, %1};" : "=l"(half) : "f"(0.5f));
    asm("mov.b64 %0, {%1, %1};" : "=l"(one) : "f"(1.f));
    asm("{\n\t.reg .b64 t;\n\t"
        "fma.rn.f32x2 t, %2, %3, %4;\n\tfma.rn.f32x2 t, %2, t, %4;\n\tmov.b64 {%0, %1}, t;\n\t}"
        : "=f"(near.x), "=f"(near.y)
        : "l"(gg), "l"(half), "l"(one));
    asm("{\n\t.reg .b64 t;\n\tmul.rn.f32x2 t, %2, %3;\n\tmov.b64 {%0, %1}, t;\n\t}"
        : "=f"(z.x), "=f"(z.y)
        : "l"(gg), "l"(log2e));
    a[0] = fabsf(g[0]) < kNear ? near.x : ex2(z.x);
    a[1] = fabsf(g[1]) < kNear ? near.y : ex2(z.y);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] = decay<LOGITS>(g[i]);
  }
}
// The backward needs a and, for logits, 1 - a, each with its own relative
// accuracy (1 - a is the gate's gradient, and small where the memory is long):
// s = min(a, 1 - a) = e / (1 + e), e = exp(-|g|), with the sign bit set where s is 1 - a.
template <bool LOGITS>
__device__ __forceinline__ float pack_decay(float g) {
  if (!LOGITS) return decay<false>(g);
  const float e = ex2(-kLog2e * fabsf(g));
  const float s = e * rcp(1.f + e);
  return __uint_as_float(__float_as_uint(s) | (~__float_as_uint(g) & 0x80000000u));
}
template <bool LOGITS>
__device__ __forceinline__ float decay_of(float p) {
  return LOGITS && int(__float_as_uint(p)) < 0 ? 1.f + p : p;
}
__device__ __forceinline__ float slope_of(float p) { return int(__float_as_uint(p)) < 0 ? -p : 1.f - p; }

__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// Shared memory of one CTA, in bytes.  With bulk copies x and d_o have two
// buffers: they are read a second time, when the rows are replayed, so that
// registers hold the gates alone.
template <typename XT, typename GT, typename OT, int V, bool BWD>
struct Smem {
  static constexpr bool kBulk = V > 1;
  using Sh = Shape<XT, BWD>;
  static constexpr int W = Sh::W, R = Sh::R, CB = 32 * V, N = Sh::TC * CB;  // elements of a tile
  static constexpr int nb = kBulk ? 2 : 1;
  static constexpr int x = 0;
  static constexpr int g = x + nb * N * int(sizeof(XT));
  static constexpr int d = g + N * int(sizeof(GT));                        // (backward)
  static constexpr int map = d + (BWD ? nb * N * int(sizeof(OT)) : 0);     // [W][CB] float2
  static constexpr int in = map + W * CB * 8;                         // [W][CB] float or float2
  static constexpr int fx = in + W * CB * (BWD ? 8 : 4);              // [W][CB] float (backward)
  static constexpr int bar = fx + (BWD ? W * CB * 4 : 0);             // mbarriers, the abort flag
  static constexpr int agg = bar + 64;                                     // [2][S][CB] float2
  static constexpr int bytes(int S) { return agg + (S > 1 ? 2 * S * CB * 8 : 0); }
};
enum { B_MAP = 0, B_DATA = 2, B_COUNT = 4 };  // two barriers each, used in turn

// ---------------------------------------------------------------- exchange
// A CTA's map of a stride goes to every CTA of its cluster by asynchronous
// stores that count on the receiver's mbarrier.  Unlike a cluster barrier this
// orders nothing else: no thread waits for its output stores to land, and only
// the column owners wait for the maps.  Two buffers and barriers alternate: a
// CTA sends the maps of stride i + 2 only after it has all those of i + 1,
// whose senders had read stride i's.
__device__ __forceinline__ uint32_t peer_addr(uint32_t local, int rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(local), "r"(rank));
  return a;
}
__device__ __forceinline__ void push_map(uint32_t slot, uint32_t bar, int rank, float2 m) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(
                   peer_addr(slot, rank)),
               "l"((uint64_t(__float_as_uint(m.y)) << 32) | __float_as_uint(m.x)), "r"(peer_addr(bar, rank))
               : "memory");
}

__device__ __forceinline__ float2 compose(float2 later, float2 m) {
  return make_float2(later.x * m.x, fmaf(later.x, m.y, later.y));
}

// Where a CTA works: its chain's batch and columns, its place in the cluster.
struct Place {
  int b, h, d0, width, rank;
  long long col0;  // first column among the B * C of the states
};
__device__ __forceinline__ Place place(const GscanParams& p, int CB) {
  const int nd = (p.D + CB - 1) / CB;
  const int chain = blockIdx.x / p.S;
  Place q;
  q.rank = blockIdx.x - chain * p.S;
  const int hd = chain % (p.H * nd);
  q.b = chain / (p.H * nd);
  q.h = hd / nd;
  q.d0 = (hd - q.h * nd) * CB;
  q.width = p.D - q.d0 < CB ? p.D - q.d0 : CB;
  q.col0 = (long long)q.h * p.D + q.d0;
  return q;
}
__device__ __forceinline__ long long offset(const long long* st, const Place& q) {
  return st[0] * q.b + st[2] * q.h + q.d0;
}

// One tensor's tiles on their way through shared memory.
template <typename T, int V, int R>
struct Tile {
  static constexpr int CB = 32 * V;
  const T* p;        // the CTA's columns at t = 0
  long long stride;  // elements per row

  // One channel per thread: this thread's rows, n of them there.
  __device__ __forceinline__ void own(T* buf, long long t0, int n, bool live, T pad) const {
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      T* slot = buf + (w * R + r) * CB + lane;
      if (r < n && live)
        Vec<T, 1>::fetch(reinterpret_cast<typename Vec<T, 1>::R*>(slot), p + (t0 + w * R + r) * stride + lane);
      else
        *slot = pad;
    }
  }
  static __device__ __forceinline__ const typename Vec<T, V>::R* at(const T* buf, int r) {
    return reinterpret_cast<const typename Vec<T, V>::R*>(buf + ((threadIdx.x >> 5) * R + r) * CB) + (threadIdx.x & 31);
  }
  // Rows n.. of this thread's columns that no copy filled.
  static __device__ __forceinline__ void pad(T* buf, int n, float v) {
    for (int r = n; r < R; ++r)
      *(reinterpret_cast<typename Vec<T, V>::R*>(buf + ((threadIdx.x >> 5) * R + r) * CB) + (threadIdx.x & 31)) =
          Vec<T, V>::fill(v);
  }
};

__device__ __forceinline__ void start(uint64_t* bars, volatile int* abort_flag, int S) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < B_COUNT; ++i) mbar_init(&bars[i], 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  // every barrier is ready before the first copy or map arrives
  if (S > 1)
    cg::this_cluster().sync();
  else
    __syncthreads();
}

// No CTA leaves while a map may still be on its way to it; a wait that ran out is reported.
__device__ __forceinline__ void leave(int S, int* status, const volatile int* abort_flag) {
  if (S > 1)
    cg::this_cluster().sync();
  else
    __syncthreads();
  if (threadIdx.x == 0 && *abort_flag && status) atomicOr(status, 1 << GDN_ERR_TIMEOUT);
}

// A tile's copies are waited for after an abort too: none may land in a CTA that has left.
__device__ __forceinline__ void wait_data(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  volatile int own = 0;
  if (!mbar_wait(bar, parity, &own)) *abort_flag = 1;
}

// Send this CTA's map of a column to the whole cluster, and wait for the others'.
template <int CB>
__device__ __forceinline__ void exchange(float2 m, float2* s_agg, uint64_t* bars, int k, int S, int rank,
                                         volatile int* abort_flag) {
  const int buf = k & 1;
  uint64_t* bar = &bars[B_MAP + buf];
  if (threadIdx.x == 0) mbar_arrive_expect_tx(bar, uint32_t(S * CB * 8));
  const uint32_t mine = smem_u32(s_agg + (buf * S + rank) * CB + threadIdx.x), b = smem_u32(bar);
  for (int r = 0; r < S; ++r) push_map(mine, b, r, m);
  if (!*abort_flag) mbar_wait(bar, (k >> 1) & 1, abort_flag);
}

// ---------------------------------------------------------------- forward
template <typename XT, typename GT, typename OT, int V, bool LOGITS>
__global__ void __launch_bounds__(Shape<XT, false>::T, 4) gscan_fwd_kernel(const __grid_constant__ GscanParams p) {
  using L = Smem<XT, GT, OT, V, false>;
  using VX = Vec<XT, V>;
  using VG = Vec<GT, V>;
  constexpr int R = L::R, W = L::W, CB = L::CB, TC = W * R;
  constexpr bool kBulk = L::kBulk;
  extern __shared__ __align__(128) uint8_t sm[];
  XT* s_x = reinterpret_cast<XT*>(sm + L::x);
  GT* s_g = reinterpret_cast<GT*>(sm + L::g);
  float2* s_map = reinterpret_cast<float2*>(sm + L::map);  // maps of this CTA's warps
  float* s_in = reinterpret_cast<float*>(sm + L::in);      // state before each warp's rows
  float2* s_agg = reinterpret_cast<float2*>(sm + L::agg);  // maps of the cluster's CTAs
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::bar);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + L::bar + 48);

  const Place q = place(p, CB);
  const int S = p.S, rank = q.rank;
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const bool live = lane * V < q.width;
  const Tile<XT, V, R> tx{static_cast<const XT*>(p.x) + offset(p.xs, q), p.xs[1]};
  const Tile<GT, V, R> tg{static_cast<const GT*>(p.g) + offset(p.gs, q), p.gs[1]};
  OT* op = static_cast<OT*>(p.o) + offset(p.os, q) + lane * V;
  const float gpad = LOGITS ? INFINITY : 0.f;  // a = 1
  auto rows_of = [&](int tile, int first, int most) {  // rows first .. first + most of a tile that exist
    const long long t = (long long)tile * TC + first;
    return t >= p.T ? 0 : (p.T - t < most ? int(p.T - t) : most);
  };
  auto fetch = [&](int tile, int k) {
    const long long t0 = (long long)tile * TC;
    if constexpr (kBulk) {
      if (tid == 0) {
        uint64_t* bar = &bars[B_DATA + (k & 1)];
        mbar_arrive_expect_tx(bar, uint32_t(L::N) * uint32_t(sizeof(XT) + sizeof(GT)));
        tma_load_4d(s_x + (k & 1) * L::N, &p.tm_x, bar, q.d0, int(t0), q.h, q.b);
        tma_load_4d(s_g, &p.tm_g, bar, q.d0, int(t0), q.h, q.b);
      }
    } else {
      const int n = rows_of(tile, w * R, R);
      tx.own(s_x, t0, n, live, XT(0.f));
      tg.own(s_g, t0, n, live, GT(gpad));
      cp_commit();
    }
  };

  start(bars, abort_flag, S);
  fetch(rank, 0);
  // the running state, held by the thread that owns the column
  const bool owner = tid < q.width;
  const long long col = q.col0 + tid;
  float H = (owner && p.h0) ? p.h0[(long long)q.b * p.C + col] : 0.f;

  int k = 0;
  for (int tile0 = 0; tile0 < p.NT; tile0 += S, ++k) {
    const int tile = tile0 + rank;
    const int n = rows_of(tile, w * R, R);
    const XT* bx = s_x + (kBulk ? (k & 1) * L::N : 0);
    if constexpr (kBulk) {
      wait_data(&bars[B_DATA + (k & 1)], (k >> 1) & 1, abort_flag);
      if (LOGITS && n < R) Tile<GT, V, R>::pad(s_g, n, gpad);  // TMA left 0 there: a = 1 only for log decays
    } else {
      cp_wait();
    }
    typename VX::R xr[kBulk ? 1 : R];
    float a[R][V], A[V], X[V];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float xv[V], gv[V];
      const typename VX::R xw = *Tile<XT, V, R>::at(bx, r);
      if constexpr (!kBulk) xr[r] = xw;
      VX::unpack(xw, xv);
      VG::unpack(*Tile<GT, V, R>::at(s_g, r), gv);
      decays<LOGITS, V>(gv, a[r]);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        X[i] = r == 0 ? xv[i] : fmaf(a[r][i], X[i], xv[i]);
        A[i] = r == 0 ? a[r][i] : A[i] * a[r][i];
      }
    }
    if (!kBulk && tile0 + S < p.NT) fetch(tile + S, k + 1);
#pragma unroll
    for (int i = 0; i < V; ++i) s_map[w * CB + lane * V + i] = make_float2(A[i], X[i]);
    __syncthreads();
    if (kBulk && tile0 + S < p.NT) fetch(tile + S, k + 1);
    if (tid < CB) {
      float2 wm[W];  // the column's map of each warp
#pragma unroll
      for (int j = 0; j < W; ++j) wm[j] = s_map[j * CB + tid];
      const float2* agg = s_agg + (k & 1) * S * CB + tid;
      if (S > 1) {
        float2 m = wm[0];
#pragma unroll
        for (int j = 1; j < W; ++j) m = compose(wm[j], m);
        exchange<CB>(m, s_agg, bars, k, S, rank, abort_flag);
        for (int i = 0; i < rank; ++i) H = fmaf(agg[i * CB].x, H, agg[i * CB].y);
      }
      if (p.states != nullptr && owner && tile < p.NT) p.states[((long long)q.b * p.NT + tile) * p.C + col] = H;
#pragma unroll
      for (int j = 0; j < W; ++j) {
        s_in[j * CB + tid] = H;
        H = fmaf(wm[j].x, H, wm[j].y);
      }
      for (int i = rank + 1; i < S; ++i) H = fmaf(agg[i * CB].x, H, agg[i * CB].y);
    }
    __syncthreads();
    float h[V];
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = s_in[w * CB + lane * V + i];
    OT* orow = op + ((long long)tile * TC + w * R) * p.os[1];
    const int nl = live ? n : 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float xv[V];
      if constexpr (kBulk)
        VX::unpack(*Tile<XT, V, R>::at(bx, r), xv);
      else
        VX::unpack(xr[r], xv);
#pragma unroll
      for (int i = 0; i < V; ++i) h[i] = fmaf(a[r][i], h[i], xv[i]);
      if (r < nl) Vec<OT, V>::store(orow, h);
      orow += p.os[1];
    }
  }
  leave(S, p.status, abort_flag);
  if (rank == 0 && owner && p.ht) p.ht[(long long)q.b * p.C + col] = H;
}

// ---------------------------------------------------------------- backward
template <typename XT, typename GT, typename OT, int V, bool LOGITS>
__global__ void __launch_bounds__(Shape<XT, true>::T, 2) gscan_bwd_kernel(const __grid_constant__ GscanParams p) {
  using L = Smem<XT, GT, OT, V, true>;
  using VX = Vec<XT, V>;
  using VG = Vec<GT, V>;
  using VO = Vec<OT, V>;
  constexpr int R = L::R, W = L::W, CB = L::CB, TC = W * R;
  constexpr bool kBulk = L::kBulk;
  extern __shared__ __align__(128) uint8_t sm[];
  XT* s_x = reinterpret_cast<XT*>(sm + L::x);
  GT* s_g = reinterpret_cast<GT*>(sm + L::g);
  OT* s_d = reinterpret_cast<OT*>(sm + L::d);
  float2* s_map = reinterpret_cast<float2*>(sm + L::map);  // (A, M) of each warp: maps of mu, in reversed time
  float2* s_in = reinterpret_cast<float2*>(sm + L::in);    // (h before, mu behind) each warp's rows
  float* s_fx = reinterpret_cast<float*>(sm + L::fx);      // X of each warp's forward map
  float2* s_agg = reinterpret_cast<float2*>(sm + L::agg);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::bar);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + L::bar + 48);

  const Place q = place(p, CB);
  const int S = p.S, rank = q.rank;
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const bool live = lane * V < q.width, has_do = p.d_o != nullptr;
  const Tile<XT, V, R> tx{static_cast<const XT*>(p.x) + offset(p.xs, q), p.xs[1]};
  const Tile<GT, V, R> tg{static_cast<const GT*>(p.g) + offset(p.gs, q), p.gs[1]};
  const Tile<OT, V, R> td{has_do ? static_cast<const OT*>(p.d_o) + offset(p.dos, q) : nullptr, p.dos[1]};
  XT* dxp = static_cast<XT*>(p.dx) + offset(p.dxs, q) + lane * V;
  GT* dgp = static_cast<GT*>(p.dg) + offset(p.dgs, q) + lane * V;
  const float gpad = LOGITS ? INFINITY : 0.f;  // a = 1
  auto rows_of = [&](int tile, int first, int most) {
    const long long t = (long long)tile * TC + first;
    return t >= p.T ? 0 : (p.T - t < most ? int(p.T - t) : most);
  };
  auto fetch = [&](int tile, int k) {
    const long long t0 = (long long)tile * TC;
    if constexpr (kBulk) {
      if (tid == 0) {
        uint64_t* bar = &bars[B_DATA + (k & 1)];
        mbar_arrive_expect_tx(bar, uint32_t(L::N) * uint32_t(sizeof(XT) + sizeof(GT) + (has_do ? sizeof(OT) : 0)));
        tma_load_4d(s_x + (k & 1) * L::N, &p.tm_x, bar, q.d0, int(t0), q.h, q.b);
        tma_load_4d(s_g, &p.tm_g, bar, q.d0, int(t0), q.h, q.b);
        if (has_do) tma_load_4d(s_d + (k & 1) * L::N, &p.tm_d, bar, q.d0, int(t0), q.h, q.b);
      }
    } else {
      const int n = rows_of(tile, w * R, R);
      tx.own(s_x, t0, n, live, XT(0.f));
      tg.own(s_g, t0, n, live, GT(gpad));
      td.own(s_d, t0, has_do ? n : 0, live, OT(0.f));
      cp_commit();
    }
  };

  start(bars, abort_flag, S);
  const bool owner = tid < q.width;
  const long long col = q.col0 + tid;
  const float* states = p.states + (long long)q.b * p.NT * p.C + col;
  int tile = (p.NT - 1) / S * S + rank;
  fetch(tile, 0);
  float hs = owner && tile < p.NT ? states[(long long)tile * p.C] : 0.f;  // state before the tile
  float MU = (owner && p.dht) ? p.dht[(long long)q.b * p.C + col] : 0.f;

  for (int k = 0; tile >= 0; tile -= S, ++k) {
    const int n = rows_of(tile, w * R, R);
    const XT* bx = s_x + (kBulk ? (k & 1) * L::N : 0);
    const OT* bd = s_d + (kBulk ? (k & 1) * L::N : 0);
    if constexpr (kBulk) {
      wait_data(&bars[B_DATA + (k & 1)], (k >> 1) & 1, abort_flag);
      if ((LOGITS && n < R) || !has_do) {
        if (LOGITS) Tile<GT, V, R>::pad(s_g, n, gpad);  // TMA left 0 there: a = 1 only for log decays
        if (!has_do) Tile<OT, V, R>::pad(const_cast<OT*>(bd), 0, 0.f);
        fence_async_smem();  // later copies write there again
      }
    } else {
      cp_wait();
    }
    typename VX::R xr[kBulk ? 1 : R];
    typename VO::R dr[kBulk ? 1 : R];
    float pa[R][V], A[V], X[V], M[V];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float xv[V], gv[V];
      const typename VX::R xw = *Tile<XT, V, R>::at(bx, r);
      if constexpr (!kBulk) {
        xr[r] = xw;
        dr[r] = *Tile<OT, V, R>::at(bd, r);
      }
      VX::unpack(xw, xv);
      VG::unpack(*Tile<GT, V, R>::at(s_g, r), gv);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        pa[r][i] = pack_decay<LOGITS>(gv[i]);
        const float a = decay_of<LOGITS>(pa[r][i]);
        X[i] = r == 0 ? xv[i] : fmaf(a, X[i], xv[i]);
        A[i] = r == 0 ? a : A[i] * a;
      }
    }
    if (!kBulk && tile >= S) fetch(tile - S, k + 1);
#pragma unroll
    for (int r = R - 1; r >= 0; --r) {
      float dv[V];
      if constexpr (kBulk)
        VO::unpack(*Tile<OT, V, R>::at(bd, r), dv);
      else
        VO::unpack(dr[r], dv);
#pragma unroll
      for (int i = 0; i < V; ++i) M[i] = decay_of<LOGITS>(pa[r][i]) * (r == R - 1 ? dv[i] : dv[i] + M[i]);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      s_map[w * CB + lane * V + i] = make_float2(A[i], M[i]);
      s_fx[w * CB + lane * V + i] = X[i];
    }
    __syncthreads();
    if (kBulk && tile >= S) fetch(tile - S, k + 1);
    if (tid < CB) {
      float2 wm[W];  // the column's maps of mu, and X of its forward maps
      float wx[W];
#pragma unroll
      for (int j = 0; j < W; ++j) {
        wm[j] = s_map[j * CB + tid];
        wx[j] = s_fx[j * CB + tid];
      }
      const float2* agg = s_agg + (k & 1) * S * CB + tid;
      if (S > 1) {
        float2 m = wm[W - 1];
#pragma unroll
        for (int j = W - 2; j >= 0; --j) m = compose(wm[j], m);
        exchange<CB>(m, s_agg, bars, k, S, rank, abort_flag);
        for (int i = S - 1; i > rank; --i) MU = fmaf(agg[i * CB].x, MU, agg[i * CB].y);
      }
      // MU behind each warp's rows takes the place of its map's M
#pragma unroll
      for (int j = W - 1; j >= 0; --j) {
        const float mu = MU;
        MU = fmaf(wm[j].x, MU, wm[j].y);
        wm[j].y = mu;
      }
#pragma unroll
      for (int j = 0; j < W; ++j) {
        s_in[j * CB + tid] = make_float2(hs, wm[j].y);
        hs = fmaf(wm[j].x, hs, wx[j]);
      }
      for (int i = rank - 1; i >= 0; --i) MU = fmaf(agg[i * CB].x, MU, agg[i * CB].y);
      hs = owner && tile >= S ? states[(long long)(tile - S) * p.C] : 0.f;
    }
    __syncthreads();
    float h[V], mu[V], hp[R][V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float2 in = s_in[w * CB + lane * V + i];
      h[i] = in.x;
      mu[i] = in.y;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float xv[V];
      if constexpr (kBulk)
        VX::unpack(*Tile<XT, V, R>::at(bx, r), xv);
      else
        VX::unpack(xr[r], xv);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        hp[r][i] = h[i];
        h[i] = fmaf(decay_of<LOGITS>(pa[r][i]), h[i], xv[i]);
      }
    }
    const int nl = live ? n : 0;
    const long long t0 = (long long)tile * TC + w * R;
    XT* dxr = dxp + (t0 + R - 1) * p.dxs[1];
    GT* dgr = dgp + (t0 + R - 1) * p.dgs[1];
#pragma unroll
    for (int r = R - 1; r >= 0; --r) {
      float lam[V], dgv[V];
      if constexpr (kBulk)
        VO::unpack(*Tile<OT, V, R>::at(bd, r), lam);
      else
        VO::unpack(dr[r], lam);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        lam[i] += mu[i];
        mu[i] = decay_of<LOGITS>(pa[r][i]) * lam[i];
        dgv[i] = mu[i] * hp[r][i];
        if (LOGITS) dgv[i] *= slope_of(pa[r][i]);
      }
      if (r < nl) {
        VX::store(dxr, lam);
        VG::store(dgr, dgv);
      }
      dxr -= p.dxs[1];
      dgr -= p.dgs[1];
    }
  }
  leave(S, p.status, abort_flag);
  if (rank == 0 && owner && p.dh0) p.dh0[(long long)q.b * p.C + col] = MU;
}

// ---------------------------------------------------------------- few tokens
// One thread per V channels walks the rows: for single tokens and sequences
// too short to split, where the launch is what counts.
template <typename XT, typename GT, typename OT, int V>
__global__ void __launch_bounds__(128) gscan_short_kernel(const GscanParams p) {
  const long long i0 = ((long long)blockIdx.x * blockDim.x + threadIdx.x) * V;
  if (i0 >= (long long)p.B * p.C) return;
  const int b = int(i0 / p.C), ch = int(i0 - (long long)b * p.C), h = ch / p.D, d = ch - h * p.D;
  const XT* xp = static_cast<const XT*>(p.x) + p.xs[0] * b + p.xs[2] * h + d;
  const GT* gp = static_cast<const GT*>(p.g) + p.gs[0] * b + p.gs[2] * h + d;
  OT* op = static_cast<OT*>(p.o) + p.os[0] * b + p.os[2] * h + d;
  float s[V];
#pragma unroll
  for (int i = 0; i < V; ++i) s[i] = 0.f;
  if (p.h0) Vec<float, V>::unpack(Vec<float, V>::load(p.h0 + i0), s);
#pragma unroll 4
  for (int t = 0; t < p.T; ++t) {
    float xv[V], gv[V];
    Vec<XT, V>::unpack(Vec<XT, V>::load(xp + t * p.xs[1]), xv);
    Vec<GT, V>::unpack(Vec<GT, V>::load(gp + t * p.gs[1]), gv);
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = fmaf(p.logits ? decay<true>(gv[i]) : decay<false>(gv[i]), s[i], xv[i]);
    Vec<OT, V>::store(op + t * p.os[1], s);
  }
  if (p.ht) Vec<float, V>::store(p.ht + i0, s);
}

// ------------------------------------------------------------------ host side
constexpr int kShortRows = 16;

enum class Pass { kFwd, kBwd };

// Per kernel and device: whether its attributes are set, and how many clusters
// of each size the device holds at once.
struct ClusterInfo {
  bool ready;
  int active[kMaxCluster + 1];
};

inline void cluster_config(cudaLaunchConfig_t* cfg, cudaLaunchAttribute* at, int clusters, int S, int threads, size_t smem,
                           cudaStream_t s) {
  memset(cfg, 0, sizeof(*cfg));
  cfg->gridDim = dim3(unsigned(clusters) * unsigned(S));
  cfg->blockDim = dim3(unsigned(threads));
  cfg->dynamicSmemBytes = smem;
  cfg->stream = s;
  at->id = cudaLaunchAttributeClusterDimension;
  at->val.clusterDim.x = unsigned(S);
  at->val.clusterDim.y = at->val.clusterDim.z = 1;
  cfg->attrs = at;
  cfg->numAttrs = 1;
}

template <typename L, typename K>
int launch_cluster(K kern, GscanParams p, int chains, cudaStream_t s, ClusterInfo* info) {
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute at;
  static std::mutex mu;
  std::unique_lock<std::mutex> lock(mu);
  if (!info->ready) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::bytes(kMaxCluster)) != cudaSuccess)
      return cuda_failed();
    for (int S = 1; S <= kMaxCluster; ++S) {
      cluster_config(&cfg, &at, 1, S, L::Sh::T, L::bytes(S), nullptr);
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
        cudaGetLastError();
        n = 0;
      }
      info->active[S] = n;
    }
    info->ready = true;
  }
  lock.unlock();
  // Cluster size: the fewest rounds of strides.  A size that leaves SMs empty
  // or needs a second wave of clusters has more of them.
  int best = 1;
  long long best_cost = -1;
  for (int S = 1; S <= kMaxCluster && S <= p.NT; ++S) {
    if (info->active[S] < 1) continue;
    const long long waves = (chains + info->active[S] - 1) / info->active[S];
    const long long cost = waves * ((p.NT + S - 1) / S);
    if (best_cost < 0 || cost < best_cost) best = S, best_cost = cost;
  }
  p.S = best;
  cluster_config(&cfg, &at, chains, best, L::Sh::T, L::bytes(best), s);
  return cudaLaunchKernelEx(&cfg, kern, p) == cudaSuccess ? GDN_OK : cuda_failed();
}

template <typename T> constexpr CUtensorMapDataType map_type();
template <> constexpr CUtensorMapDataType map_type<float>() { return CU_TENSOR_MAP_DATA_TYPE_FLOAT32; }
template <> constexpr CUtensorMapDataType map_type<__half>() { return CU_TENSOR_MAP_DATA_TYPE_FLOAT16; }
template <> constexpr CUtensorMapDataType map_type<__nv_bfloat16>() { return CU_TENSOR_MAP_DATA_TYPE_BFLOAT16; }

template <typename T>
bool make_map(CUtensorMap* m, const GscanParams& p, const void* base, const long long* st, int columns, int rows) {
  const uint64_t dims[4] = {uint64_t(p.D), uint64_t(p.T), uint64_t(p.H), uint64_t(p.B)};
  // a dimension of one element may come with any stride: it is never taken
  auto bytes = [&](long long s, int n) { return uint64_t(n > 1 ? s : p.D) * sizeof(T); };
  const uint64_t strides[3] = {bytes(st[1], p.T), bytes(st[2], p.H), bytes(st[0], p.B)};
  const uint32_t box[4] = {uint32_t(columns), uint32_t(rows), 1, 1};
  return make_tmap(m, map_type<T>(), 4, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

template <typename XT, typename GT, typename OT, int V, bool LOGITS>
int launch(GscanParams p, Pass pass, cudaStream_t s, int dev) {
  constexpr int CB = 32 * V, TC = Shape<XT, false>::TC;
  p.NT = (p.T + TC - 1) / TC;
  if (V > 1) {
    if (!make_map<XT>(&p.tm_x, p, p.x, p.xs, CB, TC) || !make_map<GT>(&p.tm_g, p, p.g, p.gs, CB, TC)) return GDN_ERR_CUDA;
    if (pass == Pass::kBwd && p.d_o && !make_map<OT>(&p.tm_d, p, p.d_o, p.dos, CB, TC)) return GDN_ERR_CUDA;
  }
  const long long chains = (long long)p.B * p.H * ((p.D + CB - 1) / CB);
  if (chains * kMaxCluster > 0x7fffffffLL) return GDN_ERR_UNSUPPORTED;
  static ClusterInfo info[2][kMaxDevices] = {};
  if (pass == Pass::kFwd)
    return launch_cluster<Smem<XT, GT, OT, V, false>>(gscan_fwd_kernel<XT, GT, OT, V, LOGITS>, p, int(chains), s,
                                                      &info[0][dev]);
  return launch_cluster<Smem<XT, GT, OT, V, true>>(gscan_bwd_kernel<XT, GT, OT, V, LOGITS>, p, int(chains), s,
                                                   &info[1][dev]);
}

template <typename XT, typename GT, typename OT, int V>
int launch(const GscanParams& p, Pass pass, cudaStream_t s, int dev) {
  if (pass == Pass::kFwd && p.T <= kShortRows && p.states == nullptr) {
    const long long n = (long long)p.B * p.C / V;
    gscan_short_kernel<XT, GT, OT, V><<<unsigned((n + 127) / 128), 128, 0, s>>>(p);
    return cudaGetLastError() == cudaSuccess ? GDN_OK : GDN_ERR_CUDA;
  }
  return p.logits ? launch<XT, GT, OT, V, true>(p, pass, s, dev) : launch<XT, GT, OT, V, false>(p, pass, s, dev);
}

template <typename XT, typename GT, typename OT>
int launch_v(const GscanParams& p, Pass pass, int vec, cudaStream_t s, int dev) {
  return vec > 1 ? launch<XT, GT, OT, kVec>(p, pass, s, dev) : launch<XT, GT, OT, 1>(p, pass, s, dev);
}

template <typename XT>
int launch_x(const GscanParams& p, Pass pass, bool g32, bool o32, int vec, cudaStream_t s, int dev) {
  if (g32) return o32 ? launch_v<XT, float, float>(p, pass, vec, s, dev) : launch_v<XT, float, XT>(p, pass, vec, s, dev);
  return o32 ? launch_v<XT, XT, float>(p, pass, vec, s, dev) : launch_v<XT, XT, XT>(p, pass, vec, s, dev);
}

// Whether every row of a tensor starts on, and is a multiple of, `align` bytes.
bool row_ok(const void* ptr, const int64_t* st, const GscanParams& p, int es, int align) {
  if (ptr == nullptr) return true;
  if (reinterpret_cast<uintptr_t>(ptr) % size_t(align) || (long long)p.D * es % align) return false;
  const int n[3] = {p.B, p.T, p.H};
  for (int i = 0; st != nullptr && i < 3; ++i)
    if (n[i] > 1 && (st[i] <= 0 || st[i] * es % align)) return false;
  return true;
}

bool bad_stride(const int64_t* st) { return st[0] < 0 || st[1] < 0 || st[2] < 0; }

bool elem_aligned(const void* ptr, int es) { return reinterpret_cast<uintptr_t>(ptr) % size_t(es) == 0; }

int validate(const gdn_gated_scan_args* a, Pass pass) {
  if (a == nullptr || a->abi_version != GDN_B200_ABI_VERSION) return GDN_ERR_INVALID_ARGUMENT;
  if (a->B < 1 || a->T < 1 || a->H < 1 || a->D < 1) return GDN_ERR_INVALID_ARGUMENT;
  if ((long long)a->H * a->D > 0x3fffffffLL || a->T > 0x7fff0000) return GDN_ERR_UNSUPPORTED;
  if ((long long)a->B * a->H * a->D > 0x1fffffffffLL) return GDN_ERR_UNSUPPORTED;
  if (a->flags & ~GDN_FLAG_G_LOGSIGMOID) return GDN_ERR_INVALID_ARGUMENT;
  for (int dt : {a->x_dtype, a->g_dtype, a->o_dtype})
    if (dt != GDN_DTYPE_F32 && dt != GDN_DTYPE_F16 && dt != GDN_DTYPE_BF16) return GDN_ERR_INVALID_ARGUMENT;
  if (a->g_dtype != GDN_DTYPE_F32 && a->g_dtype != a->x_dtype) return GDN_ERR_UNSUPPORTED;
  if (a->o_dtype != GDN_DTYPE_F32 && a->o_dtype != a->x_dtype) return GDN_ERR_UNSUPPORTED;
  if (!a->x || !a->g || bad_stride(a->x_stride) || bad_stride(a->g_stride)) return GDN_ERR_INVALID_ARGUMENT;
  const int xe = dtype_size(a->x_dtype), ge = dtype_size(a->g_dtype), oe = dtype_size(a->o_dtype);
  if (!elem_aligned(a->x, xe) || !elem_aligned(a->g, ge) || !elem_aligned(a->h0, 4) || !elem_aligned(a->ht, 4) ||
      !elem_aligned(a->states, 4))
    return GDN_ERR_ALIGNMENT;
  if (pass == Pass::kFwd) {
    if (!a->o || bad_stride(a->o_stride)) return GDN_ERR_INVALID_ARGUMENT;
    if (!elem_aligned(a->o, oe)) return GDN_ERR_ALIGNMENT;
  } else {
    if (!a->states || !a->dx || !a->dg) return GDN_ERR_INVALID_ARGUMENT;
    if (bad_stride(a->dx_stride) || bad_stride(a->dg_stride) || (a->d_o && bad_stride(a->do_stride)))
      return GDN_ERR_INVALID_ARGUMENT;
    if (!elem_aligned(a->d_o, oe) || !elem_aligned(a->dx, xe) || !elem_aligned(a->dg, ge) ||
        !elem_aligned(a->dht, 4) || !elem_aligned(a->dh0, 4))
      return GDN_ERR_ALIGNMENT;
  }
  return GDN_OK;
}

void copy3(long long* d, const int64_t* s) {
  for (int i = 0; i < 3; ++i) d[i] = s[i];
}

int run(const gdn_gated_scan_args* a, Pass pass, void* stream) {
  const int rc = validate(a, pass);
  if (rc != GDN_OK) return rc;
  int dev = 0;
  if (!device_is_sm100(&dev)) return GDN_ERR_NO_DEVICE;
  GscanParams p;
  memset(&p, 0, sizeof(p));
  p.x = a->x, p.g = a->g, p.h0 = a->h0, p.ht = a->ht, p.o = a->o, p.states = a->states;
  p.B = a->B, p.T = a->T, p.C = a->H * a->D, p.H = a->H, p.D = a->D;
  p.logits = (a->flags & GDN_FLAG_G_LOGSIGMOID) != 0;
  p.status = a->status;
  copy3(p.xs, a->x_stride);
  copy3(p.gs, a->g_stride);
  copy3(p.os, a->o_stride);
  const int xe = dtype_size(a->x_dtype), ge = dtype_size(a->g_dtype), oe = dtype_size(a->o_dtype);
  const int64_t* in[3] = {a->x_stride, a->g_stride, pass == Pass::kBwd && a->d_o ? a->do_stride : a->x_stride};
  const int64_t* out[2] = {pass == Pass::kFwd ? a->o_stride : a->dx_stride,
                           pass == Pass::kFwd ? a->o_stride : a->dg_stride};
  // Heads that lie one behind the other are one head.
  bool flat = true;
  for (auto st : {in[0], in[1], in[2], out[0], out[1]}) flat = flat && st[2] == a->D;
  if (flat || a->H == 1) p.H = 1, p.D = p.C;
  // TMA tiles and two channels per thread where every tensor's rows allow
  // them; one channel otherwise (odd head sizes, odd strides or bases).
  bool wide = row_ok(a->x, a->x_stride, p, xe, 16) && row_ok(a->g, a->g_stride, p, ge, 16);
  if (pass == Pass::kFwd) {
    wide = wide && row_ok(a->o, a->o_stride, p, oe, kVec * oe) && row_ok(a->h0, nullptr, p, 4, 4 * kVec) &&
         row_ok(a->ht, nullptr, p, 4, 4 * kVec);
  } else {
    p.d_o = a->d_o, p.dht = a->dht, p.dx = a->dx, p.dg = a->dg, p.dh0 = a->dh0;
    copy3(p.dos, a->do_stride);
    copy3(p.dxs, a->dx_stride);
    copy3(p.dgs, a->dg_stride);
    wide = wide && row_ok(a->d_o, a->do_stride, p, oe, 16) && row_ok(a->dx, a->dx_stride, p, xe, kVec * xe) &&
         row_ok(a->dg, a->dg_stride, p, ge, kVec * ge);
  }
  const bool g32 = a->g_dtype == GDN_DTYPE_F32, o32 = a->o_dtype == GDN_DTYPE_F32;
  const int vec = wide ? kVec : 1;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->x_dtype == GDN_DTYPE_F32) return launch_v<float, float, float>(p, pass, vec, s, dev);
  if (a->x_dtype == GDN_DTYPE_F16) return launch_x<__half>(p, pass, g32, o32, vec, s, dev);
  return launch_x<__nv_bfloat16>(p, pass, g32, o32, vec, s, dev);
}

}  // namespace
}  // namespace gdn

extern "C" int gdn_gated_scan_fwd_sm100(const gdn_gated_scan_args* args, void* stream) {
  return gdn::run(args, gdn::Pass::kFwd, stream);
}

extern "C" int gdn_gated_scan_bwd_sm100(const gdn_gated_scan_args* args, void* stream) {
  return gdn::run(args, gdn::Pass::kBwd, stream);
}

extern "C" uint64_t gdn_gated_scan_states_bytes(const gdn_gated_scan_args* a) {
  if (a == nullptr || a->B < 1 || a->T < 1 || a->H < 1 || a->D < 1) return 0;
  const uint64_t rows = a->x_dtype == GDN_DTYPE_F32 ? gdn::Shape<float, false>::TC : gdn::Shape<__half, false>::TC;
  return uint64_t(a->B) * ((uint64_t(a->T) + rows - 1) / rows) * uint64_t(a->H) * uint64_t(a->D) * 4ull;
}
