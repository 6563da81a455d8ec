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
// Split.  A chain's channels are the CTA's columns (32 lanes x V channels) and
// its rows are split three ways: R consecutive rows per warp, held in
// registers; 8 warps per CTA; up to 16 CTAs per cluster.  A cluster walks the
// sequence in strides of S tiles.  Per stride every warp composes its rows,
// the CTA composes its warps in shared memory and pushes its map to every CTA
// of the cluster (distributed shared memory), and after one cluster barrier
// each CTA folds the maps before its own into the running state, replays its
// rows from registers and writes them.  The order of all sums is fixed, so
// results repeat bit for bit; no CTA ever waits on global memory.
//
// The backward walks the strides from the end.  It needs h_{t-1}; instead of
// the rounded outputs it takes the fp32 state at each tile's start, which the
// forward leaves behind (one row in 8 R), and recomputes the tile from x.
#include "../../include/gdn_b200.h"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>

#include "host_util.h"

namespace gdn {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxCluster = 16;

struct GscanParams {
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
  int B, T, C, D;  // C = H * D channels
  int NT, S;       // tiles of the sequence, CTAs per cluster
  int logits;      // g holds logits: a = sigmoid(g)
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

// Rows per warp: 8 for 16-bit x.  fp32 x takes 4, so that the backward's four
// arrays of R x V values stay in registers.
template <typename XT> __host__ __device__ constexpr int rows_per_warp() { return sizeof(XT) == 4 ? 4 : 8; }

// a_t.  expf, not the raw exponential instruction: an error in a is multiplied
// by the chain's memory length, and the final state is returned in fp32.
__device__ __forceinline__ float decay(float g, bool logits) {
  return logits ? __frcp_rn(1.f + expf(-g)) : expf(g);
}

// The backward needs a and, for logits, 1 - a, each with its own relative
// accuracy: s = min(a, 1 - a) = e / (1 + e), e = exp(-|g|), is kept with the
// side it belongs to in the sign bit.
__device__ __forceinline__ float pack_decay(float g, bool logits) {
  if (!logits) return expf(g);
  const float e = expf(-fabsf(g));
  const float s = e * __frcp_rn(1.f + e);
  return g < 0.f ? s : -s;
}
__device__ __forceinline__ float decay_of(float p, bool logits) {
  return logits && (__float_as_uint(p) >> 31) ? 1.f + p : p;
}
__device__ __forceinline__ float slope_of(float p) { return (__float_as_uint(p) >> 31) ? -p : 1.f - p; }

struct Place {
  int b, ch0, rank;
  bool live;
  long long xo, go;  // element offsets of this thread's channels at t = 0
};

template <int V>
__device__ __forceinline__ long long chan_off(const long long* st, int b, int ch, int D) {
  const int h = ch / D;
  return st[0] * b + st[2] * h + (ch - h * D);
}

// ---------------------------------------------------------------- forward
template <typename XT, typename GT, typename OT, int V>
__global__ void __launch_bounds__(kThreads, 2) gscan_fwd_kernel(const GscanParams p) {
  constexpr int R = rows_per_warp<XT>();
  constexpr int CB = 32 * V;
  constexpr int TC = kWarps * R;
  extern __shared__ float4 smem_raw[];
  float2* s_map = reinterpret_cast<float2*>(smem_raw);       // [kWarps][CB] maps of this CTA's warps
  float* s_in = reinterpret_cast<float*>(s_map + kWarps * CB);  // [kWarps][CB] state before each warp's rows
  float2* s_agg = reinterpret_cast<float2*>(s_in + kWarps * CB);  // [2][S][CB] maps of the cluster's CTAs

  cg::cluster_group cluster = cg::this_cluster();
  const int S = p.S;
  const int nblk = (p.C + CB - 1) / CB;
  const int chain = blockIdx.x / S, rank = blockIdx.x - chain * S;
  const int b = chain / nblk, cb = chain - b * nblk;
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const int ch = cb * CB + lane * V;
  const bool live = ch < p.C;
  const XT* xp = static_cast<const XT*>(p.x) + (live ? chan_off<V>(p.xs, b, ch, p.D) : 0);
  const GT* gp = static_cast<const GT*>(p.g) + (live ? chan_off<V>(p.gs, b, ch, p.D) : 0);
  OT* op = static_cast<OT*>(p.o) + (live ? chan_off<V>(p.os, b, ch, p.D) : 0);
  const bool logits = p.logits != 0;

  // the running state, held by the thread that owns the column
  const int col = cb * CB + tid;
  const bool owner = tid < CB && col < p.C;
  float H = (owner && p.h0) ? p.h0[(long long)b * p.C + col] : 0.f;

  int buf = 0;
  for (int tile0 = 0; tile0 < p.NT; tile0 += S, buf ^= 1) {
    const int tile = tile0 + rank;
    const long long t0 = (long long)tile * TC + w * R;
    const int n = !live || t0 >= p.T ? 0 : (p.T - t0 < R ? int(p.T - t0) : R);
    typename Vec<XT, V>::R xr[R];
    typename Vec<GT, V>::R gr[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (r < n) {
        xr[r] = Vec<XT, V>::load(xp + (t0 + r) * p.xs[1]);
        gr[r] = Vec<GT, V>::load(gp + (t0 + r) * p.gs[1]);
      }
    float a[R][V], A[V], X[V];
#pragma unroll
    for (int i = 0; i < V; ++i) A[i] = 1.f, X[i] = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r < n) {
        float xv[V], gv[V];
        Vec<XT, V>::unpack(xr[r], xv);
        Vec<GT, V>::unpack(gr[r], gv);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          a[r][i] = decay(gv[i], logits);
          X[i] = r == 0 ? xv[i] : fmaf(a[r][i], X[i], xv[i]);
          A[i] *= a[r][i];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) s_map[w * CB + lane * V + i] = make_float2(A[i], X[i]);
    __syncthreads();
    if (S > 1) {
      if (tid < CB) {
        float2 m = s_map[tid];
#pragma unroll
        for (int j = 1; j < kWarps; ++j) {
          const float2 n2 = s_map[j * CB + tid];
          m = make_float2(n2.x * m.x, fmaf(n2.x, m.y, n2.y));
        }
        float2* mine = s_agg + (buf * S + rank) * CB + tid;
        for (int r = 0; r < S; ++r) *cluster.map_shared_rank(mine, r) = m;
      }
      cluster.sync();
    }
    if (tid < CB) {
      const float2* agg = s_agg + buf * S * CB + tid;
      for (int i = 0; i < rank; ++i) {
        const float2 m = agg[i * CB];
        H = fmaf(m.x, H, m.y);
      }
      if (p.states != nullptr && owner && tile < p.NT) p.states[((long long)b * p.NT + tile) * p.C + col] = H;
#pragma unroll
      for (int j = 0; j < kWarps; ++j) {
        s_in[j * CB + tid] = H;
        const float2 m = s_map[j * CB + tid];
        H = fmaf(m.x, H, m.y);
      }
      for (int i = rank + 1; i < S; ++i) {
        const float2 m = agg[i * CB];
        H = fmaf(m.x, H, m.y);
      }
    }
    __syncthreads();
    float h[V];
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = s_in[w * CB + lane * V + i];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r < n) {
        float xv[V];
        Vec<XT, V>::unpack(xr[r], xv);
#pragma unroll
        for (int i = 0; i < V; ++i) h[i] = fmaf(a[r][i], h[i], xv[i]);
        Vec<OT, V>::store(op + (t0 + r) * p.os[1], h);
      }
    }
  }
  if (rank == 0 && owner && p.ht) p.ht[(long long)b * p.C + col] = H;
}

// ---------------------------------------------------------------- backward
template <typename XT, typename GT, typename OT, int V>
__global__ void __launch_bounds__(kThreads, sizeof(XT) == 4 || sizeof(OT) == 4 ? 1 : 2)
    gscan_bwd_kernel(const GscanParams p) {
  constexpr int R = rows_per_warp<XT>();
  constexpr int CB = 32 * V;
  constexpr int TC = kWarps * R;
  extern __shared__ float4 smem_raw[];
  float2* s_map = reinterpret_cast<float2*>(smem_raw);       // [kWarps][CB] (A, M): mu maps, in reversed time
  float2* s_in = s_map + kWarps * CB;                           // [kWarps][CB] (h before, mu behind) each warp's rows
  float* s_x = reinterpret_cast<float*>(s_in + kWarps * CB);    // [kWarps][CB] X of the forward maps
  float2* s_agg = reinterpret_cast<float2*>(s_x + kWarps * CB);  // [2][S][CB]

  cg::cluster_group cluster = cg::this_cluster();
  const int S = p.S;
  const int nblk = (p.C + CB - 1) / CB;
  const int chain = blockIdx.x / S, rank = blockIdx.x - chain * S;
  const int b = chain / nblk, cb = chain - b * nblk;
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const int ch = cb * CB + lane * V;
  const bool live = ch < p.C;
  const XT* xp = static_cast<const XT*>(p.x) + (live ? chan_off<V>(p.xs, b, ch, p.D) : 0);
  const GT* gp = static_cast<const GT*>(p.g) + (live ? chan_off<V>(p.gs, b, ch, p.D) : 0);
  const OT* dop = static_cast<const OT*>(p.d_o) + (live ? chan_off<V>(p.dos, b, ch, p.D) : 0);
  XT* dxp = static_cast<XT*>(p.dx) + (live ? chan_off<V>(p.dxs, b, ch, p.D) : 0);
  GT* dgp = static_cast<GT*>(p.dg) + (live ? chan_off<V>(p.dgs, b, ch, p.D) : 0);
  const bool logits = p.logits != 0, has_do = p.d_o != nullptr;

  const int col = cb * CB + tid;
  const bool owner = tid < CB && col < p.C;
  float MU = (owner && p.dht) ? p.dht[(long long)b * p.C + col] : 0.f;

  int buf = 0;
  for (int tile0 = (p.NT - 1) / S * S; tile0 >= 0; tile0 -= S, buf ^= 1) {
    const int tile = tile0 + rank;
    const long long t0 = (long long)tile * TC + w * R;
    const int n = !live || t0 >= p.T ? 0 : (p.T - t0 < R ? int(p.T - t0) : R);
    typename Vec<XT, V>::R xr[R];
    typename Vec<GT, V>::R gr[R];
    typename Vec<OT, V>::R dr[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (r < n) {
        xr[r] = Vec<XT, V>::load(xp + (t0 + r) * p.xs[1]);
        gr[r] = Vec<GT, V>::load(gp + (t0 + r) * p.gs[1]);
        if (has_do) dr[r] = Vec<OT, V>::load(dop + (t0 + r) * p.dos[1]);
      }
    float hs = 0.f;  // state before this tile, for the column's owner
    if (owner && tile < p.NT) hs = p.states[((long long)b * p.NT + tile) * p.C + col];
    float pa[R][V], A[V], X[V], M[V];
#pragma unroll
    for (int i = 0; i < V; ++i) A[i] = 1.f, X[i] = M[i] = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r < n) {
        float xv[V], gv[V];
        Vec<XT, V>::unpack(xr[r], xv);
        Vec<GT, V>::unpack(gr[r], gv);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          pa[r][i] = pack_decay(gv[i], logits);
          const float a = decay_of(pa[r][i], logits);
          X[i] = r == 0 ? xv[i] : fmaf(a, X[i], xv[i]);
          A[i] *= a;
        }
      }
    }
    if (has_do) {
#pragma unroll
      for (int r = R - 1; r >= 0; --r) {
        if (r < n) {
          float dv[V];
          Vec<OT, V>::unpack(dr[r], dv);
#pragma unroll
          for (int i = 0; i < V; ++i) M[i] = decay_of(pa[r][i], logits) * (dv[i] + M[i]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      s_map[w * CB + lane * V + i] = make_float2(A[i], M[i]);
      s_x[w * CB + lane * V + i] = X[i];
    }
    __syncthreads();
    if (S > 1) {
      if (tid < CB) {
        float2 m = s_map[(kWarps - 1) * CB + tid];
#pragma unroll
        for (int j = kWarps - 2; j >= 0; --j) {
          const float2 n2 = s_map[j * CB + tid];
          m = make_float2(n2.x * m.x, fmaf(n2.x, m.y, n2.y));
        }
        float2* mine = s_agg + (buf * S + rank) * CB + tid;
        for (int r = 0; r < S; ++r) *cluster.map_shared_rank(mine, r) = m;
      }
      cluster.sync();
    }
    if (tid < CB) {
      const float2* agg = s_agg + buf * S * CB + tid;
      for (int i = S - 1; i > rank; --i) {
        const float2 m = agg[i * CB];
        MU = fmaf(m.x, MU, m.y);
      }
#pragma unroll
      for (int j = 0; j < kWarps; ++j) {
        s_in[j * CB + tid].x = hs;
        hs = fmaf(s_map[j * CB + tid].x, hs, s_x[j * CB + tid]);
      }
#pragma unroll
      for (int j = kWarps - 1; j >= 0; --j) {
        s_in[j * CB + tid].y = MU;
        const float2 m = s_map[j * CB + tid];
        MU = fmaf(m.x, MU, m.y);
      }
      for (int i = rank - 1; i >= 0; --i) {
        const float2 m = agg[i * CB];
        MU = fmaf(m.x, MU, m.y);
      }
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
      if (r < n) {
        float xv[V];
        Vec<XT, V>::unpack(xr[r], xv);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          hp[r][i] = h[i];
          h[i] = fmaf(decay_of(pa[r][i], logits), h[i], xv[i]);
        }
      }
    }
#pragma unroll
    for (int r = R - 1; r >= 0; --r) {
      if (r < n) {
        float lam[V], dgv[V];
        if (has_do) {
          Vec<OT, V>::unpack(dr[r], lam);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) lam[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          lam[i] += mu[i];
          mu[i] = decay_of(pa[r][i], logits) * lam[i];
          dgv[i] = mu[i] * hp[r][i];
          if (logits) dgv[i] *= slope_of(pa[r][i]);
        }
        Vec<XT, V>::store(dxp + (t0 + r) * p.dxs[1], lam);
        Vec<GT, V>::store(dgp + (t0 + r) * p.dgs[1], dgv);
      }
    }
  }
  if (rank == 0 && owner && p.dh0) p.dh0[(long long)b * p.C + col] = MU;
}

// ---------------------------------------------------------------- few tokens
// One thread per V channels walks the rows: for single tokens and sequences
// too short to split, where the launch is what counts.
template <typename XT, typename GT, typename OT, int V>
__global__ void __launch_bounds__(128) gscan_short_kernel(const GscanParams p) {
  const long long i0 = ((long long)blockIdx.x * blockDim.x + threadIdx.x) * V;
  if (i0 >= (long long)p.B * p.C) return;
  const int b = int(i0 / p.C), ch = int(i0 - (long long)b * p.C);
  const XT* xp = static_cast<const XT*>(p.x) + chan_off<V>(p.xs, b, ch, p.D);
  const GT* gp = static_cast<const GT*>(p.g) + chan_off<V>(p.gs, b, ch, p.D);
  OT* op = static_cast<OT*>(p.o) + chan_off<V>(p.os, b, ch, p.D);
  float h[V];
#pragma unroll
  for (int i = 0; i < V; ++i) h[i] = 0.f;
  if (p.h0) Vec<float, V>::unpack(Vec<float, V>::load(p.h0 + i0), h);
#pragma unroll 4
  for (int t = 0; t < p.T; ++t) {
    float xv[V], gv[V];
    Vec<XT, V>::unpack(Vec<XT, V>::load(xp + t * p.xs[1]), xv);
    Vec<GT, V>::unpack(Vec<GT, V>::load(gp + t * p.gs[1]), gv);
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = fmaf(decay(gv[i], p.logits != 0), h[i], xv[i]);
    Vec<OT, V>::store(op + t * p.os[1], h);
  }
  if (p.ht) Vec<float, V>::store(p.ht + i0, h);
}

// ------------------------------------------------------------------ host side
constexpr int kShortRows = 16;

enum class Pass { kFwd, kBwd };

template <typename K>
int launch_cluster(K kern, const GscanParams& p, int chains, size_t smem, cudaStream_t s, bool* configured) {
  if (!*configured) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024) != cudaSuccess)
      return cuda_failed();
    *configured = true;
  }
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(unsigned(chains) * unsigned(p.S));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = unsigned(p.S);
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p) == cudaSuccess ? GDN_OK : cuda_failed();
}

template <typename XT, typename GT, typename OT, int V>
int launch(GscanParams p, Pass pass, cudaStream_t s, int dev) {
  constexpr int CB = 32 * V, TC = kWarps * rows_per_warp<XT>();
  if (pass == Pass::kFwd && p.T <= kShortRows && p.states == nullptr) {
    const long long n = (long long)p.B * p.C / V;
    gscan_short_kernel<XT, GT, OT, V><<<unsigned((n + 127) / 128), 128, 0, s>>>(p);
    return cudaGetLastError() == cudaSuccess ? GDN_OK : GDN_ERR_CUDA;
  }
  p.NT = (p.T + TC - 1) / TC;
  const long long chains = (long long)p.B * ((p.C + CB - 1) / CB);
  if (chains * kMaxCluster > 0x7fffffffLL) return GDN_ERR_UNSUPPORTED;
  int S = 1;
  while (S < kMaxCluster && S < p.NT) S *= 2;
  p.S = S;
  static bool configured[2][kMaxDevices] = {};
  if (pass == Pass::kFwd)
    return launch_cluster(gscan_fwd_kernel<XT, GT, OT, V>, p, int(chains),
                          size_t(CB) * (kWarps * 12 + (S > 1 ? 2 * S * 8 : 0)), s, &configured[0][dev]);
  return launch_cluster(gscan_bwd_kernel<XT, GT, OT, V>, p, int(chains),
                        size_t(CB) * (kWarps * 20 + (S > 1 ? 2 * S * 8 : 0)), s, &configured[1][dev]);
}

template <typename XT, typename GT, typename OT>
int launch_v(const GscanParams& p, Pass pass, int vec, cudaStream_t s, int dev) {
  return vec == 4 ? launch<XT, GT, OT, 4>(p, pass, s, dev) : launch<XT, GT, OT, 1>(p, pass, s, dev);
}

template <typename XT>
int launch_x(const GscanParams& p, Pass pass, bool g32, bool o32, int vec, cudaStream_t s, int dev) {
  if (g32) return o32 ? launch_v<XT, float, float>(p, pass, vec, s, dev) : launch_v<XT, float, XT>(p, pass, vec, s, dev);
  return o32 ? launch_v<XT, XT, float>(p, pass, vec, s, dev) : launch_v<XT, XT, XT>(p, pass, vec, s, dev);
}

// Whether `n`-element vectors of the tensor are aligned at every (b, t, h).
bool vec_ok(const void* ptr, const int64_t* st, int es, int n) {
  if (ptr == nullptr) return true;
  if (reinterpret_cast<uintptr_t>(ptr) % (size_t(es) * n)) return false;
  return st[0] % n == 0 && st[1] % n == 0 && st[2] % n == 0;
}

bool bad_stride(const int64_t* st) { return st[0] < 0 || st[1] < 0 || st[2] < 0; }

bool elem_aligned(const void* ptr, int es) { return reinterpret_cast<uintptr_t>(ptr) % size_t(es) == 0; }

int validate(const gdn_gated_scan_args* a, Pass pass) {
  if (a == nullptr || a->abi_version != GDN_B200_ABI_VERSION) return GDN_ERR_INVALID_ARGUMENT;
  if (a->B < 1 || a->T < 1 || a->H < 1 || a->D < 1) return GDN_ERR_INVALID_ARGUMENT;
  if ((long long)a->H * a->D > 0x3fffffffLL || (long long)a->T > 0x7fffff00LL) return GDN_ERR_UNSUPPORTED;
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
  p.B = a->B, p.T = a->T, p.C = a->H * a->D, p.D = a->D;
  p.logits = (a->flags & GDN_FLAG_G_LOGSIGMOID) != 0;
  copy3(p.xs, a->x_stride);
  copy3(p.gs, a->g_stride);
  copy3(p.os, a->o_stride);
  const int xe = dtype_size(a->x_dtype), ge = dtype_size(a->g_dtype), oe = dtype_size(a->o_dtype);
  // Four channels per thread where every row of every tensor allows its
  // vectors; one channel otherwise (odd head sizes, odd strides or bases).
  bool v4 = a->D % 4 == 0 && vec_ok(a->x, a->x_stride, xe, 4) && vec_ok(a->g, a->g_stride, ge, 4);
  if (pass == Pass::kFwd) {
    v4 = v4 && vec_ok(a->o, a->o_stride, oe, 4);
    if (reinterpret_cast<uintptr_t>(a->h0) % 16 || reinterpret_cast<uintptr_t>(a->ht) % 16) v4 = false;
  } else {
    p.d_o = a->d_o, p.dht = a->dht, p.dx = a->dx, p.dg = a->dg, p.dh0 = a->dh0;
    copy3(p.dos, a->do_stride);
    copy3(p.dxs, a->dx_stride);
    copy3(p.dgs, a->dg_stride);
    v4 = v4 && vec_ok(a->d_o, a->do_stride, oe, 4) && vec_ok(a->dx, a->dx_stride, xe, 4) &&
         vec_ok(a->dg, a->dg_stride, ge, 4);
  }
  const bool g32 = a->g_dtype == GDN_DTYPE_F32, o32 = a->o_dtype == GDN_DTYPE_F32;
  const int vec = v4 ? 4 : 1;
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
  const uint64_t rows = gdn::kWarps * (a->x_dtype == GDN_DTYPE_F32 ? gdn::rows_per_warp<float>()
                                                                    : gdn::rows_per_warp<__half>());
  return uint64_t(a->B) * ((uint64_t(a->T) + rows - 1) / rows) * uint64_t(a->H) * uint64_t(a->D) * 4ull;
}
