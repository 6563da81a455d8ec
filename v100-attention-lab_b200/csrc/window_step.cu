// One token of windowed attention against a ring cache.
//
// The token at position p is written into its slot of the cache and attends to
// itself, the window behind it and the sinks:
//
//     slot(j) = j                                    for j < cap
//               sinks + (j - sinks) mod (cap - sinks)  otherwise
//     o = sum_j softmax_j(scale q . k_j) v_j  over  p - window < j <= p  and  j < min(sinks, p + 1)
//
// Memory bounds it: every visible key and value is read once per key head, for
// all query heads that share it (their rows share the tensor-core tiles).
//
// Split.  A cluster of CTAs owns one (sequence, key head, group of up to 16
// query rows); its warps take equal runs of 16-key tiles.  A warp loads K and V
// straight into MMA fragments in 16-byte pieces: the products' inner index may
// run in any order, so a lane's 16 contiguous bytes of a key are the fragments
// of two steps, and for V the columns are dealt out so that a lane's 16 bytes
// are its share of eight column tiles.  No staging in shared memory: the next
// tile's keys are fetched into the registers of the current one's while its
// softmax runs, its values under the next scores.
// Running maxima, sums and outputs are joined warp by warp in shared memory and
// CTA by CTA through distributed shared memory, in a fixed order.
//
// Probabilities enter the second product as the sum of two 16-bit terms: a
// single rounding would cost as much as the output's own.  They are scaled by a
// power of two that the sum shares, so that it cancels.  fp16 has a grid of
// 2^-24: with the largest at 2^14 the two terms are exact to 2^-39 of it (with
// the largest at 1 the second term of all below 2^-13 would be 0, and keys
// 17 nats below a dominant sink 44 % off).  bf16 terms keep their accuracy at
// any scale; there the scale is 1 over the number of keys, so that sums of
// values near the end of fp32's range stay in it, as their average does (values
// below some 2^-100 lose bits instead).
// Infinite values come out as such: a sum that is not finite is looked over.
//
// Measured: 64 sequences, 32 query and 8 key heads of 128, 4100 keys (1.08 GB):
// 206 us on the GPU alone, 5.2 TB/s (208 to 213 a call); without the overlapped
// fetch 290; with spilled registers (16 warps on an SM instead of 8) 350.
#include "../../include/gdn_b200.h"
#include "host_util.h"
#include "tc.cuh"

#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstring>

namespace gdn {
namespace ws {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxCluster = 8;

struct Params {
  const void* q;
  const void* k;
  const void* v;
  void* kc;
  void* vc;
  void* o;
  const int* positions;
  long long qs[2], ks[2], vs[2], os[2];  // (b, h)
  long long kcs[3], vcs[3];              // (b, slot, h)
  int G, HK, cap, window, sinks;
  float scale_log2;
  float shift;  // log2 of the largest probability's scale
};

// One 16 x 8 x 16 step.  With 8 query rows the lower half of A and of the result
// is zero and takes no registers.
template <typename T, int HR>
__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (HR == 2) {
    if constexpr (Cvt<T>::kIsBf16)
      asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                   : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                   : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
      asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                   : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                   : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    float d2, d3;
    if constexpr (Cvt<T>::kIsBf16)
      asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%5}, {%7,%8}, {%0,%1,%9,%9};"
                   : "+f"(c[0]), "+f"(c[1]), "=f"(d2), "=f"(d3)
                   : "r"(a0), "r"(0), "r"(a2), "r"(b0), "r"(b1), "f"(0.f));
    else
      asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%5}, {%7,%8}, {%0,%1,%9,%9};"
                   : "+f"(c[0]), "+f"(c[1]), "=f"(d2), "=f"(d3)
                   : "r"(a0), "r"(0), "r"(a2), "r"(b0), "r"(b1), "f"(0.f));
  }
}

// The visible keys of the token at position p, in order: [0, n_sink) and, from
// slot0 on around the ring, the window's up to p itself.
struct Keys {
  int n, n_sink, slot0;
  __device__ __forceinline__ Keys(const Params& P, int p) {
    n_sink = P.sinks <= p ? P.sinks : p + 1;
    const int w0 = p - P.window + 1 > n_sink ? p - P.window + 1 : n_sink;
    n = n_sink + (p - w0) + 1;
    slot0 = w0 < P.cap ? w0 : P.sinks + (w0 - P.sinks) % (P.cap - P.sinks);
  }
  __device__ __forceinline__ int slot(const Params& P, int i) const {
    if (i < n_sink) return i;
    const int s = slot0 + (i - n_sink);
    return s < P.cap ? s : s - (P.cap - P.sinks);
  }
};

// A warp's sums [rows][D] where they are not finite.  An infinite value times a
// second term that is 0 or of the other sign is NaN; what its probability, which is
// above 0, makes of it is the value itself, so the sum of the values that are not
// finite takes the place of such a sum.  (Works everything out anew: what it
// took as arguments would cost the kernel's loop registers.)
template <typename T, int D>
__device__ __noinline__ void restore_infinities(const Params& P, float* sums, int rows) {
  const int b = blockIdx.z, hk = blockIdx.y / ((P.G + rows - 1) / rows), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // rows whose sum of probabilities is not finite come out as NaN in any case
  const float* l = sums + kWarps * rows * (D + 1) + warp * rows;
  const int real = P.G - (blockIdx.y - hk * ((P.G + rows - 1) / rows)) * rows;
  bool any = false;
  __syncwarp();
  for (int r = 0; r < rows && r < real; ++r) any |= isfinite(l[r]);
  if (!any) return;
  sums += warp * rows * D;
  const Keys keys(P, P.positions[b]);
  const T* vc = static_cast<const T*>(P.vc) + P.vcs[0] * b + P.vcs[2] * hk;
  const T* vn = static_cast<const T*>(P.v) + P.vs[0] * b + P.vs[1] * hk;
  const int ntile = (keys.n + 15) / 16, per = (ntile + int(gridDim.x) - 1) / int(gridDim.x);
  const int first = int(blockIdx.x) * per, end = first + per < ntile ? first + per : ntile;
  constexpr int N = D / 32;  // columns of a lane, 2 or 4
  float total[N];
#pragma unroll
  for (int c = 0; c < N; ++c) total[c] = 0.f;
  for (int tile = first + warp; tile < end; tile += kWarps) {
    uint32_t v[16][N / 2];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int i = tile * 16 + j < keys.n ? tile * 16 + j : keys.n - 1;  // the last key twice: no other sum
      const T* src = (i == keys.n - 1 ? vn : vc + P.vcs[1] * (long long)keys.slot(P, i)) + lane * N;
#pragma unroll
      for (int c = 0; c < N / 2; ++c) v[j][c] = reinterpret_cast<const uint32_t*>(src)[c];
    }
#pragma unroll
    for (int j = 0; j < 16; ++j)
#pragma unroll
      for (int c = 0; c < N / 2; ++c) {
        const float2 x = Cvt<T>::unpack(v[j][c]);
        if (!isfinite(x.x)) total[2 * c] += x.x;
        if (!isfinite(x.y)) total[2 * c + 1] += x.y;
      }
  }
  for (int r = 0; r < rows; ++r)
#pragma unroll
    for (int c = 0; c < N; ++c) {
      float* s = sums + r * D + lane * N + c;
      if (total[c] != 0.f && !isfinite(*s)) *s = total[c];
    }
}

// ROWS query rows (8 or 16) per group; with 8 the lower half of each tile is zero.
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kThreads, 2) window_step_kernel(const __grid_constant__ Params P) {
  constexpr int KC = D / 32;   // 16-byte pieces of a key per lane
  constexpr int VH = D / 64;   // column halves of V
  constexpr int HR = ROWS / 8;
  extern __shared__ float smem[];
  float* s_o = smem;                               // [kWarps][ROWS][D]
  float* s_m = s_o + kWarps * ROWS * D;            // [kWarps][ROWS]
  float* s_l = s_m + kWarps * ROWS;                // [kWarps][ROWS]
  cg::cluster_group cluster = cg::this_cluster();
  const int C = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int ngroup = (P.G + ROWS - 1) / ROWS;
  const int hk = blockIdx.y / ngroup, grp = blockIdx.y - hk * ngroup, b = blockIdx.z;
  const int rows = P.G - grp * ROWS < ROWS ? P.G - grp * ROWS : ROWS;
  const int h0 = hk * P.G + grp * ROWS;
  const int p = P.positions[b];
  T* op = static_cast<T*>(P.o) + P.os[0] * b + P.os[1] * h0;

  if (p < 0) {  // the row is off: nothing is seen, nothing written to the cache
    if (rank == 0)
      for (int i = tid; i < rows * (D / 2); i += kThreads)
        reinterpret_cast<uint32_t*>(op + P.os[1] * (i / (D / 2)))[i % (D / 2)] = 0u;
    return;
  }
  const Keys keys(P, p);
  const int n = keys.n, n_sink = keys.n_sink;

  const T* kc = static_cast<const T*>(P.kc) + P.kcs[0] * b + P.kcs[2] * hk;
  const T* vc = static_cast<const T*>(P.vc) + P.vcs[0] * b + P.vcs[2] * hk;
  const T* kn = static_cast<const T*>(P.k) + P.ks[0] * b + P.ks[1] * hk;
  const T* vn = static_cast<const T*>(P.v) + P.vs[0] * b + P.vs[1] * hk;
  auto slot_of = [&](int i) { return keys.slot(P, i); };

  // query fragments, in the keys' order of the inner index
  uint4 qf[HR][KC];
  const T* qp = static_cast<const T*>(P.q) + P.qs[0] * b + P.qs[1] * h0;
#pragma unroll
  for (int r = 0; r < HR; ++r)
#pragma unroll
    for (int c = 0; c < KC; ++c)
      qf[r][c] = g + 8 * r < rows ? *reinterpret_cast<const uint4*>(qp + P.qs[1] * (g + 8 * r) + c * 32 + t * 8)
                                  : make_uint4(0, 0, 0, 0);

  constexpr int NC = 2 * HR;  // accumulators of a lane per 8 columns
  float acc[VH][8][NC];
#pragma unroll
  for (int i = 0; i < VH * 8 * NC; ++i) (&acc[0][0][0])[i] = 0.f;
  float m[HR], l[HR];
#pragma unroll
  for (int r = 0; r < HR; ++r) m[r] = -INFINITY, l[r] = 0.f;

  const int ntile = (n + 15) / 16;
  // A CTA's tiles are a run, dealt out to its warps one by one: what is read at
  // a time lies close together.
  const int per = (ntile + C - 1) / C;
  const int first = rank * per + warp;
  const int end = rank * per + per < ntile ? rank * per + per : ntile;
  // A lane's pieces of a tile: keys g and 8 + g of K, keys 2t, 2t+1, 2t+8, 2t+9 of V.
  uint4 kf[2][KC], vf[4][VH];
  // Most tiles are 16 slots in a row, old keys all: one address and constant steps.
  auto run_of = [&](int tile) {
    const int i0 = tile * 16;
    return i0 >= n_sink && i0 + 16 < n && slot_of(i0) + 16 <= P.cap;
  };
  auto load_k = [&](int tile) {
    const int i0 = tile * 16;
    if (run_of(tile)) {
      const T* src = kc + P.kcs[1] * (long long)(slot_of(i0) + g) + t * 8;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int c = 0; c < KC; ++c) kf[j][c] = __ldcs(reinterpret_cast<const uint4*>(src + j * 8 * P.kcs[1] + c * 32));
      return;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = i0 + j * 8 + g;
      const T* src = i == n - 1 ? kn : kc + P.kcs[1] * (long long)slot_of(i < n ? i : 0);
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        kf[j][c] = make_uint4(0, 0, 0, 0);
        if (i < n) kf[j][c] = *reinterpret_cast<const uint4*>(src + c * 32 + t * 8);
      }
      // the new key goes into the cache: the lanes that read it write it
      if (i == n - 1 && grp == 0)
#pragma unroll
        for (int c = 0; c < KC; ++c)
          *reinterpret_cast<uint4*>(const_cast<T*>(kc) + P.kcs[1] * (long long)slot_of(i) + c * 32 + t * 8) = kf[j][c];
    }
  };
  auto load_v = [&](int tile) {
    const int i0 = tile * 16;
    if (run_of(tile)) {
      const T* src = vc + P.vcs[1] * (long long)(slot_of(i0) + 2 * t) + g * 8;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < VH; ++c)
          vf[j][c] = __ldcs(reinterpret_cast<const uint4*>(src + ((j & 1) + (j >> 1) * 8) * P.vcs[1] + c * 64));
      return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // zero where there is no key
      const int i = i0 + 2 * t + (j & 1) + (j >> 1) * 8;
      const T* src = i == n - 1 ? vn : vc + P.vcs[1] * (long long)slot_of(i < n ? i : 0);
#pragma unroll
      for (int c = 0; c < VH; ++c) {
        vf[j][c] = make_uint4(0, 0, 0, 0);
        if (i < n) vf[j][c] = *reinterpret_cast<const uint4*>(src + c * 64 + g * 8);
      }
      if (i == n - 1 && grp == 0)
#pragma unroll
        for (int c = 0; c < VH; ++c)
          *reinterpret_cast<uint4*>(const_cast<T*>(vc) + P.vcs[1] * (long long)slot_of(i) + c * 64 + g * 8) = vf[j][c];
    }
  };
  if (first < end) {
    load_k(first);
    load_v(first);
  }
#pragma unroll 1
  for (int tile = first; tile < end; tile += kWarps) {
    const int i0 = tile * 16;
    float s[2][NC];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int e = 0; e < NC; ++e) s[j][e] = 0.f;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const uint4 a = qf[0][c], a8 = HR == 2 ? qf[HR - 1][c] : make_uint4(0, 0, 0, 0);
        mma16816<T, HR>(s[j], a.x, a8.x, a.y, a8.y, kf[j][c].x, kf[j][c].y);
        mma16816<T, HR>(s[j], a.z, a8.z, a.w, a8.w, kf[j][c].z, kf[j][c].w);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (i0 + j * 8 + 2 * t + e >= n)
#pragma unroll
          for (int r = 0; r < HR; ++r) s[j][2 * r + e] = -INFINITY;
    }
    // the next tile's keys are fetched under this one's softmax, its values
    // under the next one's scores: into the registers just used
    if (tile + kWarps < end) load_k(tile + kWarps);
    uint32_t ph[2][HR], pl[2][HR];  // probabilities of keys (2t, 2t+1) of each half tile, high and low terms
#pragma unroll
    for (int r = 0; r < HR; ++r) {
      float mt = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1])) * P.scale_log2;
      mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
      mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
      const float mn = fmaxf(m[r], mt);
      const float ref = mn == -INFINITY ? 0.f : mn;
      const float corr = fast_exp2(m[r] - ref);
      m[r] = mn;
      l[r] *= corr;
#pragma unroll
      for (int i = 0; i < VH * 8; ++i) {
        (&acc[0][0][0])[NC * i + 2 * r] *= corr;
        (&acc[0][0][0])[NC * i + 2 * r + 1] *= corr;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float e0 = fast_exp2(fmaf(s[j][2 * r], P.scale_log2, P.shift - ref));
        const float e1 = fast_exp2(fmaf(s[j][2 * r + 1], P.scale_log2, P.shift - ref));
        l[r] += e0 + e1;
        ph[j][r] = Cvt<T>::pack(e0, e1);
        const float2 hi = Cvt<T>::unpack(ph[j][r]);
        pl[j][r] = Cvt<T>::pack(e0 - hi.x, e1 - hi.y);
      }
    }
#pragma unroll
    for (int c = 0; c < VH; ++c)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t v0 = (&vf[0][c].x)[w], v1 = (&vf[1][c].x)[w], v2 = (&vf[2][c].x)[w], v3 = (&vf[3][c].x)[w];
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
          const uint32_t b0 = __byte_perm(v0, v1, odd ? 0x7632 : 0x5410);
          const uint32_t b1 = __byte_perm(v2, v3, odd ? 0x7632 : 0x5410);
          float* a = acc[c][2 * w + odd];
          mma16816<T, HR>(a, ph[0][0], HR == 2 ? ph[0][HR - 1] : 0u, ph[1][0], HR == 2 ? ph[1][HR - 1] : 0u, b0, b1);
          mma16816<T, HR>(a, pl[0][0], HR == 2 ? pl[0][HR - 1] : 0u, pl[1][0], HR == 2 ? pl[1][HR - 1] : 0u, b0, b1);
        }
      }
    if (tile + kWarps < end) load_v(tile + kWarps);
  }

  // ---------------------------------------------- join the warps, then the CTAs
  float odd = 0.f;  // NaN if a sum is not finite
#pragma unroll
  for (int i = 0; i < VH * 8 * NC; ++i) odd = fmaf((&acc[0][0][0])[i], 0.f, odd);
#pragma unroll
  for (int r = 0; r < HR; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    const int row = g + 8 * r;
    if (t == 0) {
      s_m[warp * ROWS + row] = m[r];
      s_l[warp * ROWS + row] = l[r];
    }
#pragma unroll
    for (int c = 0; c < VH; ++c)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // column n of tile i is d = 64 c + 8 n + i
        float* dst = s_o + (warp * ROWS + row) * D + c * 64 + (2 * t + e) * 8;
#pragma unroll
        for (int i = 0; i < 8; i += 4)
          *reinterpret_cast<float4*>(dst + i) =
              make_float4(acc[c][i][2 * r + e], acc[c][i + 1][2 * r + e], acc[c][i + 2][2 * r + e], acc[c][i + 3][2 * r + e]);
      }
  }
  if (__any_sync(0xffffffffu, odd != odd))
    restore_infinities<T, D>(P, s_o, ROWS);
  cluster.sync();
  // every CTA finishes a share of the rows' columns, four at a time
  constexpr int kPiece = D / 4;
  for (int i = rank * kThreads + tid; i < rows * kPiece; i += C * kThreads) {
    const int row = i / kPiece, d = (i - row * kPiece) * 4;
    float mx = -INFINITY;
    for (int c = 0; c < C; ++c) {
      const float* rm = cluster.map_shared_rank(s_m, c);
      for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, rm[w * ROWS + row]);
    }
    const float ref = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f, o0 = 0.f, o1 = 0.f, o2 = 0.f, o3 = 0.f;
    for (int c = 0; c < C; ++c) {
      const float* rm = cluster.map_shared_rank(s_m, c);
      const float* rl = cluster.map_shared_rank(s_l, c);
      const float* ro = cluster.map_shared_rank(s_o, c);
      for (int w = 0; w < kWarps; ++w) {
        const float f = fast_exp2(rm[w * ROWS + row] - ref);
        const float4 x = *reinterpret_cast<const float4*>(ro + (w * ROWS + row) * D + d);
        sum = fmaf(f, rl[w * ROWS + row], sum);
        o0 = fmaf(f, x.x, o0);
        o1 = fmaf(f, x.y, o1);
        o2 = fmaf(f, x.z, o2);
        o3 = fmaf(f, x.w, o3);
      }
    }
    const float inv = 1.f / sum;
    *reinterpret_cast<uint2*>(op + P.os[1] * row + d) =
        make_uint2(Cvt<T>::pack(o0 * inv, o1 * inv), Cvt<T>::pack(o2 * inv, o3 * inv));
  }
  cluster.sync();  // no CTA leaves while another reads its shared memory
}

// ------------------------------------------------------------------ host side
int validate(const gdn_window_step_args* a) {
  if (a == nullptr || a->abi_version != GDN_B200_ABI_VERSION) return GDN_ERR_INVALID_ARGUMENT;
  if (a->B < 1 || a->H < 1 || a->HK < 1 || a->D < 1 || a->H % a->HK != 0) return GDN_ERR_INVALID_ARGUMENT;
  if (a->window < 1 || a->sinks < 0 || (long long)a->window + a->sinks > a->capacity) return GDN_ERR_INVALID_ARGUMENT;
  if (!(a->scale > 0.f) || a->scale > 1.0e30f) return GDN_ERR_INVALID_ARGUMENT;
  if (a->dtype != GDN_DTYPE_F16 && a->dtype != GDN_DTYPE_BF16)
    return a->dtype == GDN_DTYPE_F32 ? GDN_ERR_UNSUPPORTED : GDN_ERR_INVALID_ARGUMENT;
  if (!a->q || !a->k || !a->v || !a->k_cache || !a->v_cache || !a->o || !a->positions) return GDN_ERR_INVALID_ARGUMENT;
  if (a->D != 64 && a->D != 128) return GDN_ERR_UNSUPPORTED;
  if (a->B > 65535 || a->H > 65535 || a->capacity > (1 << 30)) return GDN_ERR_UNSUPPORTED;
  const void* ptr[6] = {a->q, a->k, a->v, a->o, a->k_cache, a->v_cache};
  for (const void* p : ptr)
    if (reinterpret_cast<uintptr_t>(p) % 16) return GDN_ERR_ALIGNMENT;
  if (reinterpret_cast<uintptr_t>(a->positions) % 4) return GDN_ERR_ALIGNMENT;
  // a dimension of one element may come with any stride: it is never taken
  auto bad = [](int64_t s, int n) { return n > 1 && (s < 0 || s % 8 != 0); };
  const int64_t* two[4] = {a->q_stride, a->k_stride, a->v_stride, a->o_stride};
  for (int i = 0; i < 4; ++i)
    if (bad(two[i][0], a->B) || bad(two[i][1], i == 1 || i == 2 ? a->HK : a->H)) return GDN_ERR_ALIGNMENT;
  for (auto s : {a->kc_stride, a->vc_stride})
    if (bad(s[0], a->B) || bad(s[1], a->capacity) || bad(s[2], a->HK)) return GDN_ERR_ALIGNMENT;
  return GDN_OK;
}

template <typename T, int D, int ROWS>
int launch(const Params& p, int C, dim3 grid, cudaStream_t s, int dev) {
  constexpr size_t smem = size_t(kWarps) * ROWS * (D + 2) * 4;
  static bool configured[kMaxDevices] = {};
  auto kern = window_step_kernel<T, D, ROWS>;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) != cudaSuccess)
      return cuda_failed();
    configured[dev] = true;
  }
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = unsigned(C);
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p) == cudaSuccess ? GDN_OK : cuda_failed();
}

template <typename T, int D>
int launch_rows(const Params& p, int B, int sms, cudaStream_t s, int dev) {
  const int rows = p.G <= 8 ? 8 : 16;
  const int groups = p.HK * ((p.G + rows - 1) / rows);
  // CTAs along the keys: as many as still run at once, two on an SM, each warp
  // with a tile.  A second wave for the sake of a fuller last one does not pay,
  // joining costs more: 64 sequences, 8 key heads, 4100 keys take 206 us with
  // one CTA each, 215 with two, 233 with four; 16 with 2052 keys 49, 32 (two), 38.
  const long long own = (long long)B * groups;
  const int tiles = (p.window + p.sinks + 15) / 16;
  int C = kMaxCluster;
  while (C > 1 && (own * C > 2LL * sms || (C - 1) * kWarps >= tiles)) --C;
  const dim3 grid(C, groups, B);
  return rows == 8 ? launch<T, D, 8>(p, C, grid, s, dev) : launch<T, D, 16>(p, C, grid, s, dev);
}

int run(const gdn_window_step_args* a, void* stream) {
  const int rc = validate(a);
  if (rc != GDN_OK) return rc;
  int dev = 0;
  if (!device_is_sm100(&dev)) return GDN_ERR_NO_DEVICE;
  Params p;
  memset(&p, 0, sizeof(p));
  p.q = a->q, p.k = a->k, p.v = a->v, p.kc = a->k_cache, p.vc = a->v_cache, p.o = a->o, p.positions = a->positions;
  for (int j = 0; j < 2; ++j)
    p.qs[j] = a->q_stride[j], p.ks[j] = a->k_stride[j], p.vs[j] = a->v_stride[j], p.os[j] = a->o_stride[j];
  for (int j = 0; j < 3; ++j) p.kcs[j] = a->kc_stride[j], p.vcs[j] = a->vc_stride[j];
  p.G = a->H / a->HK, p.HK = a->HK;
  p.cap = a->capacity, p.window = a->window, p.sinks = a->sinks;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.shift = a->dtype == GDN_DTYPE_F16 ? 14.f : -float(std::ceil(std::log2(double(a->window) + a->sinks)));
  int sms = 0;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms < 1) return cuda_failed();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf = a->dtype == GDN_DTYPE_BF16;
  if (a->D == 128)
    return bf ? launch_rows<__nv_bfloat16, 128>(p, a->B, sms, s, dev) : launch_rows<__half, 128>(p, a->B, sms, s, dev);
  return bf ? launch_rows<__nv_bfloat16, 64>(p, a->B, sms, s, dev) : launch_rows<__half, 64>(p, a->B, sms, s, dev);
}

}  // namespace
}  // namespace ws
}  // namespace gdn

extern "C" int gdn_window_step_sm100(const gdn_window_step_args* args, void* stream) {
  return gdn::ws::run(args, stream);
}
