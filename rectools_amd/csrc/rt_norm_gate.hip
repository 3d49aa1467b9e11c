// The norm behind a block, its gate, its residual scale and the norm in front of the next block in one pass over the rows:
//
//   n = N_post(f);   y = alpha x + s * sigmoid(z) * drop(n);   h = N_pre(y)
//
// N is LayerNorm (mean and variance, weight and bias) or the root-mean-square norm (weight; bias optional).  N_post, z, s and N_pre are each
// optional.  The dropout is the counter-based mask of the row kernels (rt_common.h: rt_drop_bits), never stored.
//
// Memory bound: forward reads f, z, x and writes y, h; backward reads the two gradients, y, f, z and writes the three input gradients — a
// row stays in the registers of its threads (16 to 1,024 of them, at most 8 columns each), statistics are two-pass over those
// registers.  The column sums behind the parameters' gradients stay in registers over all rows of a workgroup, are written once per
// workgroup and joined by a second launch in a fixed order: no atomics, the same bits every run.  16,384 rows of 2,048, every part: forward
// 136 us = 4.9 TB/s, backward 197 us = 5.4 TB/s, joining 11 us; 25,600 rows of 256: 25 us = 5.2 TB/s, 38 us, 5 us; 40,001 rows of 50: 12.2, 22.1 and 4.5 us (3.3
// and 2.9 TB/s): accesses of 8 bytes, a pair of columns each, and 14 of a row's 64 column slots idle.  Two such rows are 400 bytes, 25 loads of 16; a flat stream of a
// workgroup's rows through LDS has not been tried.  Dropout hashes once per element, where one hash holds the bits of four: p = 0.2 against 0, 25,600 rows of 256
// 28.6 | 25.8 us forward, 37.1 | 34.4 backward; 16,384 of 2,048 150 | 143 and 185 | 172.
#include "rt_common.h"

namespace {

struct NgArgs {
  const float* x; const float* f; const float* z; const float* s; const float* pw; const float* pb; const float* nw; const float* nb;
  float* y; float* h; float* stat;      // stat [M, 4]: mean and 1 / deviation of f, of y (training)
  long long M; int d;
  int post, pre;
  float alpha, eps, p; unsigned long long seed, stream;
  // backward
  const float* gy; const float* gh; const float* yin;
  float* dx; float* df; float* dz; float* part;      // part [workgroups][5][d]: s, pw, pb, nw, nb
};

template <int TPR> __device__ __forceinline__ float row_sum(float v, float* sm) {
  if (TPR <= 64) {
#pragma unroll
    for (int o = TPR / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
  }
  v = wave_sum(v);      // TPR > 64: the workgroup is one row
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int w = 0; w < (TPR + 63) / 64; ++w) v += sm[w];
  return v;
}

template <int VW> __device__ __forceinline__ void ld(const float* p, float* v) {
  if (VW == 4) { const f32x4 t = *reinterpret_cast<const f32x4*>(p); v[0] = t[0]; v[1 % VW] = t[1]; v[2 % VW] = t[2]; v[3 % VW] = t[3]; }
  else if (VW == 2) { const float2 t = *reinterpret_cast<const float2*>(p); v[0] = t.x; v[1 % VW] = t.y; }
  else v[0] = p[0];
}
template <int VW> __device__ __forceinline__ void st(float* p, const float* v) {
  if (VW == 4) *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1 % VW], v[2 % VW], v[3 % VW]};
  else if (VW == 2) *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1 % VW]);
  else p[0] = v[0];
}
// the factor of element i under the dropout mask: 0 or 1 / (1 - p)
__device__ __forceinline__ float drop_factor(const NgArgs& a, long long i, unsigned thr, float inv_keep) {
  const uint2 r = rt_drop_bits(a.seed, a.stream, (unsigned long long)(i >> 2));
  const unsigned w = (i & 2) ? r.y : r.x;
  return (((i & 1) ? (w >> 16) : (w & 0xFFFFu)) >= thr) ? inv_keep : 0.f;
}
__device__ __forceinline__ float sigmoid(float z) { return 1.f / (1.f + expf(-z)); }
// and one minus it, without the cancellation behind large z
__device__ __forceinline__ float sigmoid(float z, float& rest) {
  const float e = expf(-fabsf(z)), near = 1.f / (1.f + e), far = e * near;
  rest = z > 0.f ? far : near;
  return z > 0.f ? near : far;
}

// mean (LayerNorm) and 1 / deviation of a row held in registers; v becomes the normalised row
template <int TPR, int NE, bool LAYER>
__device__ __forceinline__ void normalise(float (&v)[NE], const bool (&on)[NE], float inv_d, float eps, float& mean, float& rstd, float* sm) {
  mean = 0.f;
  if (LAYER) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < NE; ++e) s += on[e] ? v[e] : 0.f;
    mean = row_sum<TPR>(s, sm) * inv_d;
  }
  float q = 0.f;
#pragma unroll
  for (int e = 0; e < NE; ++e) { v[e] -= mean; q += on[e] ? v[e] * v[e] : 0.f; }
  rstd = 1.f / sqrtf(row_sum<TPR>(q, sm) * inv_d + eps);
#pragma unroll
  for (int e = 0; e < NE; ++e) v[e] *= rstd;
}

template <int TPR, int VW, int NV, bool LAYER>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_gate_fwd_kernel(NgArgs a) {
  constexpr int NT = TPR > 256 ? TPR : 256, NE = VW * NV, RPW = NT / TPR;
  __shared__ float sm[16];
  const int t = threadIdx.x % TPR;
  const float inv_d = 1.f / (float)a.d;
  const unsigned thr = rt_drop_thr16(a.p);
  const float inv_keep = a.p > 0.f ? 1.f / (1.f - a.p) : 1.f;
  int col[NV];
  bool on[NE];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    col[k] = (k * TPR + t) * VW;
#pragma unroll
    for (int e = 0; e < VW; ++e) on[k * VW + e] = col[k] < a.d;      // (VW divides d)
  }
  const long long step = (long long)gridDim.x * RPW;
  for (long long row = (long long)blockIdx.x * RPW + threadIdx.x / TPR; row < a.M; row += step) {
    const long long base = row * a.d;
    float v[NE], x[NE], z[NE];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int e = 0; e < VW; ++e) { v[k * VW + e] = 0.f; x[k * VW + e] = 0.f; z[k * VW + e] = 0.f; }
      if (on[k * VW]) {
        ld<VW>(a.f + base + col[k], v + k * VW);
        ld<VW>(a.x + base + col[k], x + k * VW);
        if (a.z != nullptr) ld<VW>(a.z + base + col[k], z + k * VW);
      }
    }
    float m1 = 0.f, r1 = 1.f, m2 = 0.f, r2 = 1.f;
    if (a.post) normalise<TPR, NE, LAYER>(v, on, inv_d, a.eps, m1, r1, sm);
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (on[k * VW]) {
        float w[VW], b[VW], s[VW];
        if (a.post) ld<VW>(a.pw + col[k], w);
        if (a.pb != nullptr) ld<VW>(a.pb + col[k], b);
        if (a.s != nullptr) ld<VW>(a.s + col[k], s);
#pragma unroll
        for (int e = 0; e < VW; ++e) {
          float n = v[k * VW + e];
          if (a.post) n = a.pb != nullptr ? n * w[e] + b[e] : n * w[e];
          if (a.p > 0.f) n *= drop_factor(a, base + col[k] + e, thr, inv_keep);
          if (a.z != nullptr) n *= sigmoid(z[k * VW + e]);
          if (a.s != nullptr) n *= s[e];
          v[k * VW + e] = a.alpha * x[k * VW + e] + n;
        }
        st<VW>(a.y + base + col[k], v + k * VW);
      }
    if (a.pre) {
      normalise<TPR, NE, LAYER>(v, on, inv_d, a.eps, m2, r2, sm);
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (on[k * VW]) {
          float w[VW], b[VW];
          ld<VW>(a.nw + col[k], w);
          if (a.nb != nullptr) ld<VW>(a.nb + col[k], b);
#pragma unroll
          for (int e = 0; e < VW; ++e) v[k * VW + e] = a.nb != nullptr ? v[k * VW + e] * w[e] + b[e] : v[k * VW + e] * w[e];
          st<VW>(a.h + base + col[k], v + k * VW);
        }
    }
    if (a.stat != nullptr && t == 0) *reinterpret_cast<f32x4*>(a.stat + row * 4) = f32x4{m1, r1, m2, r2};
  }
}

template <int TPR, int VW, int NV, bool LAYER>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_gate_bwd_kernel(NgArgs a) {
  constexpr int NT = TPR > 256 ? TPR : 256, NE = VW * NV, RPW = NT / TPR;
  __shared__ float sm[16];
  __shared__ float colsum[RPW > 1 ? TPR * NE : 1];
  const int t = threadIdx.x % TPR, in_wg = threadIdx.x / TPR;
  const float inv_d = 1.f / (float)a.d;
  const unsigned thr = rt_drop_thr16(a.p);
  const float inv_keep = a.p > 0.f ? 1.f / (1.f - a.p) : 1.f;
  int col[NV];
  bool on[NE];
  float acc[5][NE], pw[NE], pb[NE], s[NE], nw[NE];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    col[k] = (k * TPR + t) * VW;
#pragma unroll
    for (int e = 0; e < VW; ++e) {
      on[k * VW + e] = col[k] < a.d;
      pw[k * VW + e] = 1.f; pb[k * VW + e] = 0.f; s[k * VW + e] = 1.f; nw[k * VW + e] = 0.f;
    }
    if (on[k * VW]) {
      if (a.post) ld<VW>(a.pw + col[k], pw + k * VW);
      if (a.pb != nullptr) ld<VW>(a.pb + col[k], pb + k * VW);
      if (a.s != nullptr) ld<VW>(a.s + col[k], s + k * VW);
      if (a.pre) ld<VW>(a.nw + col[k], nw + k * VW);
    }
  }
#pragma unroll
  for (int q = 0; q < 5; ++q)
#pragma unroll
    for (int e = 0; e < NE; ++e) acc[q][e] = 0.f;

  const long long step = (long long)gridDim.x * RPW;
  for (long long row = (long long)blockIdx.x * RPW + in_wg; row < a.M; row += step) {
    const long long base = row * a.d;
    float g[NE], gh[NE], t2[NE], u[NE], z[NE];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int e = 0; e < VW; ++e) { g[k * VW + e] = 0.f; gh[k * VW + e] = 0.f; t2[k * VW + e] = 0.f; u[k * VW + e] = 0.f; z[k * VW + e] = 0.f; }
      if (on[k * VW]) {
        if (a.gy != nullptr) ld<VW>(a.gy + base + col[k], g + k * VW);
        if (a.gh != nullptr) { ld<VW>(a.gh + base + col[k], gh + k * VW); ld<VW>(a.yin + base + col[k], t2 + k * VW); }
        ld<VW>(a.f + base + col[k], u + k * VW);
        if (a.z != nullptr) ld<VW>(a.z + base + col[k], z + k * VW);
      }
    }
    const f32x4 sv = *reinterpret_cast<const f32x4*>(a.stat + row * 4);
    if (a.gh != nullptr) {
      float c1 = 0.f, c2 = 0.f;
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        t2[e] = on[e] ? (t2[e] - sv[2]) * sv[3] : 0.f;
        acc[3][e] += gh[e] * t2[e];
        acc[4][e] += gh[e];
        gh[e] *= nw[e];
        c1 += gh[e];
        c2 += gh[e] * t2[e];
      }
      c2 = row_sum<TPR>(c2, sm) * inv_d;
      c1 = LAYER ? row_sum<TPR>(c1, sm) * inv_d : 0.f;
#pragma unroll
      for (int e = 0; e < NE; ++e) g[e] += sv[3] * (gh[e] - c1 - t2[e] * c2);
    }
    float c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float o[VW], oz[VW];
#pragma unroll
      for (int e = 0; e < VW; ++e) {
        const int i = k * VW + e;
        o[e] = a.alpha * g[i];
        const float uu = a.post ? (u[i] - sv[0]) * sv[1] : u[i];
        float n = a.post ? uu * pw[i] + pb[i] : uu;
        float rest = 0.f;
        const float gate = a.z != nullptr ? sigmoid(z[i], rest) : 1.f;
        const float keep = a.p > 0.f ? drop_factor(a, base + col[k] + e, thr, inv_keep) : 1.f;
        n *= keep;
        const float gs = g[i] * s[i];
        oz[e] = gs * n * gate * rest;
        const float gn = gs * gate * keep;
        if (on[i]) {
          acc[0][i] += g[i] * gate * n;
          acc[1][i] += gn * uu;
          acc[2][i] += gn;
        }
        u[i] = on[i] ? uu : 0.f;
        g[i] = on[i] ? gn * pw[i] : 0.f;
        c1 += g[i];
        c2 += g[i] * u[i];
      }
      if (on[k * VW]) {
        st<VW>(a.dx + base + col[k], o);
        if (a.dz != nullptr) st<VW>(a.dz + base + col[k], oz);
      }
    }
    if (a.post) {
      c2 = row_sum<TPR>(c2, sm) * inv_d;
      c1 = LAYER ? row_sum<TPR>(c1, sm) * inv_d : 0.f;
#pragma unroll
      for (int e = 0; e < NE; ++e) g[e] = sv[1] * (g[e] - c1 - u[e] * c2);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (on[k * VW]) st<VW>(a.df + base + col[k], g + k * VW);
  }
  if (a.part == nullptr) return;
  float* out = a.part + (long long)blockIdx.x * 5 * a.d;
#pragma unroll
  for (int q = 0; q < 5; ++q) {
    if (RPW > 1) {      // the row groups of the workgroup, one after the other
      for (int r = 0; r < RPW; ++r) {
        if (in_wg == r) {
#pragma unroll
          for (int e = 0; e < NE; ++e) colsum[e * TPR + t] = (r == 0 ? 0.f : colsum[e * TPR + t]) + acc[q][e];
        }
        __syncthreads();
      }
      if (in_wg == 0) {
#pragma unroll
        for (int e = 0; e < NE; ++e) acc[q][e] = colsum[e * TPR + t];
      }
      __syncthreads();
    }
    if (in_wg == 0) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (on[k * VW]) st<VW>(out + (long long)q * a.d + col[k], acc[q] + k * VW);
    }
  }
}

// [n][5][d] partial sums -> the five column vectors (the ones that are asked for): 16 columns x 64 shares of the workgroups
struct ColOut { float* o[5]; };
__global__ __launch_bounds__(1024) void norm_gate_sums_kernel(const float* part, int n, int d, ColOut out) {
  __shared__ float sm[64][17];
  const int c = threadIdx.x & 15, sl = threadIdx.x >> 4;
  const long long W = 5LL * d, at = (long long)blockIdx.x * 16 + c;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (at < W)
    for (int r = sl; r < n; r += 256) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (r + 64 * k < n) s[k] += part[(r + 64 * k) * W + at];
    }
  sm[sl][c] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  for (int half = 32; half > 0; half >>= 1) {
    if (sl < half) sm[sl][c] += sm[sl + half][c];
    __syncthreads();
  }
  if (sl == 0 && at < W) {
    float* o = out.o[at / d];
    if (o != nullptr) o[at % d] = sm[0][c];
  }
}

// Threads per row and columns per thread by width: at most 8 columns, so that the backward pass (five column sums, four parameters and five
// row values per column) stays below 170 registers — with 16 columns it takes 256 and one wave per SIMD (2,048 columns: 255 us, with 8 197).  Up
// to 256 columns four (256 columns: 37 us backward and 26 forward, with eight 46 and 30).  Narrow rows share a wave.
struct Shape { int tpr, ne; };
Shape shape_of(int d) {
  if (d <= 64) return {16, 4};
  if (d <= 128) return {32, 4};
  if (d <= 256) return {64, 4};
  if (d <= 512) return {64, 8};
  if (d <= 2048) return {256, 8};
  if (d <= 4096) return {512, 8};
  return {1024, 8};
}
int rows_per_wg(const Shape& s) { return s.tpr < 256 ? 256 / s.tpr : 1; }
int vec_of(int d, const void* const* ps, int n) {
  uintptr_t all = 0;
  for (int i = 0; i < n; ++i) all |= (uintptr_t)ps[i];
  if (d % 4 == 0 && (all & 15u) == 0) return 4;
  if (d % 2 == 0 && (all & 7u) == 0) return 2;
  return 1;
}
// Workgroups of the backward pass: every one of them leaves 5 d partial sums for the second launch.  512 against 1,024, both launches: 2,048 columns 207
// us against 242, 256 columns 45.0 against 44.5, 50 columns 27.2 against 27.6.
long long bwd_wgs(long long M, int d) {
  const int rpw = rows_per_wg(shape_of(d));
  const long long need = (M + rpw - 1) / rpw;
  return need < 1 ? 1 : (need < 512 ? need : 512);
}

template <int TPR, int VW, int NV>
void launch_shape(const NgArgs& a, bool layer, bool backward, unsigned grid, hipStream_t stream) {
  constexpr int NTHR = TPR > 256 ? TPR : 256;
  if (backward) {
    if (layer) norm_gate_bwd_kernel<TPR, VW, NV, true><<<grid, NTHR, 0, stream>>>(a);
    else norm_gate_bwd_kernel<TPR, VW, NV, false><<<grid, NTHR, 0, stream>>>(a);
  } else {
    if (layer) norm_gate_fwd_kernel<TPR, VW, NV, true><<<grid, NTHR, 0, stream>>>(a);
    else norm_gate_fwd_kernel<TPR, VW, NV, false><<<grid, NTHR, 0, stream>>>(a);
  }
}
template <int TPR, int NE>
void launch_width(const NgArgs& a, int vw, bool layer, bool backward, unsigned grid, hipStream_t stream) {
  if (vw == 4) launch_shape<TPR, 4, NE / 4>(a, layer, backward, grid, stream);
  else if (vw == 2) launch_shape<TPR, 2, NE / 2>(a, layer, backward, grid, stream);
  else launch_shape<TPR, 1, NE>(a, layer, backward, grid, stream);
}
int launch(const NgArgs& a, int vw, bool layer, bool backward, unsigned grid, hipStream_t stream) {
  switch (shape_of(a.d).tpr * 16 + shape_of(a.d).ne) {
    case 16 * 16 + 4: launch_width<16, 4>(a, vw, layer, backward, grid, stream); break;
    case 32 * 16 + 4: launch_width<32, 4>(a, vw, layer, backward, grid, stream); break;
    case 64 * 16 + 4: launch_width<64, 4>(a, vw, layer, backward, grid, stream); break;
    case 64 * 16 + 8: launch_width<64, 8>(a, vw, layer, backward, grid, stream); break;
    case 256 * 16 + 8: launch_width<256, 8>(a, vw, layer, backward, grid, stream); break;
    case 512 * 16 + 8: launch_width<512, 8>(a, vw, layer, backward, grid, stream); break;
    default: launch_width<1024, 8>(a, vw, layer, backward, grid, stream); break;
  }
  RT_CHECK_LAUNCH();
  return RT_OK;
}

int check(int64_t M, int32_t d, const float* pw, const float* pb, const float* nw, const float* nb, float p) {
  if (M < 0 || d <= 0 || (pb != nullptr && pw == nullptr) || (nb != nullptr && nw == nullptr) || !(p >= 0.f && p < 1.f)) return RT_ERR_INVALID_ARG;
  if (d > 8192) return RT_ERR_UNSUPPORTED;
  return RT_OK;
}

}  // namespace

extern "C" {

int rt_norm_gate_fwd(const float* x, const float* f, const float* z, const float* scale, const float* post_w, const float* post_b, const float* pre_w,
                     const float* pre_b, int32_t layer, float alpha, float eps, float p, uint64_t seed, uint64_t stream_id, int64_t M, int32_t d, float* y,
                     float* h, float* stat, hipStream_t stream) {
  const int rc = check(M, d, post_w, post_b, pre_w, pre_b, p);
  if (rc != RT_OK) return rc;
  if (M == 0) return RT_OK;
  if (!(eps > 0.f) || x == nullptr || f == nullptr || y == nullptr || (pre_w != nullptr) != (h != nullptr) || ((uintptr_t)stat & 15u) != 0) return RT_ERR_INVALID_ARG;
  NgArgs a{};
  a.x = x; a.f = f; a.z = z; a.s = scale; a.pw = post_w; a.pb = post_b; a.nw = pre_w; a.nb = pre_b; a.y = y; a.h = h; a.stat = stat;
  a.M = M; a.d = d; a.post = post_w != nullptr; a.pre = pre_w != nullptr; a.alpha = alpha; a.eps = eps; a.p = p; a.seed = seed; a.stream = stream_id;
  const void* ps[] = {x, f, z, scale, post_w, post_b, pre_w, pre_b, y, h};
  const int vw = vec_of(d, ps, 10);
  const int rpw = rows_per_wg(shape_of(d));
  const long long need = (M + rpw - 1) / rpw;
  return launch(a, vw, layer != 0, false, (unsigned)(need < (1LL << 20) ? need : 1LL << 20), stream);      // (a launch holds less than 2^32 threads; workgroups loop)
}

size_t rt_norm_gate_bwd_workspace_bytes(int64_t M, int32_t d) {
  if (M <= 0 || d <= 0 || d > 8192) return 0;
  return (size_t)bwd_wgs(M, d) * 5 * d * sizeof(float);
}

int rt_norm_gate_bwd(const float* gy, const float* gh, const float* y, const float* f, const float* z, const float* scale, const float* post_w,
                     const float* post_b, const float* pre_w, int32_t layer, float alpha, float p, uint64_t seed, uint64_t stream_id, int64_t M, int32_t d,
                     const float* stat, float* dx, float* df, float* dz, float* dscale, float* dpost_w, float* dpost_b, float* dpre_w, float* dpre_b,
                     void* ws, size_t ws_bytes, hipStream_t stream) {
  const int rc = check(M, d, post_w, post_b, pre_w, nullptr, p);
  if (rc != RT_OK) return rc;
  const bool sums = dscale != nullptr || dpost_w != nullptr || dpost_b != nullptr || dpre_w != nullptr || dpre_b != nullptr;
  if (M > 0 && (f == nullptr || stat == nullptr || dx == nullptr || df == nullptr || (z != nullptr) != (dz != nullptr) || ((uintptr_t)stat & 15u) != 0 ||
                (gh != nullptr && (pre_w == nullptr || y == nullptr))))
    return RT_ERR_INVALID_ARG;
  if (sums && M > 0 && (ws == nullptr || ws_bytes < rt_norm_gate_bwd_workspace_bytes(M, d) || ((uintptr_t)ws & 15u) != 0)) return RT_ERR_WORKSPACE;
  const long long n = M > 0 ? bwd_wgs(M, d) : 0;
  if (M > 0) {
    NgArgs a{};
    a.f = f; a.z = z; a.s = scale; a.pw = post_w; a.pb = post_b; a.nw = pre_w; a.stat = const_cast<float*>(stat); a.M = M; a.d = d;
    a.post = post_w != nullptr; a.pre = pre_w != nullptr; a.alpha = alpha; a.p = p; a.seed = seed; a.stream = stream_id;
    a.gy = gy; a.gh = gh; a.yin = y; a.dx = dx; a.df = df; a.dz = dz; a.part = sums ? (float*)ws : nullptr;
    const void* ps[] = {gy, gh, y, f, z, scale, post_w, post_b, pre_w, dx, df, dz, ws};
    const int vw = vec_of(d, ps, 13);
    const int rc2 = launch(a, vw, layer != 0, true, (unsigned)n, stream);
    if (rc2 != RT_OK) return rc2;
  }
  if (sums) {
    const ColOut out{{dscale, dpost_w, dpost_b, dpre_w, dpre_b}};
    norm_gate_sums_kernel<<<(5 * d + 15) / 16, 1024, 0, stream>>>((const float*)ws, (int)n, d, out);
    RT_CHECK_LAUNCH();
  }
  return RT_OK;
}

}  // extern "C"
