// Differential attention: the difference of two softmax maps with a learned weight, normalised per head.
//
//   A_m = softmax(scale q_m k_m^T + mask),  m = 1, 2;   o = (A_1 - lam_h A_2) v;   y = out_scale * w * o / sqrt(mean(o^2) + eps)
//
// q rows carry [H][2][hd] columns (the two maps' queries of a head next to each other), k rows [Hkv][2][hd], v rows [Hkv][2 hd]; query head
// h reads key head h / (H / Hkv).  Sessions are packed rows (cu) or equal windows; inside a session the last query is aligned with the last
// key (causal: key j is seen by query i iff j <= i + nk - nq), so one launch serves whole sessions and the newest rows of stored ones.
// Keys whose item id is 0 are masked; their K and V rows are replaced by zeros when they are staged, whatever they hold.  A query that
// sees no key has o = 0, y = 0 and no gradients.
//
// Arithmetic: fp32 in, fp32 out.  The products run on the bf16 matrix instructions, six terms of an exact three-way split per product
// (rt_attn_planes.h: split2): h m l are the top, middle and low 8 bits of the significand, the dropped terms are below 2^-24 of the product.
// Softmax statistics, sums and accumulators are fp32.  Scores live in the base-2 domain.
//
// Geometry: a workgroup is 4 waves = 2 row groups of 32 owner rows x the 2 maps; v_mfma_f32_32x32x16_bf16 tiles, the OWNER row (a query;
// in the dK/dV pass a key) is the lane, the partner rows are the registers, so probabilities and dS feed the next product from the
// registers they were made in.  Partner rows stream through LDS 32 at a time as plane images, both maps' waves read the same V.
// One wave per map rather than one wave for both: its operands and accumulators are half as many registers, which leaves two waves on a
// SIMD (one's softmax runs under the other's products).
#include "rt_attn_planes.h"

namespace {
using namespace rt_planes;

constexpr int NT = 256;
constexpr int OWN = 64;    // owner rows per workgroup
constexpr int CH = 32;     // partner rows per staged chunk

struct Args {
  const float* q; const float* k; const float* v; long long ldq, ldk, ldv;
  const float* lam;                      // [H]
  const long long* cu_q; const long long* cu_k; const long long* key_ids;
  int B, H, Hkv, hd, Lq, Lk;
  long long Nq, Nk;
  float scale; int causal;
  const float* norm_w; float out_scale, eps;
  float* y; long long ldy;
  float* o12;                            // [Nq, H, 2, 2 hd] normalised outputs of the two maps (training)
  float* lse;                            // [Nq, H, 2] log2-sum-exp2 of the two maps (training)
  float* part; float* ml;                // split keys: [n_split, Nq, H, 2, 2 hd] and [n_split, Nq, H, 2, 2] (maximum, sum)
  int n_split;
  int n_tiles;                           // owner tiles per session in the grid (longer sessions loop)
  // backward
  const float* dout; long long lddo;     // gradient of o, [Nq, H * 2 hd] (the pass in front makes it)
  const float* delta;                    // [Nq, H, 2]
  float* dq; float* dk; float* dv; long long lddq, lddk, lddv;
};

__device__ __forceinline__ void rows_of(const long long* cu, int b, int len, long long N, long long& row0, int& n) {
  // a malformed offset table cannot lead a kernel out of its buffers: both ends are clamped to the rows that exist
  if (cu != nullptr) {
    const long long s = cu[b], e = cu[b + 1];
    row0 = s < 0 ? 0 : (s > N ? N : s);
    const long long end = e > N ? N : e;
    n = end > row0 ? (int)(end - row0) : 0;
  } else {
    row0 = (long long)b * len;
    n = len;
  }
}
__device__ __forceinline__ long long rows_used(const long long* cu, int B, long long N) {      // rows behind the last session start here
  if (cu == nullptr) return N;
  const long long e = cu[B];
  return e < 0 ? 0 : (e > N ? N : e);
}

// LDS images: row r = [h | m | l] planes of C bf16 columns + 16 bytes, so that rows lie an odd number of 16-byte units apart: the 32-row
// b128 fragment reads and the 4-row transpose reads both spread over the banks, with constant offsets and no address arithmetic.
template <int C> struct Img {
  static constexpr int PLANE = C * 2, ROW = 3 * PLANE + 16, BYTES = CH * ROW;
};

// ncol columns of up to CH rows -> image; rows whose bit in `live` is 0 and columns behind ncol are zeros
template <int C, int MODE>
__device__ __forceinline__ void stage(const float* __restrict__ src, long long ld, int ncol, unsigned live, float scale, unsigned char* img, int tid) {
  constexpr int C4 = C / 4, U = CH * C4 / NT;
  f32x4 x[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int idx = tid + u * NT, r = idx / C4, c = (idx % C4) * 4;
    x[u] = f32x4{0.f, 0.f, 0.f, 0.f};
    if ((live >> r) & 1u) {
      const float* p = src + (long long)r * ld + c;
      if (MODE < 2) {
        if (MODE == 0 || c < ncol) x[u] = *reinterpret_cast<const f32x4*>(p);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + j < ncol) x[u][j] = p[j];
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int idx = tid + u * NT, r = idx / C4, c = (idx % C4) * 4;
    const f32x4 t = x[u] * scale;
    unsigned h0, m0, l0, h1, m1, l1;
    split2(t[0], t[1], h0, m0, l0);
    split2(t[2], t[3], h1, m1, l1);
    unsigned char* p = img + r * Img<C>::ROW + c * 2;
    *reinterpret_cast<u32x2*>(p) = u32x2{h0, h1};
    *reinterpret_cast<u32x2*>(p + Img<C>::PLANE) = u32x2{m0, m1};
    *reinterpret_cast<u32x2*>(p + 2 * Img<C>::PLANE) = u32x2{l0, l1};
  }
}

// 8 values of one global row at columns c .. c + 7 (zeros behind ncol), times scale, as planes
template <int MODE>
__device__ __forceinline__ P3 load_planes(const float* __restrict__ row, int c, int ncol, bool ok, float scale) {
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = 0.f;
  if (ok) {
    if (MODE < 2) {
#pragma unroll
      for (int j = 0; j < 8; j += 4)
        if (MODE == 0 || c + j < ncol) {
          const f32x4 t = *reinterpret_cast<const f32x4*>(row + c + j);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[j + e] = t[e] * scale;
        }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < ncol) x[j] = row[c + j] * scale;
    }
  }
  return split8(x);
}

__device__ __forceinline__ f32x16 mfma6(const P3& A, const P3& B, f32x16 acc) {
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A.l, B.h, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A.h, B.l, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A.m, B.m, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A.m, B.h, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A.h, B.m, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A.h, B.h, acc, 0, 0, 0);
  return acc;
}

// acc[r] += sum_c img[row(r)][c0 + c] * own[c], row(r) = 8 (r / 4) + 4 g + r % 4: the partner rows are the registers, the owner the lane
template <int C, int NS>
__device__ __forceinline__ void rows_dot(const unsigned char* img, int c0, const P3 (&own)[NS], int i, int g, f32x16& acc) {
  const unsigned char* p = img + i * Img<C>::ROW + c0 * 2 + 16 * g;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    P3 A;
    A.h = *reinterpret_cast<const bf16x8*>(p + 32 * s);
    A.m = *reinterpret_cast<const bf16x8*>(p + 32 * s + Img<C>::PLANE);
    A.l = *reinterpret_cast<const bf16x8*>(p + 32 * s + 2 * Img<C>::PLANE);
    acc = mfma6(A, own[s], acc);
  }
}

// acc[cb][r] += sum over the 32 partner rows of img[row][c0 + 32 cb + col(r)] * w[row], the lane's weights in the accumulator order of rows_dot
// (slot j of step t = register 8 t + j = row 16 t + 8 (j / 4) + 4 g + j % 4): the partner rows are the reduction index, read transposed
template <int C, int NB>
__device__ __forceinline__ void cols_dot(const unsigned char* img, int c0, const P3 (&w)[2], int lane, f32x16 (&acc)[NB]) {
  const int g = lane >> 5;
  const unsigned char* p = img + (4 * g + ((lane & 15) >> 2)) * Img<C>::ROW + (c0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int cb = 0; cb < NB; ++cb) {
      const unsigned char* a = p + 16 * t * Img<C>::ROW + 64 * cb;
      const unsigned char* b = a + 8 * Img<C>::ROW;
      P3 A;
      A.h = __builtin_bit_cast(bf16x8, (s16x8)__builtin_shufflevector(tr_read(a), tr_read(b), 0, 1, 2, 3, 4, 5, 6, 7));
      A.m = __builtin_bit_cast(bf16x8, (s16x8)__builtin_shufflevector(tr_read(a + Img<C>::PLANE), tr_read(b + Img<C>::PLANE), 0, 1, 2, 3, 4, 5, 6, 7));
      A.l = __builtin_bit_cast(bf16x8, (s16x8)__builtin_shufflevector(tr_read(a + 2 * Img<C>::PLANE), tr_read(b + 2 * Img<C>::PLANE), 0, 1, 2, 3, 4, 5, 6, 7));
      acc[cb] = mfma6(A, w[t], acc[cb]);
    }
}

__device__ __forceinline__ void split16(const float (&x)[16], P3 (&out)[2]) {
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const float y[8] = {x[8 * t], x[8 * t + 1], x[8 * t + 2], x[8 * t + 3], x[8 * t + 4], x[8 * t + 5], x[8 * t + 6], x[8 * t + 7]};
    out[t] = split8(y);
  }
}
__device__ __forceinline__ int reg_row(int r, int g) { return 8 * (r >> 2) + 4 * g + (r & 3); }
__device__ __forceinline__ f32x16 zero16() { f32x16 z; for (int r = 0; r < 16; ++r) z[r] = 0.f; return z; }

// bit j: key t0 + j exists and is not masked
__device__ __forceinline__ unsigned live_keys(const Args& a, long long row0, int t0, int n, int lane) {
  const int left = n - t0;
  unsigned bits = left >= 32 ? 0xFFFFFFFFu : (left <= 0 ? 0u : (1u << left) - 1u);
  if (a.key_ids != nullptr) {
    const int j = lane & 31;
    const bool on = j < left && a.key_ids[row0 + t0 + j] != 0;
    bits = (unsigned)__ballot(on);
  }
  return bits;
}

template <int MODE>
__device__ __forceinline__ void put4(float* row, int c, int ncol, f32x4 x) {
  if (MODE < 2) {
    if (MODE == 0 || c < ncol) *reinterpret_cast<f32x4*>(row + c) = x;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < ncol) row[c + j] = x[j];
  }
}

// blockIdx -> (owner tile, session, head, split); the LAST tile of a session first where it is the heaviest (causal queries)
struct Work { int tile, b, h, split; };
__device__ __forceinline__ Work work_of(int n_tiles, int B1, int H, bool last_first) {
  const int per = B1 * H, o = (int)blockIdx.x / per, bh = (int)blockIdx.x % per;
  Work w;
  w.tile = last_first ? n_tiles - 1 - o : o;
  w.b = bh / H;
  w.h = bh % H;
  w.split = blockIdx.y;
  return w;
}

// ---- forward ----------------------------------------------------------------------------------------------------------------------------
template <int HD, int MODE>
__global__ __launch_bounds__(NT, 2) void diff_fwd_kernel(Args a) {
  constexpr int DV = 2 * HD, NS = HD / 16, NB = DV / 32;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  unsigned char* Kimg = smem;      // the first map's image, the second one's behind it
  unsigned char* Vimg = smem + 2 * Img<HD>::BYTES;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, mp = wave & 1, rg = wave >> 1, i = lane & 31, g = lane >> 5;
  const Work wk = work_of(a.n_tiles, a.B + (a.cu_q != nullptr ? 1 : 0), a.H, a.causal != 0);
  const int h = wk.h, hk = h / (a.H / a.Hkv), hd = a.hd, dv = 2 * hd;

  if (wk.b == a.B) {      // rows behind the last session: zeros
    if (wk.split != 0) return;
    const long long r0 = rows_used(a.cu_q, a.B, a.Nq);
    for (long long r = r0 + wk.tile; r < a.Nq; r += a.n_tiles) {
      for (int c = tid; c < dv; c += NT) a.y[r * a.ldy + (long long)h * dv + c] = 0.f;
      if (a.o12 != nullptr) for (int c = tid; c < 2 * dv; c += NT) a.o12[(r * a.H + h) * 2 * dv + c] = 0.f;
      if (a.lse != nullptr && tid < 2) a.lse[(r * a.H + h) * 2 + tid] = 0.f;
    }
    return;
  }
  long long qr0, kr0; int nq, nk;
  rows_of(a.cu_q, wk.b, a.Lq, a.Nq, qr0, nq);
  rows_of(a.cu_k, wk.b, a.Lk, a.Nk, kr0, nk);
  const int off = nk - nq;
  const float qscale = a.scale * LOG2E;
  const float lam = a.lam[h];

  for (int tile = wk.tile; tile * OWN < nq; tile += a.n_tiles) {
    const int q0 = tile * OWN + 32 * rg, qi = q0 + i;
    const bool qok = qi < nq;
    const float* qrow = a.q + (qr0 + (qok ? qi : 0)) * a.ldq + (long long)(2 * h + mp) * hd;
    P3 Qp[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) Qp[s] = load_planes<MODE>(qrow, 16 * s + 8 * g, hd, qok, qscale);
    f32x16 O[NB];
#pragma unroll
    for (int cb = 0; cb < NB; ++cb) O[cb] = zero16();
    float m = -INFINITY, lsum = 0.f;

    const int k_end = a.causal ? min(nk, tile * OWN + OWN + off) : nk;      // keys that some row of the tile sees
    int c_lo = 0, c_hi = k_end > 0 ? (k_end + CH - 1) / CH : 0;
    if (a.n_split > 1) {
      const int each = (c_hi + a.n_split - 1) / a.n_split;
      c_lo = min(c_hi, wk.split * each);
      c_hi = min(c_hi, c_lo + each);
    }
    for (int c = c_lo; c < c_hi; ++c) {
      const int t0 = c * CH;
      const unsigned live = live_keys(a, kr0, t0, nk, lane);
      if (live == 0u) continue;
      __syncthreads();
      {
        const float* kb = a.k + (kr0 + t0) * a.ldk + (long long)(2 * hk) * hd;
        stage<HD, MODE>(kb, a.ldk, hd, live, 1.f, Kimg, tid);
        stage<HD, MODE>(kb + hd, a.ldk, hd, live, 1.f, Kimg + Img<HD>::BYTES, tid);
        stage<DV, MODE>(a.v + (kr0 + t0) * a.ldv + (long long)hk * dv, a.ldv, dv, live, 1.f, Vimg, tid);
      }
      __syncthreads();
      if (q0 >= nq || (a.causal && t0 > q0 + 31 + off)) continue;      // (wave-uniform) nothing of the chunk is visible to the row group
      f32x16 S = zero16();
      rows_dot<HD, NS>(Kimg + mp * Img<HD>::BYTES, 0, Qp, i, g, S);
      float sc[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[r] = S[r];
      if (live != 0xFFFFFFFFu || (a.causal && t0 + 31 > q0 + off)) {
        const int last = a.causal ? qi + off - t0 : 31;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int j = reg_row(r, g);
          sc[r] = (j <= last && ((live >> j) & 1u)) ? sc[r] : -INFINITY;
        }
      }
      float mx = sc[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) mx = fmaxf(mx, sc[r]);
      mx = fmaxf(m, fmaxf(mx, __shfl_xor(mx, 32, 64)));
      const float base = mx == -INFINITY ? 0.f : mx;      // a row that has seen no key yet
      const float alpha = __builtin_amdgcn_exp2f(m - base);
      float ps = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) { sc[r] = __builtin_amdgcn_exp2f(sc[r] - base); ps += sc[r]; }
      lsum = lsum * alpha + ps;
      if (__any(mx != m)) {
#pragma unroll
        for (int cb = 0; cb < NB; ++cb) O[cb] *= alpha;
      }
      m = mx;
      P3 Pp[2];
      split16(sc, Pp);
      cols_dot<DV, NB>(Vimg, 0, Pp, lane, O);
    }
    const float l = lsum + __shfl_xor(lsum, 32, 64);
    if (a.n_split > 1) {      // partial sums as they are; diff_combine_kernel joins the splits
      if (qok) {
        const long long at = (((long long)wk.split * a.Nq + qr0 + qi) * a.H + h) * 2 + mp;
        if (g == 0) { a.ml[2 * at] = m; a.ml[2 * at + 1] = l; }
        float* o = a.part + at * dv;
#pragma unroll
        for (int cb = 0; cb < NB; ++cb)
#pragma unroll
          for (int r = 0; r < 4; ++r) put4<MODE>(o, 32 * cb + 8 * r + 4 * g, dv, f32x4{O[cb][4 * r], O[cb][4 * r + 1], O[cb][4 * r + 2], O[cb][4 * r + 3]});
      }
      continue;
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);      // (a NaN sum stays one)
#pragma unroll
    for (int cb = 0; cb < NB; ++cb) O[cb] *= inv;
    if (qok && a.lse != nullptr && g == 0) a.lse[((qr0 + qi) * a.H + h) * 2 + mp] = l > 0.f ? m + __builtin_amdgcn_logf(l) : 0.f;
    if (qok && a.o12 != nullptr) {
      float* o = a.o12 + (((qr0 + qi) * a.H + h) * 2 + mp) * (long long)dv;
#pragma unroll
      for (int cb = 0; cb < NB; ++cb)
#pragma unroll
        for (int r = 0; r < 4; ++r) put4<MODE>(o, 32 * cb + 8 * r + 4 * g, dv, f32x4{O[cb][4 * r], O[cb][4 * r + 1], O[cb][4 * r + 2], O[cb][4 * r + 3]});
    }
    // the second map's wave hands its output over; the first one's subtracts, normalises and writes
    __syncthreads();
    f32x4* x = reinterpret_cast<f32x4*>(smem) + rg * (NB * 4 * 64);
    if (mp == 1) {
#pragma unroll
      for (int cb = 0; cb < NB; ++cb)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[(cb * 4 + r) * 64 + lane] = f32x4{O[cb][4 * r], O[cb][4 * r + 1], O[cb][4 * r + 2], O[cb][4 * r + 3]};
    }
    __syncthreads();
    if (mp == 0) {
      float ss = 0.f;
#pragma unroll
      for (int cb = 0; cb < NB; ++cb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const f32x4 o2 = x[(cb * 4 + r) * 64 + lane];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            O[cb][4 * r + e] -= lam * o2[e];
            ss += O[cb][4 * r + e] * O[cb][4 * r + e];
          }
        }
      ss += __shfl_xor(ss, 32, 64);
      const float f = a.norm_w != nullptr ? a.out_scale / sqrtf(ss / (float)dv + a.eps) : a.out_scale;
      if (qok) {
        float* o = a.y + (qr0 + qi) * a.ldy + (long long)h * dv;
#pragma unroll
        for (int cb = 0; cb < NB; ++cb)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int col = 32 * cb + 8 * r + 4 * g;
            f32x4 t;
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = O[cb][4 * r + e] * f * ((a.norm_w != nullptr && col + e < dv) ? a.norm_w[col + e] : 1.f);
            put4<MODE>(o, col, dv, t);
          }
      }
    }
  }
}

// join of the key splits: one workgroup per (row, head); a lane holds the statistics of a split (n_split <= 64), then a thread sums one value
// column over its share of the splits
__global__ __launch_bounds__(NT) void diff_combine_kernel(Args a) {
  __shared__ float wgt[2][64], sums[NT], res[2][128], ssq[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, dv = 2 * a.hd;
  const long long at = blockIdx.x, row = at / a.H, plane = a.Nq * a.H;
  const int h = (int)(at % a.H);
  if (row >= rows_used(a.cu_q, a.B, a.Nq)) return;      // (zeros already)
  if (wave < 2) {
    const bool on = lane < a.n_split;
    const long long p = ((long long)lane * plane + at) * 2 + wave;
    const float m = on ? a.ml[2 * p] : -INFINITY, l = on ? a.ml[2 * p + 1] : 0.f, mx = wave_max(m), base = mx == -INFINITY ? 0.f : mx;
    const float e = on ? __builtin_amdgcn_exp2f(m - base) : 0.f, total = wave_sum(l * e);
    wgt[wave][lane] = e * (total > 0.f ? 1.f / total : (total == 0.f ? 0.f : total));
    if (a.lse != nullptr && lane == 0) a.lse[at * 2 + wave] = total > 0.f ? mx + __builtin_amdgcn_logf(total) : 0.f;
  }
  const int slots = NT / dv, c = tid % dv, sub = tid / dv;
  for (int mp = 0; mp < 2; ++mp) {
    __syncthreads();
    float x = 0.f;
    if (sub < slots)
      for (int s = sub; s < a.n_split; s += slots) x = fmaf(a.part[(((long long)s * plane + at) * 2 + mp) * dv + c], wgt[mp][s], x);
    sums[tid] = x;
    __syncthreads();
    if (tid < dv) {
      for (int k = 1; k < slots; ++k) x += sums[k * dv + tid];
      res[mp][tid] = x;
      if (a.o12 != nullptr) a.o12[(at * 2 + mp) * dv + tid] = x;
    }
  }
  const float o = tid < dv ? res[0][tid] - a.lam[h] * res[1][tid] : 0.f;      // (its own columns: no barrier)
  if (tid < 128) {
    const float q = wave_sum(o * o);
    if (lane == 0) ssq[wave] = q;
  }
  __syncthreads();
  const float f = a.norm_w != nullptr ? a.out_scale / sqrtf((ssq[0] + ssq[1]) / (float)dv + a.eps) : a.out_scale;
  if (tid < dv) a.y[row * a.ldy + (long long)h * dv + tid] = o * f * (a.norm_w != nullptr ? a.norm_w[tid] : 1.f);
}

// ---- backward, in front: gradient of o, delta_m = do . o_m, and the sums behind dlam and dw -----------------------------------------------
// HD / 2 lanes per (row, head), four columns each; a lane group keeps its head, so dlam and dw stay in registers over all of its rows.  They
// are summed in 64 bits, per workgroup, in a fixed order.
constexpr int PRE_WG = 1024;      // workgroups at most: the partials are [PRE_WG][H + 2 hd] doubles

template <int LANES> __device__ __forceinline__ float group_sum(float v) {      // 16 or 32 neighbouring lanes
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, true));
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x4E, 0xF, 0xF, true));
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x141, 0xF, 0xF, true));
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x140, 0xF, 0xF, true));
  if (LANES == 32) v += __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, v), 0x401F));
  return v;
}
template <bool VEC> __device__ __forceinline__ f32x4 get4(const float* p, int c, int ncol) {
  f32x4 x{0.f, 0.f, 0.f, 0.f};
  if (VEC) {
    if (c < ncol) x = *reinterpret_cast<const f32x4*>(p + c);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < ncol) x[e] = p[c + e];
  }
  return x;
}

template <int HD, bool VEC>
__global__ __launch_bounds__(NT) void diff_bwd_pre_kernel(Args a, const float* dy, long long lddy, float* dout, float* delta, double* part) {
  constexpr int LANES = HD / 2, GROUPS = NT / LANES;
  __shared__ double sw[GROUPS][2 * HD], sl[GROUPS];
  const int tid = threadIdx.x, gid = tid / LANES, c = (tid % LANES) * 4, dv = 2 * a.hd, H = a.H;
  const long long used = rows_used(a.cu_q, a.B, a.Nq);
  const long long gg = (long long)blockIdx.x * GROUPS + gid, n_groups = (long long)gridDim.x * GROUPS;
  const int h = (int)(gg % H);
  const long long step = n_groups / H;                       // rows are dealt to the step lane groups of a head; leftover groups do nothing
  const float lam = a.lam[h], inv = 1.f / (float)dv;
  const f32x4 w = a.norm_w != nullptr ? get4<VEC>(a.norm_w, c, dv) * a.out_scale : f32x4{a.out_scale, a.out_scale, a.out_scale, a.out_scale};
  double dw[4] = {0.0, 0.0, 0.0, 0.0}, dl = 0.0;
  for (long long row = gg < step * H ? gg / H : a.Nq; row < a.Nq; row += step) {
    const long long at = row * H + h;
    float* dst = dout + at * dv;
    if (row >= used) {
      put4<VEC ? 1 : 2>(dst, c, dv, f32x4{0.f, 0.f, 0.f, 0.f});
      if (c == 0) { delta[at * 2] = 0.f; delta[at * 2 + 1] = 0.f; }
      continue;
    }
    const f32x4 o1 = get4<VEC>(a.o12 + at * 2 * dv, c, dv), o2 = get4<VEC>(a.o12 + (at * 2 + 1) * dv, c, dv);
    const f32x4 g = get4<VEC>(dy + row * lddy + (long long)h * dv, c, dv), e = g * w;
    f32x4 d = e;
    if (a.norm_w != nullptr) {
      const f32x4 x = o1 - o2 * lam;
      const float r = 1.f / sqrtf(group_sum<LANES>(x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3]) * inv + a.eps);
      const f32x4 u = x * r;
      const float mean = group_sum<LANES>(e[0] * u[0] + e[1] * u[1] + e[2] * u[2] + e[3] * u[3]) * inv;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        d[k] = r * (e[k] - u[k] * mean);
        dw[k] += (double)(a.out_scale * g[k] * u[k]);
      }
    }
    put4<VEC ? 1 : 2>(dst, c, dv, d);
    const float s1 = group_sum<LANES>(d[0] * o1[0] + d[1] * o1[1] + d[2] * o1[2] + d[3] * o1[3]);
    const float s2 = group_sum<LANES>(d[0] * o2[0] + d[1] * o2[1] + d[2] * o2[2] + d[3] * o2[3]);
    if (c == 0) { delta[at * 2] = s1; delta[at * 2 + 1] = s2; }
    dl -= (double)s2;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) sw[gid][c + k] = dw[k];
  if (c == 0) sl[gid] = dl;
  __syncthreads();
  double* out = part + (long long)blockIdx.x * (H + dv);
  for (int x = tid; x < dv; x += NT) {
    double s = sw[0][x];
    for (int k = 1; k < GROUPS; ++k) s += sw[k][x];
    out[H + x] = s;
  }
  for (int x = tid; x < H; x += NT) {
    double s = 0.0;
    for (int k = 0; k < GROUPS; ++k)
      if ((int)(((long long)blockIdx.x * GROUPS + k) % H) == x) s += sl[k];
    out[x] = s;
  }
}

__global__ __launch_bounds__(64) void diff_bwd_sums_kernel(const double* part, int n, int H, int dv, float* dlam, float* dw) {
  const int W = H + dv, c = blockIdx.x;
  double s = 0.0;
  for (int r = threadIdx.x; r < n; r += 64) s += part[(long long)r * W + c];
  s = wave_sum_d(s);
  if (threadIdx.x == 0) {
    if (c < H) dlam[c] = (float)s;
    else if (dw != nullptr) dw[c - H] = (float)s;
  }
}

// ---- backward, dQ: the owner is a query; both maps need G^T = V dO^T, each wave makes it over half of V's columns and they swap halves ------
template <int HD, int MODE>
__global__ __launch_bounds__(NT, 2) void diff_bwd_dq_kernel(Args a) {
  constexpr int DV = 2 * HD, NS = HD / 16, NB = HD / 32;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  unsigned char* Kimg = smem;      // the first map's image, the second one's behind it
  unsigned char* Vimg = smem + 2 * Img<HD>::BYTES;
  f32x4* swap = reinterpret_cast<f32x4*>(smem + 2 * Img<HD>::BYTES + Img<DV>::BYTES);      // [wave][4][64]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, mp = wave & 1, rg = wave >> 1, i = lane & 31, g = lane >> 5;
  const Work wk = work_of(a.n_tiles, a.B + (a.cu_q != nullptr ? 1 : 0), a.H, a.causal != 0);
  const int h = wk.h, hk = h / (a.H / a.Hkv), hd = a.hd, dv = 2 * hd;
  if (wk.b == a.B) {      // rows behind the last session have no gradient
    for (long long r = rows_used(a.cu_q, a.B, a.Nq) + wk.tile; r < a.Nq; r += a.n_tiles)
      for (int c = tid; c < dv; c += NT) a.dq[r * a.lddq + (long long)h * dv + c] = 0.f;
    return;
  }
  long long qr0, kr0; int nq, nk;
  rows_of(a.cu_q, wk.b, a.Lq, a.Nq, qr0, nq);
  rows_of(a.cu_k, wk.b, a.Lk, a.Nk, kr0, nk);
  const int off = nk - nq;
  const float qscale = a.scale * LOG2E, sign = mp == 0 ? 1.f : -a.lam[h];

  for (int tile = wk.tile; tile * OWN < nq; tile += a.n_tiles) {
    const int q0 = tile * OWN + 32 * rg, qi = q0 + i;
    const bool qok = qi < nq;
    const long long grow = qr0 + (qok ? qi : 0);
    P3 Qp[NS], Dp[NS];      // dO: columns mp * HD .. of the padded 2 HD
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      Qp[s] = load_planes<MODE>(a.q + grow * a.ldq + (long long)(2 * h + mp) * hd, 16 * s + 8 * g, hd, qok, qscale);
      Dp[s] = load_planes<MODE>(a.dout + grow * a.lddo + (long long)h * dv, mp * HD + 16 * s + 8 * g, dv, qok, 1.f);
    }
    const float lse = qok ? a.lse[(grow * a.H + h) * 2 + mp] : 0.f, dl = qok ? a.delta[(grow * a.H + h) * 2 + mp] : 0.f;
    f32x16 dQ[NB];
#pragma unroll
    for (int cb = 0; cb < NB; ++cb) dQ[cb] = zero16();
    const int k_end = a.causal ? min(nk, tile * OWN + OWN + off) : nk;
    const int n_ch = k_end > 0 ? (k_end + CH - 1) / CH : 0;
    for (int c = 0; c < n_ch; ++c) {
      const int t0 = c * CH;
      const unsigned live = live_keys(a, kr0, t0, nk, lane);
      if (live == 0u) continue;
      __syncthreads();
      {
        const float* kb = a.k + (kr0 + t0) * a.ldk + (long long)(2 * hk) * hd;
        stage<HD, MODE>(kb, a.ldk, hd, live, 1.f, Kimg, tid);
        stage<HD, MODE>(kb + hd, a.ldk, hd, live, 1.f, Kimg + Img<HD>::BYTES, tid);
        stage<DV, MODE>(a.v + (kr0 + t0) * a.ldv + (long long)hk * dv, a.ldv, dv, live, 1.f, Vimg, tid);
      }
      __syncthreads();
      const bool on = q0 < nq && !(a.causal && t0 > q0 + 31 + off);      // (the same for the two waves of a row group)
      f32x16 S = zero16(), G = zero16();
      if (on) {
        rows_dot<HD, NS>(Kimg + mp * Img<HD>::BYTES, 0, Qp, i, g, S);
        rows_dot<DV, NS>(Vimg, mp * HD, Dp, i, g, G);
#pragma unroll
        for (int r = 0; r < 4; ++r) swap[(wave * 4 + r) * 64 + lane] = f32x4{G[4 * r], G[4 * r + 1], G[4 * r + 2], G[4 * r + 3]};
      }
      __syncthreads();
      if (!on) continue;
      float ds[16];
      const bool edge = live != 0xFFFFFFFFu || (a.causal && t0 + 31 > q0 + off);
      const int last = a.causal ? qi + off - t0 : 31;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x4 other = swap[((wave ^ 1) * 4 + r) * 64 + lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = reg_row(4 * r + e, g);
          float p = __builtin_amdgcn_exp2f(S[4 * r + e] - lse);
          if (edge) p = (j <= last && ((live >> j) & 1u)) ? p : 0.f;
          ds[4 * r + e] = p * ((G[4 * r + e] + other[e]) - dl);
        }
      }
      P3 dsp[2];
      split16(ds, dsp);
      cols_dot<HD, NB>(Kimg + mp * Img<HD>::BYTES, 0, dsp, lane, dQ);
    }
    if (qok) {
      float* o = a.dq + grow * a.lddq + (long long)(2 * h + mp) * hd;
      const float f = a.scale * sign;
#pragma unroll
      for (int cb = 0; cb < NB; ++cb)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          put4<MODE>(o, 32 * cb + 8 * r + 4 * g, hd, f32x4{dQ[cb][4 * r] * f, dQ[cb][4 * r + 1] * f, dQ[cb][4 * r + 2] * f, dQ[cb][4 * r + 3] * f});
    }
  }
}

// ---- backward, dK and dV: the owner is a key; the query heads of its group are summed in a fixed order ---------------------------------------
// The two waves of a row group swap their halves of G and their probabilities: each makes dK of its map and dV of its half of the columns.
template <int HD, int MODE>
__global__ __launch_bounds__(NT, 2) void diff_bwd_dkv_kernel(Args a) {
  constexpr int DV = 2 * HD, NS = HD / 16, NB = HD / 32;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  unsigned char* Qimg = smem;      // the first map's image, the second one's behind it
  unsigned char* Dimg = smem + 2 * Img<HD>::BYTES;
  f32x4* swap = reinterpret_cast<f32x4*>(smem + 2 * Img<HD>::BYTES + Img<DV>::BYTES);      // [wave][8][64]: G halves, probabilities
  float* stat = reinterpret_cast<float*>(swap + 4 * 8 * 64);                               // [map][lse 32 | delta 32]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, mp = wave & 1, rg = wave >> 1, i = lane & 31, g = lane >> 5;
  const Work wk = work_of(a.n_tiles, a.B + (a.cu_k != nullptr ? 1 : 0), a.Hkv, false);
  const int hk = wk.h, rep = a.H / a.Hkv, hd = a.hd, dv = 2 * hd;
  if (wk.b == a.B) {
    for (long long r = rows_used(a.cu_k, a.B, a.Nk) + wk.tile; r < a.Nk; r += a.n_tiles)
      for (int c = tid; c < dv; c += NT) {
        a.dk[r * a.lddk + (long long)hk * dv + c] = 0.f;
        a.dv[r * a.lddv + (long long)hk * dv + c] = 0.f;
      }
    return;
  }
  long long qr0, kr0; int nq, nk;
  rows_of(a.cu_q, wk.b, a.Lq, a.Nq, qr0, nq);
  rows_of(a.cu_k, wk.b, a.Lk, a.Nk, kr0, nk);
  const int off = nk - nq;
  const float kscale = a.scale * LOG2E;

  for (int tile = wk.tile; tile * OWN < nk; tile += a.n_tiles) {
    const int k0 = tile * OWN + 32 * rg, ki = k0 + i;
    const bool kin = ki < nk;
    const bool kok = kin && (a.key_ids == nullptr || a.key_ids[kr0 + ki] != 0);
    const long long grow = kr0 + (kin ? ki : 0);
    P3 Kp[NS], Vp[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      Kp[s] = load_planes<MODE>(a.k + grow * a.ldk + (long long)(2 * hk + mp) * hd, 16 * s + 8 * g, hd, kok, kscale);
      Vp[s] = load_planes<MODE>(a.v + grow * a.ldv + (long long)hk * dv, mp * HD + 16 * s + 8 * g, dv, kok, 1.f);
    }
    f32x16 dK[NB], dV[NB];
#pragma unroll
    for (int cb = 0; cb < NB; ++cb) { dK[cb] = zero16(); dV[cb] = zero16(); }
    const int c_lo = a.causal ? max(0, tile * OWN - off) / CH : 0, c_hi = (nq + CH - 1) / CH;
    for (int hh = 0; hh < rep; ++hh) {
      const int h = hk * rep + hh;
      const float lam = a.lam[h], sign = mp == 0 ? 1.f : -lam;
      for (int c = c_lo; c < c_hi; ++c) {
        const int t0 = c * CH, left = nq - t0;
        const unsigned rows = left >= 32 ? 0xFFFFFFFFu : (1u << left) - 1u;
        __syncthreads();
        {
          const float* qb = a.q + (qr0 + t0) * a.ldq + (long long)(2 * h) * hd;
          stage<HD, MODE>(qb, a.ldq, hd, rows, 1.f, Qimg, tid);
          stage<HD, MODE>(qb + hd, a.ldq, hd, rows, 1.f, Qimg + Img<HD>::BYTES, tid);
          stage<DV, MODE>(a.dout + (qr0 + t0) * a.lddo + (long long)h * dv, a.lddo, dv, rows, 1.f, Dimg, tid);
          if (tid < 128) {      // a row behind the session's end: exp2(-inf) = 0
            const int m = tid >> 6, what = (tid >> 5) & 1, r = tid & 31;
            const long long at = ((qr0 + t0 + r) * a.H + h) * 2 + m;
            stat[tid] = r < left ? (what == 0 ? a.lse[at] : a.delta[at]) : (what == 0 ? INFINITY : 0.f);
          }
        }
        __syncthreads();
        const bool on = k0 < nk && !(a.causal && t0 + 31 + off < k0);
        f32x16 S = zero16(), G = zero16();
        float p[16];
        if (on) {
          rows_dot<HD, NS>(Qimg + mp * Img<HD>::BYTES, 0, Kp, i, g, S);
          rows_dot<DV, NS>(Dimg, mp * HD, Vp, i, g, G);
          const bool edge = a.causal && t0 + off < k0 + 31;
          const int first = a.causal ? ki - off - t0 : -1;      // the first row of the chunk that sees this key
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const f32x4 ls = *reinterpret_cast<const f32x4*>(stat + mp * 64 + 8 * r + 4 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = __builtin_amdgcn_exp2f(S[4 * r + e] - ls[e]);
              p[4 * r + e] = (kok && (!edge || reg_row(4 * r + e, g) >= first)) ? x : 0.f;
            }
            swap[(wave * 8 + r) * 64 + lane] = f32x4{G[4 * r], G[4 * r + 1], G[4 * r + 2], G[4 * r + 3]};
            swap[(wave * 8 + 4 + r) * 64 + lane] = f32x4{p[4 * r], p[4 * r + 1], p[4 * r + 2], p[4 * r + 3]};
          }
        }
        __syncthreads();
        if (!on) continue;
        float ds[16], d[16];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const f32x4 og = swap[((wave ^ 1) * 8 + r) * 64 + lane], op = swap[((wave ^ 1) * 8 + 4 + r) * 64 + lane];
          const f32x4 dl = *reinterpret_cast<const f32x4*>(stat + mp * 64 + 32 + 8 * r + 4 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int x = 4 * r + e;
            ds[x] = sign * p[x] * ((G[x] + og[e]) - dl[e]);
            d[x] = mp == 0 ? p[x] - lam * op[e] : op[e] - lam * p[x];
          }
        }
        P3 w[2];
        split16(ds, w);
        cols_dot<HD, NB>(Qimg + mp * Img<HD>::BYTES, 0, w, lane, dK);
        split16(d, w);
        cols_dot<DV, NB>(Dimg, mp * HD, w, lane, dV);
      }
    }
    if (kin) {
      float* ok = a.dk + grow * a.lddk + (long long)(2 * hk + mp) * hd;
      float* ov = a.dv + grow * a.lddv + (long long)hk * dv;
#pragma unroll
      for (int cb = 0; cb < NB; ++cb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int col = 32 * cb + 8 * r + 4 * g;
          put4<MODE>(ok, col, hd, f32x4{dK[cb][4 * r] * a.scale, dK[cb][4 * r + 1] * a.scale, dK[cb][4 * r + 2] * a.scale, dK[cb][4 * r + 3] * a.scale});
          put4<MODE>(ov, mp * HD + col, dv, f32x4{dV[cb][4 * r], dV[cb][4 * r + 1], dV[cb][4 * r + 2], dV[cb][4 * r + 3]});
        }
    }
  }
}

// ---- few query rows: the products are matrix-vector products, the keys and values are read once and the loads are the work ---------------------
// A workgroup takes the R queries (rows x heads) that share a key head through its share of the keys.  A wave reads TK keys at a time straight
// into registers: a key's two maps (and its value row) lie across 2 HD / 4 lanes, four columns each, so every load is whole cache lines; a
// dot product is four multiply-adds and a sum over the lanes of its map (cross-lane adds, no LDS), the value sums stay with the lanes' columns.  Every wave
// keeps its own running maximum and sum; no barrier in the loop, 16 loads of 16 bytes in flight per lane.
constexpr int MAXR = 8;

template <int CTRL> __device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
template <int HD> __device__ __forceinline__ float map_sum(float v) {      // over the HD / 4 lanes of a key's map
  v += dpp<0xB1>(v);       // lane ^ 1
  v += dpp<0x4E>(v);       // lane ^ 2
  v += dpp<0x141>(v);      // mirrored in 8 lanes
  if (HD == 64) v += dpp<0x140>(v);      // mirrored in 16 lanes
  return v;
}
template <int HD> __device__ __forceinline__ float other_map(float v) {
  if (HD == 32) return dpp<0x128>(v);      // rotated by 8 in 16 lanes
  return __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, v), 0x401F));      // lane ^ 16
}
template <int HD> __device__ __forceinline__ float keys_max(float v) {      // over the keys of one load
  if (HD == 32) v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
template <int HD> __device__ __forceinline__ float keys_sum(float v) {
  if (HD == 32) v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}
constexpr int decode_keys(int HDP) { return HDP == 32 ? 32 : 16; }      // TK

template <int HD, int MODE, int R>
__global__ __launch_bounds__(NT, 2) void diff_decode_kernel(Args a) {
  constexpr int DV = 2 * HD, LPK = HD / 2, KPL = 64 / LPK, NL = 8, TK = KPL * NL;
  __shared__ float wstat[4][R][2][2], wacc[4][R][2][DV];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, kk = lane / LPK, c4 = lane % LPK, mp = c4 / (HD / 4), col = (c4 % (HD / 4)) * 4;
  const int b = blockIdx.x / a.Hkv, hk = blockIdx.x % a.Hkv, rep = a.H / a.Hkv, hd = a.hd, dv = 2 * hd;
  if (b == a.B) {      // rows behind the last session: zeros
    if (blockIdx.y != 0) return;
    const long long r0 = rows_used(a.cu_q, a.B, a.Nq), cols = (long long)rep * dv;
    for (long long x = tid; x < (a.Nq - r0) * cols; x += NT) a.y[(r0 + x / cols) * a.ldy + (long long)hk * rep * dv + x % cols] = 0.f;
    return;
  }
  long long qr0, kr0; int nq, nk;
  rows_of(a.cu_q, b, a.Lq, a.Nq, qr0, nq);
  rows_of(a.cu_k, b, a.Lk, a.Nk, kr0, nk);
  const int off = nk - nq, per = R / rep;          // query rows of a pass: every one of them with its `rep` heads
  const float qscale = a.scale * LOG2E;
  for (int first = 0; first < nq; first += per) {
    const int rows = min(per, nq - first);
    f32x4 qv[R], acc[R][2];
    float m[R], l[R];
#pragma unroll
    for (int w = 0; w < R; ++w) {                  // query w = (row w / rep, head w % rep)
      qv[w] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (w < rows * rep) {
        const float* p = a.q + (qr0 + first + w / rep) * a.ldq + (long long)(2 * (hk * rep + w % rep) + mp) * hd + col;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (MODE == 0 || col + e < hd) qv[w][e] = p[e] * qscale;
      }
      acc[w][0] = acc[w][1] = f32x4{0.f, 0.f, 0.f, 0.f};
      m[w] = -INFINITY;
      l[w] = 0.f;
    }
    const int k_end = a.causal ? max(0, min(nk, first + rows + off)) : nk;
    const int n_t = (k_end + TK - 1) / TK, each = (n_t + a.n_split - 1) / a.n_split, t_lo = min(n_t, (int)blockIdx.y * each), t_hi = min(n_t, t_lo + each);
    for (int t = t_lo + wave; t < t_hi; t += 4) {
      f32x4 kf[NL], vf[NL];
      unsigned live = 0u;
#pragma unroll
      for (int u = 0; u < NL; ++u) {
        const int key = t * TK + u * KPL + kk;
        kf[u] = vf[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (key < k_end && (a.key_ids == nullptr || a.key_ids[kr0 + key] != 0)) {
          live |= 1u << u;
          const float* kp = a.k + (kr0 + key) * a.ldk + (long long)(2 * hk + mp) * hd + col;
          const float* vp = a.v + (kr0 + key) * a.ldv + (long long)hk * dv + 4 * c4;
          if (MODE < 2) {
            if (MODE == 0 || col < hd) kf[u] = *reinterpret_cast<const f32x4*>(kp);
            if (MODE == 0 || 4 * c4 < dv) vf[u] = *reinterpret_cast<const f32x4*>(vp);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (col + e < hd) kf[u][e] = kp[e];
              if (4 * c4 + e < dv) vf[u][e] = vp[e];
            }
          }
        }
      }
#pragma unroll
      for (int w = 0; w < R; ++w) {
        if (w >= rows * rep) break;
        const int last = a.causal ? first + w / rep + off : 0x7FFFFFFF;
        float s[NL], mx = m[w];
#pragma unroll
        for (int u = 0; u < NL; ++u) {
          s[u] = map_sum<HD>(fmaf(qv[w][0], kf[u][0], qv[w][1] * kf[u][1]) + fmaf(qv[w][2], kf[u][2], qv[w][3] * kf[u][3]));
          if (((live >> u) & 1u) == 0u || t * TK + u * KPL + kk > last) s[u] = -INFINITY;
          mx = fmaxf(mx, s[u]);
        }
        mx = keys_max<HD>(mx);
        const float base = mx == -INFINITY ? 0.f : mx, alpha = __builtin_amdgcn_exp2f(m[w] - base);
        m[w] = mx;
        const float alpha_o = other_map<HD>(alpha);
        acc[w][0] *= mp == 0 ? alpha : alpha_o;
        acc[w][1] *= mp == 0 ? alpha_o : alpha;
        float ps = 0.f;
#pragma unroll
        for (int u = 0; u < NL; ++u) {
          const float p = __builtin_amdgcn_exp2f(s[u] - base), po = other_map<HD>(p), p0 = mp == 0 ? p : po, p1 = mp == 0 ? po : p;
          ps += p;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            acc[w][0][e] = fmaf(p0, vf[u][e], acc[w][0][e]);
            acc[w][1][e] = fmaf(p1, vf[u][e], acc[w][1][e]);
          }
        }
        l[w] = l[w] * alpha + ps;
      }
    }
    __syncthreads();      // (the previous pass's readers are done)
#pragma unroll
    for (int w = 0; w < R; ++w) {
      const float lt = keys_sum<HD>(l[w]);
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[w][q][e] = keys_sum<HD>(acc[w][q][e]);
      if (kk == 0) {
        if (c4 % (HD / 4) == 0) { wstat[wave][w][mp][0] = m[w]; wstat[wave][w][mp][1] = lt; }
        *reinterpret_cast<f32x4*>(&wacc[wave][w][0][4 * c4]) = acc[w][0];
        *reinterpret_cast<f32x4*>(&wacc[wave][w][1][4 * c4]) = acc[w][1];
      }
    }
    __syncthreads();
    for (int u = wave; u < rows * rep; u += 4) {            // query u: this wave
      const long long row = qr0 + first + u / rep;
      const int h = hk * rep + u % rep;
      float o[2][2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float mx = -INFINITY, lt = 0.f, s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) mx = fmaxf(mx, wstat[k][u][q][0]);
        const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float e = __builtin_amdgcn_exp2f(wstat[k][u][q][0] - base);
          lt = fmaf(wstat[k][u][q][1], e, lt);
          s0 = fmaf(wacc[k][u][q][lane], e, s0);      // (DV >= 64)
          if (DV > 64) s1 = fmaf(wacc[k][u][q][(lane + 64) % DV], e, s1);
        }
        if (a.n_split > 1) {
          const long long at = (((long long)blockIdx.y * a.Nq + row) * a.H + h) * 2 + q;
          if (lane == 0) { a.ml[2 * at] = mx; a.ml[2 * at + 1] = lt; }
          if (lane < dv) a.part[at * dv + lane] = s0;
          if (lane + 64 < dv) a.part[at * dv + lane + 64] = s1;
        }
        const float inv = lt > 0.f ? 1.f / lt : (lt == 0.f ? 0.f : lt);
        o[q][0] = s0 * inv;
        o[q][1] = s1 * inv;
      }
      if (a.n_split > 1) continue;
      const float lam = a.lam[h];
      const float x0 = o[0][0] - lam * o[1][0], x1 = o[0][1] - lam * o[1][1];      // (columns behind dv hold zeros)
      const float ss = wave_sum(x0 * x0 + x1 * x1);
      const float f = a.norm_w != nullptr ? a.out_scale / sqrtf(ss / (float)dv + a.eps) : a.out_scale;
      float* y = a.y + row * a.ldy + (long long)h * dv;
      if (lane < dv) y[lane] = x0 * f * (a.norm_w != nullptr ? a.norm_w[lane] : 1.f);
      if (lane + 64 < dv) y[lane + 64] = x1 * f * (a.norm_w != nullptr ? a.norm_w[lane + 64] : 1.f);
    }
  }
}

// ---- lam = exp(q1 . k1) - exp(q2 . k2) + init, one wave per head ----------------------------------------------------------------------------
__device__ __forceinline__ float wave_dot(const float* x, const float* y, int n, int lane) {
  float s = 0.f;
  for (int c = lane; c < n; c += 64) s = fmaf(x[c], y[c], s);
  return wave_sum(s);
}
__global__ __launch_bounds__(64) void diff_lambda_fwd_kernel(const float* q1, const float* k1, const float* q2, const float* k2, float init, int hd, float* lam) {
  const long long o = (long long)blockIdx.x * hd;
  const float e1 = expf(wave_dot(q1 + o, k1 + o, hd, threadIdx.x)), e2 = expf(wave_dot(q2 + o, k2 + o, hd, threadIdx.x));
  if (threadIdx.x == 0) lam[blockIdx.x] = e1 - e2 + init;
}
__global__ __launch_bounds__(64) void diff_lambda_bwd_kernel(const float* dlam, const float* q1, const float* k1, const float* q2, const float* k2, int hd,
                                                             float* dq1, float* dk1, float* dq2, float* dk2) {
  const long long o = (long long)blockIdx.x * hd;
  const float g = dlam[blockIdx.x];
  const float e1 = g * expf(wave_dot(q1 + o, k1 + o, hd, threadIdx.x)), e2 = -g * expf(wave_dot(q2 + o, k2 + o, hd, threadIdx.x));
  for (int c = threadIdx.x; c < hd; c += 64) {
    dq1[o + c] = e1 * k1[o + c];
    dk1[o + c] = e1 * q1[o + c];
    dq2[o + c] = e2 * k2[o + c];
    dk2[o + c] = e2 * q2[o + c];
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------------------
bool vec_ok(const void* p, long long ld) { return ((uintptr_t)p & 15u) == 0 && ld % 4 == 0; }
int pad_hd(int hd) { return hd <= 32 ? 32 : 64; }

struct Plan { bool decode; int n_split; };
// Training keeps the outputs of both maps and always takes the matrix kernel.  Otherwise queries that share a key head and are few
// (<= MAXR of them per session) go through diff_decode_kernel.  Keys are split over workgroups until the launch has about 4 (decode) or 2
// workgroups per CU, at least 2 (decode) or 4 chunks each.
Plan plan_of(int B, int H, int Hkv, int hd, int Lq, int Lk, bool train) {
  Plan p;
  const int rep = H / Hkv;
  p.decode = !train && (long long)rep * Lq <= MAXR;
  const long long wgs = p.decode ? (long long)B * Hkv : (long long)B * H * ((Lq + OWN - 1) / OWN);
  const int chunk = p.decode ? 4 * decode_keys(pad_hd(hd)) : CH;      // keys a workgroup takes at once
  const long long want = (long long)rt_num_cus() * (p.decode ? 4 : 2);
  long long s = wgs > 0 ? want / wgs : 1;
  const long long most = Lk / (p.decode ? 2 * chunk : 4 * chunk);
  if (s > most) s = most;
  if (s > 64) s = 64;
  p.n_split = s > 1 ? (int)s : 1;
  return p;
}
size_t part_floats(const Plan& p, long long Nq, int H, int hd) {
  return p.n_split > 1 ? (size_t)p.n_split * (size_t)Nq * H * 2 * (2 * (size_t)hd + 2) : 0;
}

int check(int B, int H, int Hkv, int hd, int Lq, int Lk, long long Nq, long long Nk, const void* cu_q, const void* cu_k) {
  if (B < 0 || H <= 0 || Hkv <= 0 || hd <= 0 || Lq < 0 || Lk < 0 || Nq < 0 || Nk < 0 || H % Hkv != 0) return RT_ERR_INVALID_ARG;
  if (hd > 64) return RT_ERR_UNSUPPORTED;
  if (cu_q == nullptr && Nq != (long long)B * Lq) return RT_ERR_INVALID_ARG;
  if (cu_k == nullptr && Nk != (long long)B * Lk) return RT_ERR_INVALID_ARG;
  return RT_OK;
}
bool grid_ok(long long blocks) { return blocks > 0 && blocks <= 0x7FFFFFFFLL; }

template <typename K>
int start(K kernel, dim3 grid, size_t lds, hipStream_t stream, const Args& a) {
  if (lds > 65536) RT_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  kernel<<<grid, NT, lds, stream>>>(a);
  RT_CHECK_LAUNCH();
  return RT_OK;
}
// mode: 0 the head fills its tile and rows are 16-byte aligned, 1 aligned, columns checked, 2 single columns, checked
#define RT_DIFF_START(KERNEL, HDP, MODE, ...)                                                                                        \
  ((HDP) == 32 ? ((MODE) == 0 ? start(KERNEL<32, 0>, __VA_ARGS__) : (MODE) == 1 ? start(KERNEL<32, 1>, __VA_ARGS__) : start(KERNEL<32, 2>, __VA_ARGS__)) \
               : ((MODE) == 0 ? start(KERNEL<64, 0>, __VA_ARGS__) : (MODE) == 1 ? start(KERNEL<64, 1>, __VA_ARGS__) : start(KERNEL<64, 2>, __VA_ARGS__)))

template <int R>
int start_decode(int HDP, int mode, dim3 grid, hipStream_t stream, const Args& a) {
  if (HDP == 32)
    return mode == 0 ? start(diff_decode_kernel<32, 0, R>, grid, 0, stream, a) : mode == 1 ? start(diff_decode_kernel<32, 1, R>, grid, 0, stream, a)
                                                                                           : start(diff_decode_kernel<32, 2, R>, grid, 0, stream, a);
  return mode == 0 ? start(diff_decode_kernel<64, 0, R>, grid, 0, stream, a) : mode == 1 ? start(diff_decode_kernel<64, 1, R>, grid, 0, stream, a)
                                                                                         : start(diff_decode_kernel<64, 2, R>, grid, 0, stream, a);
}

size_t img_bytes(int HDP) { return HDP == 32 ? 2 * Img<32>::BYTES + Img<64>::BYTES : 2 * Img<64>::BYTES + Img<128>::BYTES; }

}  // namespace

extern "C" {

size_t rt_diffattn_fwd_workspace_bytes(int32_t B, int32_t H, int32_t Hkv, int32_t hd, int32_t Lq, int32_t Lk, int64_t Nq, int32_t train) {
  if (B <= 0 || H <= 0 || Hkv <= 0 || hd <= 0 || hd > 64 || Lq <= 0 || Lk <= 0 || Nq <= 0 || H % Hkv != 0) return 0;
  return part_floats(plan_of(B, H, Hkv, hd, Lq, Lk, train != 0), Nq, H, hd) * sizeof(float);
}

int rt_diffattn_fwd(const float* q, int64_t ldq, const float* k, int64_t ldk, const float* v, int64_t ldv, const float* lam, const int64_t* cu_q,
                    const int64_t* cu_k, const int64_t* key_ids, int32_t B, int32_t H, int32_t Hkv, int32_t hd, int32_t Lq, int32_t Lk, int64_t Nq,
                    int64_t Nk, float scale, int32_t causal, const float* norm_w, float out_scale, float eps, float* y, int64_t ldy, float* o12,
                    float* lse, void* ws, size_t ws_bytes, hipStream_t stream) {
  const int rc = check(B, H, Hkv, hd, Lq, Lk, Nq, Nk, cu_q, cu_k);
  if (rc != RT_OK) return rc;
  if (Nq == 0) return RT_OK;
  const long long wq = 2LL * H * hd, wk = 2LL * Hkv * hd;
  if (q == nullptr || lam == nullptr || y == nullptr || ldq < wq || ldy < wq || (o12 == nullptr) != (lse == nullptr)) return RT_ERR_INVALID_ARG;
  if (Nk > 0 && (k == nullptr || v == nullptr || ldk < wk || ldv < wk)) return RT_ERR_INVALID_ARG;
  Args a{};
  a.q = q; a.k = k; a.v = v; a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.lam = lam;
  a.cu_q = (const long long*)cu_q; a.cu_k = (const long long*)cu_k; a.key_ids = (const long long*)key_ids;
  a.B = B; a.H = H; a.Hkv = Hkv; a.hd = hd; a.Lq = Lq; a.Lk = Lk; a.Nq = Nq; a.Nk = Nk;
  a.scale = scale > 0.f ? scale : 1.f / sqrtf((float)hd); a.causal = causal;
  a.norm_w = norm_w; a.out_scale = out_scale; a.eps = eps; a.y = y; a.ldy = ldy; a.o12 = o12; a.lse = lse;
  const Plan p = plan_of(B > 0 ? B : 1, H, Hkv, hd, Lq > 0 ? Lq : 1, Lk, o12 != nullptr);
  a.n_split = p.n_split;
  if (p.n_split > 1) {
    const size_t need = part_floats(p, Nq, H, hd) * sizeof(float);
    if (ws == nullptr || ws_bytes < need) return RT_ERR_WORKSPACE;
    a.part = (float*)ws;
    a.ml = a.part + (size_t)p.n_split * Nq * H * 2 * 2 * hd;
  }
  const int HDP = pad_hd(hd);
  const bool vec = hd % 4 == 0 && vec_ok(q, ldq) && vec_ok(k, ldk) && vec_ok(v, ldv) && vec_ok(y, ldy) && (o12 == nullptr || vec_ok(o12, 4)) &&
                   (ws == nullptr || vec_ok(ws, 4));
  const int mode = !vec ? 2 : (hd == HDP ? 0 : 1);
  const long long B1 = B + (cu_q != nullptr ? 1 : 0);
  if (p.decode) {
    if (!grid_ok(B1 * Hkv)) return RT_ERR_INVALID_ARG;
    const long long queries = (long long)(H / Hkv) * (Lq > 0 ? Lq : 1);
    const dim3 grid((unsigned)(B1 * Hkv), p.n_split);
    const int rc2 = queries <= 1 ? start_decode<1>(HDP, mode, grid, stream, a) : queries <= 2 ? start_decode<2>(HDP, mode, grid, stream, a)
                    : queries <= 4 ? start_decode<4>(HDP, mode, grid, stream, a) : start_decode<8>(HDP, mode, grid, stream, a);
    if (rc2 != RT_OK) return rc2;
  } else {
    a.n_tiles = (Lq + OWN - 1) / OWN > 0 ? (Lq + OWN - 1) / OWN : 1;
    if (!grid_ok(B1 * H * a.n_tiles)) return RT_ERR_INVALID_ARG;
    const int rc2 = RT_DIFF_START(diff_fwd_kernel, HDP, mode, dim3((unsigned)(B1 * H * a.n_tiles), p.n_split), img_bytes(HDP), stream, a);
    if (rc2 != RT_OK) return rc2;
  }
  if (p.n_split > 1) {
    if (!grid_ok(Nq * H)) return RT_ERR_INVALID_ARG;
    diff_combine_kernel<<<(unsigned)(Nq * H), NT, 0, stream>>>(a);
    RT_CHECK_LAUNCH();
  }
  return RT_OK;
}

size_t rt_diffattn_bwd_workspace_bytes(int32_t H, int32_t hd, int64_t Nq) {
  if (H <= 0 || hd <= 0 || Nq <= 0) return 0;
  return sizeof(float) * ((size_t)Nq * H * 2 * hd + (size_t)Nq * H * 2) + sizeof(double) * (size_t)PRE_WG * (H + 2 * hd) + 16;
}

int rt_diffattn_bwd(const float* q, int64_t ldq, const float* k, int64_t ldk, const float* v, int64_t ldv, const float* lam, const int64_t* cu_q,
                    const int64_t* cu_k, const int64_t* key_ids, int32_t B, int32_t H, int32_t Hkv, int32_t hd, int32_t Lq, int32_t Lk, int64_t Nq,
                    int64_t Nk, float scale, int32_t causal, const float* norm_w, float out_scale, float eps, const float* o12, const float* lse,
                    const float* dy, int64_t lddy, float* dq, int64_t lddq, float* dk, int64_t lddk, float* dv, int64_t lddv, float* dlam,
                    float* dw, void* ws, size_t ws_bytes, hipStream_t stream) {
  const int rc = check(B, H, Hkv, hd, Lq, Lk, Nq, Nk, cu_q, cu_k);
  if (rc != RT_OK) return rc;
  const long long wq = 2LL * H * hd, wk = 2LL * Hkv * hd;
  if (lam == nullptr || dlam == nullptr || (norm_w != nullptr) != (dw != nullptr)) return RT_ERR_INVALID_ARG;
  if (Nq > 0 && (q == nullptr || o12 == nullptr || lse == nullptr || dy == nullptr || dq == nullptr || ldq < wq || lddy < wq || lddq < wq)) return RT_ERR_INVALID_ARG;
  if (Nk > 0 && (k == nullptr || v == nullptr || dk == nullptr || dv == nullptr || ldk < wk || ldv < wk || lddk < wk || lddv < wk)) return RT_ERR_INVALID_ARG;
  if (ws == nullptr || ws_bytes < rt_diffattn_bwd_workspace_bytes(H, hd, Nq > 0 ? Nq : 1) || ((uintptr_t)ws & 15u) != 0) return RT_ERR_WORKSPACE;
  Args a{};
  a.q = q; a.k = k; a.v = v; a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.lam = lam;
  a.cu_q = (const long long*)cu_q; a.cu_k = (const long long*)cu_k; a.key_ids = (const long long*)key_ids;
  a.B = B; a.H = H; a.Hkv = Hkv; a.hd = hd; a.Lq = Lq; a.Lk = Lk; a.Nq = Nq; a.Nk = Nk;
  a.scale = scale > 0.f ? scale : 1.f / sqrtf((float)hd); a.causal = causal;
  a.norm_w = norm_w; a.out_scale = out_scale; a.eps = eps; a.o12 = const_cast<float*>(o12); a.lse = const_cast<float*>(lse);
  a.dq = dq; a.dk = dk; a.dv = dv; a.lddq = lddq; a.lddk = lddk; a.lddv = lddv;
  double* part = (double*)ws;
  float* dout = (float*)(part + (size_t)PRE_WG * (H + 2 * hd));
  dout = (float*)(((uintptr_t)dout + 15u) & ~(uintptr_t)15u);
  float* delta = dout + (size_t)Nq * H * 2 * hd;
  a.dout = dout; a.lddo = wq; a.delta = delta;
  hipStream_t s = stream;

  const int HDP = pad_hd(hd), groups = NT / (HDP / 2);
  long long n_pre = (Nq * H + groups - 1) / groups, least = (H + groups - 1) / groups;      // (one lane group per head at least)
  n_pre = n_pre > PRE_WG ? PRE_WG : n_pre;
  n_pre = n_pre < least ? least : n_pre;
  if (n_pre > PRE_WG) return RT_ERR_UNSUPPORTED;
  const bool pre_vec = hd % 2 == 0 && vec_ok(dy, lddy) && vec_ok(o12, 4) && (norm_w == nullptr || vec_ok(norm_w, 4));
  if (HDP == 32) {
    if (pre_vec) diff_bwd_pre_kernel<32, true><<<(unsigned)n_pre, NT, 0, s>>>(a, dy, lddy, dout, delta, part);
    else diff_bwd_pre_kernel<32, false><<<(unsigned)n_pre, NT, 0, s>>>(a, dy, lddy, dout, delta, part);
  } else {
    if (pre_vec) diff_bwd_pre_kernel<64, true><<<(unsigned)n_pre, NT, 0, s>>>(a, dy, lddy, dout, delta, part);
    else diff_bwd_pre_kernel<64, false><<<(unsigned)n_pre, NT, 0, s>>>(a, dy, lddy, dout, delta, part);
  }
  RT_CHECK_LAUNCH();
  diff_bwd_sums_kernel<<<H + 2 * hd, 64, 0, s>>>(part, (int)n_pre, H, 2 * hd, dlam, dw);
  RT_CHECK_LAUNCH();

  const bool vec = hd % 4 == 0 && vec_ok(q, ldq) && vec_ok(k, ldk) && vec_ok(v, ldv) && vec_ok(dq, lddq) && vec_ok(dk, lddk) && vec_ok(dv, lddv);
  const int mode = !vec ? 2 : (hd == HDP ? 0 : 1);
  const size_t img = img_bytes(HDP);
  if (Nq > 0) {
    const long long B1 = B + (cu_q != nullptr ? 1 : 0);
    a.n_tiles = Lq > 0 ? (Lq + OWN - 1) / OWN : 1;
    if (!grid_ok(B1 * H * a.n_tiles)) return RT_ERR_INVALID_ARG;
    const int rc2 = RT_DIFF_START(diff_bwd_dq_kernel, HDP, mode, dim3((unsigned)(B1 * H * a.n_tiles)), img + 4 * 4 * 64 * 16, s, a);
    if (rc2 != RT_OK) return rc2;
  }
  if (Nk > 0) {
    const long long B1 = B + (cu_k != nullptr ? 1 : 0);
    a.n_tiles = Lk > 0 ? (Lk + OWN - 1) / OWN : 1;
    if (!grid_ok(B1 * Hkv * a.n_tiles)) return RT_ERR_INVALID_ARG;
    const int rc2 = RT_DIFF_START(diff_bwd_dkv_kernel, HDP, mode, dim3((unsigned)(B1 * Hkv * a.n_tiles)), img + 4 * 8 * 64 * 16 + 512, s, a);
    if (rc2 != RT_OK) return rc2;
  }
  return RT_OK;
}

int rt_diff_lambda_fwd(const float* q1, const float* k1, const float* q2, const float* k2, float init, int32_t H, int32_t hd, float* lam, hipStream_t stream) {
  if (H < 0 || hd <= 0 || (H > 0 && (q1 == nullptr || k1 == nullptr || q2 == nullptr || k2 == nullptr || lam == nullptr))) return RT_ERR_INVALID_ARG;
  if (H == 0) return RT_OK;
  diff_lambda_fwd_kernel<<<H, 64, 0, stream>>>(q1, k1, q2, k2, init, hd, lam);
  RT_CHECK_LAUNCH();
  return RT_OK;
}

int rt_diff_lambda_bwd(const float* dlam, const float* q1, const float* k1, const float* q2, const float* k2, int32_t H, int32_t hd, float* dq1, float* dk1,
                       float* dq2, float* dk2, hipStream_t stream) {
  if (H < 0 || hd <= 0) return RT_ERR_INVALID_ARG;
  if (H == 0) return RT_OK;
  if (dlam == nullptr || q1 == nullptr || k1 == nullptr || q2 == nullptr || k2 == nullptr || dq1 == nullptr || dk1 == nullptr || dq2 == nullptr || dk2 == nullptr)
    return RT_ERR_INVALID_ARG;
  diff_lambda_bwd_kernel<<<H, 64, 0, stream>>>(dlam, q1, k1, q2, k2, hd, dq1, dk1, dq2, dk2);
  RT_CHECK_LAUNCH();
  return RT_OK;
}

}  // extern "C"
