// Differential attention: the difference of two softmax maps with a learned weight, normalised per head.
//
//   A_m = softmax(scale q_m k_m^T + mask),  m = 1, 2;   o = (A_1 - lam_h A_2) v;   y = out_scale * w * o / sqrt(mean(o^2) + eps)
//
// q rows carry [H][2][hd] columns (the two maps' queries of a head next to each other), k rows [Hkv][2][hd], v rows [Hkv][2 hd]; query head
// h reads key head h / (H / Hkv).  Sessions are packed rows (cu) or equal windows; inside a session the last query is aligned with the last
// key (causal: key j is seen by query i iff j <= i + nk - nq), so one launch serves whole sessions and the newest rows of stored ones.
// Keys whose item id is 0 are masked, whatever their rows hold.  A query that sees no key has o = 0, y = 0 and no gradients.
//
// Arithmetic: fp32 in, fp32 out.  A product runs on the fp16 matrix instruction as three terms of a two-way split: x = 2^e (h + l), e from the
// largest magnitude of the row, h = fp16(x 2^-e), l = fp16 of the rest; x y ~ h h' + h l' + l h'.  h and l hold 11 bits each and a sign, so x
// is held to 2^-23 of itself (values below 2^-17 of their row's largest: to 2^-38 of that) and the dropped l l' is below 2^-22 of the product: 8 u of a
// product (u = 2^-24) where fp32 takes u, and sums over many of them come out as near as those of fp32 tensors: over 150 drawn training calls the error
// against 64 bits is 0.85 x theirs (median; outputs, dq, dk, dv; 90 % below 1.25), with 85 % of the queries without a gradient, the others' at 1e-6, and half of
// the value rows zero 0.9 - 1.15 x (90 % below 1.55).  Where a result is what is left of a few products that cancel (a row whose maps nearly cancel; dlam of
// one head, p90 2.4 x) the 8 u show.  Weights are split with one unit per lane, not per row: their bits last because every row's planes have one
// size and rows of zeros the least exponent (row_exp).  Three bf16 planes, the exact split, take six terms: two sessions of 4,096 rows, 4 heads of hd 64,
// forward and backward 1,840 us with them, 1,100 with these.
// The split is made ONCE per call by diff_planes_kernel (one pass over q, k, v: memory bound), not at every staging: a 4,096-row session
// stages each of its rows 64 times.  Softmax statistics, sums and accumulators are fp32; scores live in the base-2 domain.
//
// Geometry: a workgroup is 4 waves = 2 row groups of 32 owner rows x the 2 maps; v_mfma_f32_32x32x16_f16 tiles, the OWNER row (a query;
// in the dK/dV pass a key) is the lane, the partner rows are the registers, so probabilities and dS feed the next product from the
// registers they were made in.  One wave per map rather than one wave for both: its operands and accumulators are half as many registers, which
// leaves two waves on a SIMD (one's softmax runs under the other's products).  Partner rows stream through LDS 32 at a time, copied as they
// lie by LDS DMA (global_load_lds: no registers, no address arithmetic): the planes are stored head-major with 48 bytes behind every row, so
// rows lie 3 sixteen-byte units apart modulo the 256 bytes of the banks: 32 rows of 16 bytes without a conflict, 4-row transpose blocks two-way (with 16
// bytes behind them: four-way, 192 conflict cycles per wave and chunk of the forward pass).
//
// What bounds it (two sessions of 4,096, 4 heads of hd 64, causal): forward 193 us, backward 466 us (on a card that has worked for 100 ms; 217 and 518 in
// the first passes behind a pause).  Least matrix work, three terms each, at the rate a large 16-bit matrix product reaches on this card (1,385 TFLOP/s): 112 and 260 us.  Counters: the matrix pipe is busy 36 - 38 % of the time, the vector
// pipe 43 % (exponentials, scales, splits), and the two waves of a SIMD overlap them little; two waves are what 256 registers each leave.
#include "rt_attn_planes.h"

namespace {
using rt_planes::LOG2E;
using rt_planes::s16x4;
using rt_planes::tr_read;

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef short s16x8v __attribute__((ext_vector_type(8)));

constexpr int NT = 256;
constexpr int OWN = 64;    // owner rows per workgroup
constexpr int CH = 32;     // partner rows per staged chunk
constexpr int PAD = 32;    // rows behind the last one that a chunk may copy (never used)

// Work of a matrix launch: owner tiles per session (longer sessions loop), (session, head) pairs as they are counted, order (work_of)
struct Grid { int n_tiles, bhs, blocks; };

struct Args {
  const float* q; const float* k; const float* v; long long ldq, ldk, ldv;
  const float* lam;                      // [H]
  const long long* cu_q; const long long* cu_k; const long long* key_ids;
  int B, H, Hkv, hd, Lq, Lk;
  long long Nq, Nk;
  float scale; int causal;
  const float* norm_w; float out_scale, eps;
  float* y; long long ldy;
  // planes: rows of [map 1: h | l][map 2: h | l] (q, k) or [h | l] (v, dO), 8 HD bytes + 48, head-major with N + PAD rows per head; scales 2^e
  unsigned char* qp; unsigned char* kp; unsigned char* vp; unsigned char* dp;
  float* qs; float* ks;                  // [H][2][Nq + PAD], [Hkv][2][Nk + PAD]
  float* vs; float* ivs; float* lvb;     // [Hkv][Nk + PAD]: 2^e, 2^-e, e (minus infinity: the key is masked)
  float* o12;                            // [Nq, H, 2, 2 hd] normalised outputs of the two maps (training)
  float* lse; float* lsf;                // [H][2][Nq + PAD] of the two maps (training): probability = exp2(s - lse) lsf, lse a whole number
  float* part; float* ml;                // split keys: [n_split, Nq, H, 2, 2 hd] and [n_split, Nq, H, 2, 2] (maximum, sum)
  int n_split, share;                    // share (diff_decode_kernel): TK-key tiles of a split at least; 0: sessions of one length
  Grid own_q, own_k;                     // launches whose owner rows are queries / keys
  // backward
  float* delta; float* dc;               // [H][2][Nq + PAD]: do . o_m 2^-e, e of dO's row; what turns exp2(s - lse) into the map's weight on dO's plane
  float* dq; float* dk; float* dv; long long lddq, lddk, lddv; int vec_q, vec_kv;
  int vec_y;
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

template <int CTRL> __device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ float lane_xor16(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, v), 0x401F)); }
template <int LANES> __device__ __forceinline__ float group_sum(float v) {      // 8, 16 or 32 neighbouring lanes
  v += dpp<0xB1>(v);       // lane ^ 1
  v += dpp<0x4E>(v);       // lane ^ 2
  v += dpp<0x141>(v);      // mirrored in 8 lanes
  if (LANES > 8) v += dpp<0x140>(v);      // mirrored in 16 lanes
  if (LANES > 16) v += lane_xor16(v);
  return v;
}
template <int CTRL> __device__ __forceinline__ double dpp_d(double v) {
  const long long b = __builtin_bit_cast(long long, v);
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)b, CTRL, 0xF, 0xF, true), hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, 0xF, 0xF, true);
  return __builtin_bit_cast(double, (unsigned long long)lo | (unsigned long long)hi << 32);
}
template <int LANES> __device__ __forceinline__ double group_sum(double v) {
  v += dpp_d<0xB1>(v);
  v += dpp_d<0x4E>(v);
  v += dpp_d<0x141>(v);
  if (LANES > 8) v += dpp_d<0x140>(v);
  if (LANES > 16) v += __shfl_xor(v, 16, 64);
  return v;
}
template <int LANES> __device__ __forceinline__ float group_max(float v) {
  v = fmaxf(v, dpp<0xB1>(v));
  v = fmaxf(v, dpp<0x4E>(v));
  v = fmaxf(v, dpp<0x141>(v));
  if (LANES > 8) v = fmaxf(v, dpp<0x140>(v));
  if (LANES > 16) v = fmaxf(v, lane_xor16(v));
  return v;
}
template <int MODE>      // 0 the row fills its columns, 1 aligned, 2 single columns
__device__ __forceinline__ f32x4 get4(const float* p, int c, int ncol) {
  f32x4 x{0.f, 0.f, 0.f, 0.f};
  if (MODE < 2) {
    if (MODE == 0 || c < ncol) x = *reinterpret_cast<const f32x4*>(p + c);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < ncol) x[e] = p[c + e];
  }
  return x;
}
__device__ __forceinline__ void put4(float* row, int c, int ncol, f32x4 x, bool vec) {
  if (vec) {
    if (c < ncol) *reinterpret_cast<f32x4*>(row + c) = x;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < ncol) row[c + j] = x[j];
  }
}

// ---- the planes --------------------------------------------------------------------------------------------------------------------------
template <int HD> struct Row {
  static constexpr int BYTES = 8 * HD + 48, CHUNK = CH * BYTES, UNITS = CHUNK / 16;      // UNITS of 16 bytes per chunk
};
// exponent of the row's scale: its largest magnitude comes to 2^13 .. 2^14 (2 x below the fp16 range; what is 2^-18 of it keeps all 22 bits)
// `least`: values below 2^(least + 14) lose bits.  -126 keeps 2^e a normal number; v takes -80, so that a row sum of weights that carry 2^-e
// stays finite over any number of keys.
// `zero`: of a row of zeros.  It adds nothing to a product, but its weights, which carry its 2^e, stand beside the other rows' where those are split into
// halves with one unit: with exponent 0 they drove the bits of rows of ordinary size out of the fp16 range (dV beside queries without a gradient, |dO| = 1e-6:
// 3 % off; outputs beside one zero value row, |v| = 1e-6: 1 %).  q, k and dO take the least there is.  A zero value row's weight is counted in the row sum
// through s + e - m, rounded at its size: -40 keeps that at 7e-7 of it beside values of size one (-80: 3e-6) and all bits of values down to 1e-12.
constexpr int LEAST = -126, LEAST_V = -80, ZERO_V = -40;
__device__ __forceinline__ int row_exp(float top, int least, int zero) {
  if (top == 0.f) return zero;
  if (!(top <= 3.0e38f)) return 0;      // infinities and NaN stay what they are
  const int e = __builtin_amdgcn_frexp_expf(top) - 14;
  return e < least ? least : e;
}
__device__ __forceinline__ float pow2(int e) { return __builtin_amdgcn_ldexpf(1.f, e); }
// four columns of a row, scaled by 2^-e: h plane at p, l plane `plane` bytes behind
__device__ __forceinline__ void put_planes(unsigned char* p, int plane, f32x4 x, int e) {
  h4 h, l;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float t = __builtin_amdgcn_ldexpf(x[k], -e);
    h[k] = (_Float16)t;
    l[k] = (_Float16)(t - (float)h[k]);
  }
  *reinterpret_cast<h4*>(p) = h;
  *reinterpret_cast<h4*>(p + plane) = l;
}
__device__ __forceinline__ float top4(f32x4 x) { return fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))); }

// q, k and v -> planes and scales: HD / 2 lanes per (row, head), four columns each; blocks [0, q_blocks) q, then k, then v.  Memory bound: 8,192 rows of 4
// heads of hd 64, 50 MB in and 55 MB out, 19.5 us = 5.4 TB/s; 14,381 rows of 4 heads of hd 32 19 us = 5.1 TB/s.
template <int HD, int MODE>
__global__ __launch_bounds__(NT) void diff_planes_kernel(Args a, unsigned q_blocks, unsigned kv_blocks) {
  constexpr int LANES = HD / 2, GROUPS = NT / LANES;
  const int tid = threadIdx.x, c4 = tid % LANES, hd = a.hd;
  const int what = blockIdx.x < q_blocks ? 0 : (blockIdx.x < q_blocks + kv_blocks ? 1 : 2);
  const long long block = what == 0 ? blockIdx.x : (what == 1 ? blockIdx.x - q_blocks : blockIdx.x - q_blocks - kv_blocks);
  const int heads = what == 0 ? a.H : a.Hkv;
  const long long N = what == 0 ? a.Nq : a.Nk, at = block * GROUPS + tid / LANES, row = at / heads;
  const int h = (int)(at % heads);
  if (row >= N) return;      // (whole lane groups)
  const bool live = what == 0 || a.key_ids == nullptr || a.key_ids[row] != 0;
  const long long slot = h * (N + PAD) + row;
  if (what == 2) {
    const f32x4 x = live ? get4<MODE>(a.v + row * a.ldv + (long long)h * 2 * hd, 4 * c4, 2 * hd) : f32x4{0.f, 0.f, 0.f, 0.f};
    const int e = row_exp(group_max<LANES>(top4(x)), LEAST_V, ZERO_V);
    put_planes(a.vp + slot * Row<HD>::BYTES + 8 * c4, 4 * HD, x, e);
    if (c4 == 0) {
      a.vs[slot] = pow2(e);
      a.ivs[slot] = pow2(-e);
      a.lvb[slot] = live ? (float)e : -INFINITY;
    }
    return;
  }
  const int mp = c4 / (HD / 4), col = (c4 % (HD / 4)) * 4;
  const float* src = what == 0 ? a.q + row * a.ldq + (long long)(2 * h + mp) * hd : a.k + row * a.ldk + (long long)(2 * h + mp) * hd;
  const f32x4 x = live ? get4<MODE>(src, col, hd) : f32x4{0.f, 0.f, 0.f, 0.f};
  const int e = row_exp(group_max<LANES / 2>(top4(x)), LEAST, LEAST);
  put_planes((what == 0 ? a.qp : a.kp) + slot * Row<HD>::BYTES + mp * 4 * HD + 2 * col, 2 * HD, x, e);
  if (c4 % (HD / 4) == 0) (what == 0 ? a.qs : a.ks)[(2 * h + mp) * (N + PAD) + row] = pow2(e);
}

__device__ __forceinline__ int wave_of(int tid) { return __builtin_amdgcn_readfirstlane(tid >> 6); }      // known to be the same in all lanes: scalar branches

// ---- staging -----------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned lds_addr(const void* p) { return (unsigned)(unsigned long long)(RT_LDS const void*)p; }
__device__ __forceinline__ void dma16(const void* src, unsigned dst) {      // lane i: 16 bytes to dst + 16 i
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0" : "=&s"(keep) : "v"(src), "s"(dst) : "memory");
}
__device__ __forceinline__ void dma4(const void* src, unsigned dst) {       // lane i: 4 bytes to dst + 4 i
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, off\n\ts_mov_b32 m0, %0" : "=&s"(keep) : "v"(src), "s"(dst) : "memory");
}
__device__ __forceinline__ void dma_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void barrier() {      // LDS writes of this wave are visible behind it; LDS DMA is waited for by dma_done
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
template <int HD> __device__ __forceinline__ void copy_chunk(const unsigned char* src, unsigned dst, int tid) {
  const unsigned wave0 = __builtin_amdgcn_readfirstlane(tid & ~63);
#pragma unroll
  for (int i = 0; i < (Row<HD>::UNITS + NT - 1) / NT; ++i)
    if (tid + i * NT < Row<HD>::UNITS) dma16(src + (size_t)(tid + i * NT) * 16, dst + (wave0 + i * NT) * 16);
}
// rows [left, CH) of two staged images: zeros (they belong to the next session, or to nobody)
template <int HD> __device__ __forceinline__ void clear_rows(unsigned char* img, int left, int tid) {
  constexpr int U = Row<HD>::BYTES / 16;
  for (int u = left * U + tid; u < CH * U; u += NT) {
    *reinterpret_cast<f32x4*>(img + u * 16) = f32x4{0.f, 0.f, 0.f, 0.f};
    *reinterpret_cast<f32x4*>(img + Row<HD>::CHUNK + u * 16) = f32x4{0.f, 0.f, 0.f, 0.f};
  }
}

// ---- products ----------------------------------------------------------------------------------------------------------------------------
struct P2 { h8 h, l; };
__device__ __forceinline__ f32x16 mfma3(const P2& A, const P2& B, f32x16 acc) {      // smallest terms first
  acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(A.l, B.h, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(A.h, B.l, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(A.h, B.h, acc, 0, 0, 0);
  return acc;
}
__device__ __forceinline__ int reg_row(int r, int g) { return 8 * (r >> 2) + 4 * g + (r & 3); }
__device__ __forceinline__ f32x16 zero16() { f32x16 z; for (int r = 0; r < 16; ++r) z[r] = 0.f; return z; }

// columns c0 + 16 s + 8 g .. + 7 of one stored row (l plane `plane` bytes behind h)
template <int NS> __device__ __forceinline__ void load_own(const unsigned char* row, int c0, int plane, int g, P2 (&out)[NS]) {
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    out[s].h = *reinterpret_cast<const h8*>(row + (c0 + 16 * s + 8 * g) * 2);
    out[s].l = *reinterpret_cast<const h8*>(row + (c0 + 16 * s + 8 * g) * 2 + plane);
  }
}
// acc[r] = sum_c img[row(r)][c0 + c] * own[c], row(r) = 8 (r / 4) + 4 g + r % 4: the partner rows are the registers, the owner the lane
// All fragments are read in front of the products (the compiler reads each in front of the instruction that needs it: an LDS latency per step).
template <int HD, int NS>
__device__ __forceinline__ void rows_dot(const unsigned char* img, int c0, int plane, const P2 (&own)[NS], int i, int g, f32x16& out) {
  const unsigned char* p = img + i * Row<HD>::BYTES + c0 * 2 + 16 * g;
  P2 A[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    A[s].h = *reinterpret_cast<const h8*>(p + 32 * s);
    A[s].l = *reinterpret_cast<const h8*>(p + 32 * s + plane);
  }
  f32x16 acc = zero16();      // (the first product's constant operand)
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int s = 0; s < NS; ++s) acc = mfma3(A[s], own[s], acc);
  __builtin_amdgcn_s_setprio(0);
  out = acc;
}
// acc[cb][r] += sum over the 32 partner rows of img[row][c0 + 32 cb + col(r)] * w[row], the lane's weights in the accumulator order of rows_dot
// (slot j of step t = register 8 t + j = row 16 t + 8 (j / 4) + 4 g + j % 4): the partner rows are the reduction index, read transposed
// The next fragment is read under the products of the one before.
template <int HD, int NB>
__device__ __forceinline__ void cols_dot(const unsigned char* img, int c0, int plane, const P2 (&w)[2], int lane, f32x16 (&acc)[NB]) {
  const int g = lane >> 5;
  const unsigned char* p = img + (4 * g + ((lane & 15) >> 2)) * Row<HD>::BYTES + (c0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2;
  auto read = [&](int n) {
    const unsigned char* a = p + 16 * (n / NB) * Row<HD>::BYTES + 64 * (n % NB);
    const unsigned char* b = a + 8 * Row<HD>::BYTES;
    P2 A;
    A.h = __builtin_bit_cast(h8, (s16x8v)__builtin_shufflevector(tr_read(a), tr_read(b), 0, 1, 2, 3, 4, 5, 6, 7));
    A.l = __builtin_bit_cast(h8, (s16x8v)__builtin_shufflevector(tr_read(a + plane), tr_read(b + plane), 0, 1, 2, 3, 4, 5, 6, 7));
    return A;
  };
  constexpr int AHEAD = 2;
  P2 A[AHEAD + 1];
#pragma unroll
  for (int n = 0; n < AHEAD; ++n) A[n] = read(n);
  __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int n = 0; n < 2 * NB; ++n) {
    if (n + AHEAD < 2 * NB) A[(n + AHEAD) % (AHEAD + 1)] = read(n + AHEAD);
    __builtin_amdgcn_sched_barrier(0);
    acc[n % NB] = mfma3(A[n % (AHEAD + 1)], w[n / NB], acc[n % NB]);
  }
  __builtin_amdgcn_s_setprio(0);
}
// x factor as two halves; h and the rest of it leave one mixed-precision multiply-add each
__device__ __forceinline__ void split16(const float (&x)[16], float factor, P2 (&out)[2]) {
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float v = x[8 * t + j];
      out[t].h[j] = (_Float16)fmaf(v, factor, 0.f);
      out[t].l[j] = (_Float16)fmaf(v, factor, -(float)out[t].h[j]);
    }
}
// The same for weights of unknown size (dS; the difference map times dO's scales): the lane's unit follows the largest magnitude it has met, as
// the running maximum of a softmax does; when it grows, the lane's accumulators are rescaled (powers of two: exact).  That keeps the result's bits if a
// large weight meets a row of large plane values: every row's planes are scaled to one size, and a zero row's weight is the least there is (row_exp).
template <int NB>
__device__ __forceinline__ void split16_scaled(const float (&x)[16], float& inv, f32x16 (&acc)[NB], P2 (&out)[2]) {
  float top = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(x[r]));
  top = fmaxf(top, __shfl_xor(top, 32, 64));
  const bool grows = top * inv > 32768.f;
  if (__any(grows)) {
    const int e = __builtin_amdgcn_frexp_expf(top);      // top < 2^e: it comes to 2^12 .. 2^13
    const float now = grows ? pow2(min(13 - e, 126)) : inv, ratio = now / inv;
#pragma unroll
    for (int cb = 0; cb < NB; ++cb) acc[cb] *= ratio;
    inv = now;
  }
  split16(x, inv, out);
}
constexpr float NO_UNIT = 0x1p126f;      // before the first weight

// The backward pass recomputes a probability as exp2(s - n) f: n the nearest whole number to the row's log2-sum-exp2, f in 0.7 .. 1.5 the rest.  The log
// itself, 10 to 30 in magnitude, would be rounded to 2^-20 and make every probability of the row wrong by that (it did: dq, dk, dv were off by
// 7e-7 in one direction).  base: what was taken from the scores; total: the sum of exp2(s - base).
__device__ __forceinline__ void row_norm(float base, float total, float& n, float& f) {
  if (!(total > 0.f)) { n = 0.f; f = total; return; }      // an empty row: every probability 0 (a NaN sum stays one)
  const float whole = floorf(base);
  n = rintf(base + __builtin_amdgcn_logf(total));
  f = __builtin_amdgcn_ldexpf(__builtin_amdgcn_exp2f(whole - base) / total, (int)(n - whole));
}

// blockIdx -> (owner tile, session, head, split): the tiles of the real sessions, then (b == B) the rows behind the last one.
// Heavy tiles first (causal: a session's last queries, its first keys): where the launch is many times the machine, the light ones fill the gaps
// at its end.
// Workgroups go to the eight dies in turn and each die has its own 4 MB of L2: with the (session, head) pairs counted in a multiple of eight (`bhs`:
// rounded up where there are many), all tiles of a pair, which stream the same chunks, meet on one die (forward, 33 sessions of 1,000, 3 heads of hd 64: 384 ->
// 365 us; 7 of 2,000, 11 heads: 974 -> 911).
struct Work { int tile, b, h, split; bool any; };
__device__ __forceinline__ Work work_of(const Args& a, const Grid& n, int blk, int H, bool last_first) {
  const int real = n.bhs * n.n_tiles, bh = blk % n.bhs, o = blk / n.bhs;
  Work w;
  w.split = blockIdx.y;
  if (blk >= real) {
    w.b = a.B;
    w.h = (blk - real) % H;
    w.tile = (blk - real) / H;
    w.any = true;
    return w;
  }
  w.tile = last_first ? n.n_tiles - 1 - o : o;
  w.b = bh / H;
  w.h = bh % H;
  w.any = bh < a.B * H;
  return w;
}
// A value that the optimiser takes for new at this point: comparisons with it stay here, instead of being made once per column in front of the
// loops and kept in hundreds of spilled scalar registers.
__device__ __forceinline__ int fresh(int x) {
  asm volatile("" : "+s"(x));
  return x;
}

// ---- forward ----------------------------------------------------------------------------------------------------------------------------
// Values carry their row's scale 2^e: the running maximum is that of s + e, so the weights exp2(s + e - m) stay below one whatever the scales
// are, and the row sum takes them back by 2^-e.  m is a whole number, taken up only when a logit passes it (by the next whole number above it): e - m is
// exact then and the weight's argument has one rounding, at its own size — s + e, 10 and more in magnitude, would carry 5e-7 into every
// weight (outputs were off by 3.2e-7 for it, where the plain form is by 1.5e-7).
template <int HD> constexpr int fwd_stage() { return 2 * Row<HD>::CHUNK + 512; }      // K | V | key scales of the maps | e, 2^-e

template <int HD, int KH>
__global__ __launch_bounds__(KH * NT, HD == 32 && KH == 1 ? 3 : 2) void diff_fwd_kernel(Args a) {
  constexpr int DV = 2 * HD, NS = HD / 16, NB = DV / 32, STAGE = KH * fwd_stage<HD>();
  constexpr float UP = 0x1p14f;      // weights of at most 1 come to the fp16 planes as 2^14
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x % NT, kh = KH == 1 ? 0 : wave_of(threadIdx.x) / 4, lane = tid & 63, wave = wave_of(tid), mp = wave & 1, rg = wave >> 1, i = lane & 31, g = lane >> 5;
  const Work wk = work_of(a, a.own_q, blockIdx.x, a.H, a.causal != 0);
  if (!wk.any) return;
  const int h = wk.h, hk = h / (a.H / a.Hkv), dv = 2 * a.hd;
  const long long NqP = a.Nq + PAD, NkP = a.Nk + PAD;

  if (wk.b == a.B) {      // rows behind the last session: zeros
    if (wk.split != 0) return;
    const long long r0 = rows_used(a.cu_q, a.B, a.Nq);
    for (long long r = r0 + wk.tile; r < a.Nq && kh == 0; r += a.own_q.n_tiles) {
      for (int c = tid; c < dv; c += NT) a.y[r * a.ldy + (long long)h * dv + c] = 0.f;
      if (a.o12 != nullptr) for (int c = tid; c < 2 * dv; c += NT) a.o12[(r * a.H + h) * 2 * dv + c] = 0.f;
    }
    return;
  }
  long long qr0, kr0; int nq, nk;
  rows_of(a.cu_q, wk.b, a.Lq, a.Nq, qr0, nq);
  rows_of(a.cu_k, wk.b, a.Lk, a.Nk, kr0, nk);
  const int off = nk - nq;
  const float lam = a.lam[h];
  const unsigned lds0 = lds_addr(smem) + kh * fwd_stage<HD>();
  const long long krow = hk * NkP + kr0;
  auto issue = [&](int c, int st) {
    const unsigned dst = lds0 + st * STAGE;
    const long long r = krow + c * CH;
    copy_chunk<HD>(a.kp + r * Row<HD>::BYTES, dst, tid);
    copy_chunk<HD>(a.vp + r * Row<HD>::BYTES, dst + Row<HD>::CHUNK, tid);
    const long long at = kr0 + c * CH + i;
    if (wave == 0) dma4(a.ks + (2 * hk + g) * NkP + at, dst + 2 * Row<HD>::CHUNK);
    if (wave == 1) dma4((g == 0 ? a.lvb : a.ivs) + hk * NkP + at, dst + 2 * Row<HD>::CHUNK + 256);
  };

  for (int tile = wk.tile; tile * OWN < nq; tile += a.own_q.n_tiles) {
    const int q0 = tile * OWN + 32 * rg, qi = q0 + i;
    const bool qok = qi < nq;
    const long long qrow = qr0 + min(qi, nq - 1);
    P2 Qp[NS];
    load_own<NS>(a.qp + (h * NqP + qrow) * Row<HD>::BYTES + mp * 4 * HD, 0, 2 * HD, g, Qp);
    const float qsc = a.qs[(2 * h + mp) * NqP + qrow] * (a.scale * LOG2E);
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
    barrier();      // (the previous tile's readers are done)
    if (c_lo + kh < c_hi) issue(c_lo + kh, 0);
    int st = 0;
    for (int c0 = c_lo; c0 < c_hi; c0 += KH, st ^= 1) {
      const int c = c0 + kh;
      const int t0 = c * CH, left = nk - t0;
      unsigned char* img = smem + st * STAGE + kh * fwd_stage<HD>();
      float* sc = reinterpret_cast<float*>(img + 2 * Row<HD>::CHUNK);
      dma_done();
      barrier();                                    // chunk c is here, chunk c - 1 has been read
      if (c + KH < c_hi) issue(c + KH, st ^ 1);
      if (nk - (c0 + KH - 1) * CH < CH) {      // (the same in all waves)
        if (left < CH && c < c_hi) {
          clear_rows<HD>(img, left, tid);
          if (tid < 128 && (tid & 31) >= left) sc[tid] = 0.f;
        }
        barrier();
      }
      if (c >= c_hi || q0 >= nq || (a.causal && t0 > q0 + 31 + off)) continue;      // (wave-uniform) nothing of the chunk is visible to the row group
      f32x16 S;
      rows_dot<HD, NS>(img + mp * 4 * HD, 0, 2 * HD, Qp, i, g, S);
      float x[16];
      const bool edge = left < CH || (a.causal && t0 + 31 > q0 + off);
      const int last = a.causal ? min(qi + off - t0, left - 1) : left - 1;
      auto logits = [&](float from) {      // s + e - from, one rounding: e and `from` are whole numbers
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const f32x4 k4 = *reinterpret_cast<const f32x4*>(sc + 32 * mp + 8 * r + 4 * g), e4 = *reinterpret_cast<const f32x4*>(sc + 64 + 8 * r + 4 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[4 * r + e] = fmaf(S[4 * r + e] * k4[e], qsc, e4[e] - from);
        }
        if (edge) {
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] = reg_row(r, g) <= last ? x[r] : -INFINITY;
        }
      };
      const float was = m == -INFINITY ? 0.f : m;      // a row that has seen no key yet
      logits(was);
      float top = x[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) top = fmaxf(top, x[r]);
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const bool grows = top > 0.f || (m == -INFINITY && top > -INFINITY);
      if (__any(grows)) {
        const float now = grows ? was + ceilf(top) : was, alpha = __builtin_amdgcn_exp2f(m - now);
        m = grows ? now : m;
        lsum *= alpha;
#pragma unroll
        for (int cb = 0; cb < NB; ++cb) O[cb] *= alpha;
        logits(now);
      }
      float ps = 0.f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x4 i4 = *reinterpret_cast<const f32x4*>(sc + 96 + 8 * r + 4 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[4 * r + e] = __builtin_amdgcn_exp2f(x[4 * r + e]);
          ps = fmaf(x[4 * r + e], i4[e], ps);
        }
      }
      lsum += ps;
      P2 Pp[2];
      float up = UP;      // (opaque: or the multiply-adds become conversions and differences, four instructions for two)
      asm("" : "+s"(up));
      split16(x, up, Pp);
      cols_dot<HD, NB>(img + Row<HD>::CHUNK, 0, 4 * HD, Pp, lane, O);
    }
    float l = lsum + __shfl_xor(lsum, 32, 64);
    if (KH == 2) {      // the second half's maximum, sum and outputs join the first's
      f32x4* xh = reinterpret_cast<f32x4*>(smem) + wave * (NB * 4 + 1) * 64;
      barrier();
      if (kh == 1) {
#pragma unroll
        for (int cb = 0; cb < NB; ++cb)
#pragma unroll
          for (int r = 0; r < 4; ++r) xh[(cb * 4 + r) * 64 + lane] = f32x4{O[cb][4 * r], O[cb][4 * r + 1], O[cb][4 * r + 2], O[cb][4 * r + 3]};
        xh[NB * 4 * 64 + lane] = f32x4{m, l, 0.f, 0.f};
      }
      barrier();
      if (kh == 0) {
        const f32x4 ml = xh[NB * 4 * 64 + lane];
        const float mx = fmaxf(m, ml[0]), base = mx == -INFINITY ? 0.f : mx, e0 = __builtin_amdgcn_exp2f(m - base), e1 = __builtin_amdgcn_exp2f(ml[0] - base);
        m = mx;
        l = l * e0 + ml[1] * e1;
#pragma unroll
        for (int cb = 0; cb < NB; ++cb)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const f32x4 o = xh[(cb * 4 + r) * 64 + lane];
#pragma unroll
            for (int e = 0; e < 4; ++e) O[cb][4 * r + e] = fmaf(o[e], e1, O[cb][4 * r + e] * e0);
          }
      }
    }
    if (a.n_split > 1) {      // partial sums as they are; diff_combine_kernel joins the splits
      if (kh == 0 && qok) {
        const int n = fresh(dv);
        const long long at = (((long long)wk.split * a.Nq + qr0 + qi) * a.H + h) * 2 + mp;
        if (g == 0) { a.ml[2 * at] = m; a.ml[2 * at + 1] = l; }
        float* o = a.part + at * dv;
#pragma unroll
        for (int cb = 0; cb < NB; ++cb)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            put4(o, 32 * cb + 8 * r + 4 * g, n, f32x4{O[cb][4 * r], O[cb][4 * r + 1], O[cb][4 * r + 2], O[cb][4 * r + 3]} * 0x1p-14f, (n & 3) == 0);
      }
      continue;
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);      // (a NaN sum stays one)
#pragma unroll
    for (int cb = 0; cb < NB; ++cb) O[cb] *= inv * (1.f / UP);
    if (kh == 0 && qok && a.lse != nullptr && g == 0) row_norm(m, l, a.lse[(2 * h + mp) * NqP + qr0 + qi], a.lsf[(2 * h + mp) * NqP + qr0 + qi]);
    if (kh == 0 && qok && a.o12 != nullptr) {
      const int n = fresh(dv);
      float* o = a.o12 + (((qr0 + qi) * a.H + h) * 2 + mp) * (long long)n;
#pragma unroll
      for (int cb = 0; cb < NB; ++cb)
#pragma unroll
        for (int r = 0; r < 4; ++r) put4(o, 32 * cb + 8 * r + 4 * g, n, f32x4{O[cb][4 * r], O[cb][4 * r + 1], O[cb][4 * r + 2], O[cb][4 * r + 3]}, (n & 3) == 0);
    }
    // the second map's wave hands its output over; the first one's subtracts, normalises and writes
    barrier();
    f32x4* xo = reinterpret_cast<f32x4*>(smem) + rg * (NB * 4 * 64);
    if (kh == 0 && mp == 1) {
#pragma unroll
      for (int cb = 0; cb < NB; ++cb)
#pragma unroll
        for (int r = 0; r < 4; ++r) xo[(cb * 4 + r) * 64 + lane] = f32x4{O[cb][4 * r], O[cb][4 * r + 1], O[cb][4 * r + 2], O[cb][4 * r + 3]};
    }
    barrier();
    if (kh == 0 && mp == 0) {
      float ss = 0.f;
#pragma unroll
      for (int cb = 0; cb < NB; ++cb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const f32x4 o2 = xo[(cb * 4 + r) * 64 + lane];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            O[cb][4 * r + e] -= lam * o2[e];
            ss += O[cb][4 * r + e] * O[cb][4 * r + e];
          }
        }
      ss += __shfl_xor(ss, 32, 64);
      const float f = a.norm_w != nullptr ? a.out_scale / sqrtf(ss / (float)dv + a.eps) : a.out_scale;
      if (qok) {
        const int n = fresh(dv), vec = fresh(a.vec_y);
        float* o = a.y + (qr0 + qi) * a.ldy + (long long)h * n;
#pragma unroll
        for (int cb = 0; cb < NB; ++cb)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int col = 32 * cb + 8 * r + 4 * g;
            f32x4 t;
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = O[cb][4 * r + e] * f * ((a.norm_w != nullptr && col + e < n) ? a.norm_w[col + e] : 1.f);
            put4(o, col, n, t, vec != 0);
          }
      }
    }
  }
}

// join of the key splits: one workgroup per (row, head); a lane holds the statistics of a split (n_split <= 64), then a thread sums one value
// column over its share of the splits.  8 rows of 8 heads, 32 splits: 8 us, two dependent reads of memory
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
    if (a.lse != nullptr && lane == 0) row_norm(mx, total, a.lse[(2 * h + wave) * (a.Nq + PAD) + row], a.lsf[(2 * h + wave) * (a.Nq + PAD) + row]);
  }
  const int slots = NT / dv, c = tid % dv, sub = tid / dv;
  for (int mp = 0; mp < 2; ++mp) {
    __syncthreads();
    float x = 0.f;
    if (sub < slots)
      for (int s0 = sub; s0 < a.n_split; s0 += 8 * slots) {      // eight loads in flight
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int s = s0 + k * slots;
          v[k] = s < a.n_split ? a.part[(((long long)s * plane + at) * 2 + mp) * dv + c] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float w = wgt[mp][min(s0 + k * slots, 63)];
          if (a.share > 0) v[k] = w != 0.f ? v[k] : 0.f;      // (an empty share's sums were not written)
          x = fmaf(v[k], w, x);
        }
      }
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

// ---- backward, in front: gradient of o (as planes), delta_m = do . o_m, and the sums behind dlam and dw --------------------------------------
// HD / 2 lanes per (row, head), four columns each; a lane group keeps its head, so dlam and dw stay in registers over all of its rows.  They
// are summed in 64 bits, per workgroup, in a fixed order.  do stands at right angles to o (but for eps) and do . o_m is what is left of that: formed in
// 64 bits, from the outputs as they are (in 32 the gradient of lam was 2 - 5 x further off; 15.5 -> 17 us).  Memory bound: 8,192 rows of 4 heads of hd 64,
// 70 MB, 17 us = 4.1 TB/s.
//
// A row that sees ONE key has that key's values for both maps' outputs, whatever the logits are: dO stands at right angles to them but for eps, and the
// row's share of dlam, 1e-5 of its terms, would be the two outputs' own roundings (sessions of one row: 0.3 to 3 % off).  o_2 is o_1 there.  Which rows
// those are is looked up where the saved outputs nearly agree (128 packed sessions of up to 200, 4 heads of hd 32: 16.5 -> 18.9 us; two of 4,096: 17.0 -> 17.6).
constexpr int PRE_WG = 1024;      // workgroups at most: the partials are [PRE_WG][H + 2 hd] doubles

// whether query row `row` sees one key: its session by bisection, its keys by the lane group, which stops at the second one
template <int LANES>
__device__ __forceinline__ bool sees_one_key(const Args& a, long long row, int lane) {
  int b = 0;
  if (a.cu_q != nullptr) {
    for (int e = a.B; e - b > 1;) {
      const int mid = b + (e - b) / 2;
      if (a.cu_q[mid] <= row) b = mid;
      else e = mid;
    }
  } else {
    b = (int)(row / a.Lq);
  }
  long long qr0, kr0; int nq, nk;
  rows_of(a.cu_q, b, a.Lq, a.Nq, qr0, nq);
  rows_of(a.cu_k, b, a.Lk, a.Nk, kr0, nk);
  const long long at = row - qr0;
  if (at < 0 || at >= nq) return false;
  const int end = a.causal ? min(nk, (int)at + nk - nq + 1) : nk;
  if (a.key_ids == nullptr) return end == 1;
  float seen = 0.f;
  for (int j0 = 0; j0 < end && seen < 2.f; j0 += LANES)
    seen += group_sum<LANES>(j0 + lane < end && a.key_ids[kr0 + j0 + lane] != 0 ? 1.f : 0.f);
  return seen == 1.f;
}

template <int HD, int MODE>
__global__ __launch_bounds__(NT) void diff_bwd_pre_kernel(Args a, const float* dy, long long lddy, double* part) {
  constexpr int LANES = HD / 2, GROUPS = NT / LANES;
  __shared__ double sw[GROUPS][2 * HD], sl[GROUPS];
  const int tid = threadIdx.x, gid = tid / LANES, c = (tid % LANES) * 4, dv = 2 * a.hd, H = a.H;
  const long long used = rows_used(a.cu_q, a.B, a.Nq), NqP = a.Nq + PAD;
  const long long gg = (long long)blockIdx.x * GROUPS + gid, n_groups = (long long)gridDim.x * GROUPS;
  const int h = (int)(gg % H);
  const long long step = n_groups / H;                       // rows are dealt to the `step` lane groups of a head; leftover groups do nothing
  const float lam = a.lam[h], inv = 1.f / (float)dv;
  const f32x4 w = a.norm_w != nullptr ? get4<MODE>(a.norm_w, c, dv) * a.out_scale : f32x4{a.out_scale, a.out_scale, a.out_scale, a.out_scale};
  double dw[4] = {0.0, 0.0, 0.0, 0.0}, dl = 0.0;
  for (long long row = gg < step * H ? gg / H : used; row < used; row += step) {
    const long long at = row * H + h;
    const f32x4 o1 = get4<MODE>(a.o12 + at * 2 * dv, c, dv);
    f32x4 o2 = get4<MODE>(a.o12 + (at * 2 + 1) * dv, c, dv);
    const f32x4 g = get4<MODE>(dy + row * lddy + (long long)h * dv, c, dv), e = g * w;
    double t[4] = {e[0], e[1], e[2], e[3]};
    if (a.norm_w != nullptr) {
      // (outputs of one key's values: each off by 2 u for the values' halves, 8 u for the product, 4 u for the row sum's reciprocal and the products with it, u = 2^-24)
      const float top = group_max<LANES>(top4(o1)), apart = group_max<LANES>(top4(o1 - o2));
      const bool near = apart <= 0x1p-19f * top;
      if (__builtin_expect(__any(near), 0)) {
        if (near && apart > 0.f && sees_one_key<LANES>(a, row, c / 4)) o2 = o1;
      }
      double x[4], xx = 0.0, ex = 0.0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[k] = (double)o1[k] - (double)lam * (double)o2[k];
        xx += x[k] * x[k];
        ex += t[k] * x[k];
      }
      xx = group_sum<LANES>(xx) + (double)dv * (double)a.eps;
      const float r = 1.f / sqrtf((float)xx * inv);
      const double part_x = group_sum<LANES>(ex) / xx;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        t[k] = (double)r * (t[k] - part_x * x[k]);
        dw[k] += (double)(a.out_scale * g[k] * r) * x[k];
      }
    }
    f32x4 d;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (MODE != 0) t[k] = c + k < dv ? t[k] : 0.0;
      d[k] = (float)t[k];
    }
    const int ex = row_exp(group_max<LANES>(top4(d)), LEAST, LEAST);
    put_planes(a.dp + (h * NqP + row) * Row<HD>::BYTES + 2 * c, 4 * HD, d, ex);
    const double s1 = group_sum<LANES>(t[0] * o1[0] + t[1] * o1[1] + t[2] * o1[2] + t[3] * o1[3]);
    const double s2 = group_sum<LANES>(t[0] * o2[0] + t[1] * o2[1] + t[2] * o2[2] + t[3] * o2[3]);
    if (c == 0) {
      const long long m1 = 2 * h * NqP + row, m2 = m1 + NqP;
      a.delta[m1] = __builtin_amdgcn_ldexpf((float)s1, -ex);
      a.delta[m2] = __builtin_amdgcn_ldexpf((float)s2, -ex);
      a.dc[m1] = a.lsf[m1] * pow2(ex);
      a.dc[m2] = a.lsf[m2] * -lam * pow2(ex);
    }
    dl -= s2;
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

struct Sums { const double* part; int n, blocks; float* dlam; float* dw; };      // of n workgroups of diff_bwd_pre_kernel
// the partials' column sums: a wave per column (H of dlam, then 2 hd of dw)
__device__ __forceinline__ void bwd_sums(const Args& a, const Sums& m, int blk) {
  const int W = a.H + 2 * a.hd, c = blk * (NT / 64) + (int)(threadIdx.x >> 6);
  if (c >= W) return;
  double s = 0.0;
  for (int r = threadIdx.x & 63; r < m.n; r += 64) s += m.part[(long long)r * W + c];
  s = wave_sum_d(s);
  if ((threadIdx.x & 63) == 0) {
    if (c < a.H) m.dlam[c] = (float)s;
    else if (m.dw != nullptr) m.dw[c - a.H] = (float)s;
  }
}

// dS = p (G - delta), delta the row's mean of G under p.  delta comes from the outputs (do . o: rows as long as one likes, one number), which is off by
// the rounding of o; where one key holds nearly all of the weight G - delta cancels down to that.  Rows with 32 keys at most up to their last
// visible one — a session's first rows, short sessions — take the mean of the very G - delta in a second step: a row with one key has a gradient of exactly zero.
// (A mask that leaves one key of a longer session does not: dS is rounding there, 1e-7 of |do| |v|.)
// ---- backward, dQ: the owner is a query; both maps need G^T = V dO^T, each wave makes it over half of V's columns and they swap halves ------
// STAGES: two where two workgroups with two chunk buffers fit a CU's LDS (HD 32; training passes with two | with one: 128 sessions of 200 285 | 290 us,
// 16 of 2,048 1,021 | 1,028), else one: the other workgroup's products run under the copy.
template <int HD> constexpr int bwd_stages() { return HD == 32 ? 2 : 1; }
template <int HD> constexpr int dkv_stage() { return 2 * Row<HD>::CHUNK + 1024; }
template <int HD> constexpr int bwd_lds() { return bwd_stages<HD>() * dkv_stage<HD>() + 4 * 8 * 64 * 16; }      // (dQ needs less)

template <int HD>
__device__ __forceinline__ void bwd_dq(const Args& a, unsigned char* smem, int blk) {
  constexpr int NS = HD / 16, NB = HD / 32, STAGE = fwd_stage<HD>(), STAGES = bwd_stages<HD>();
  f32x4* swap = reinterpret_cast<f32x4*>(smem + STAGES * STAGE);      // [wave][4][64]
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_of(tid), mp = wave & 1, rg = wave >> 1, i = lane & 31, g = lane >> 5;
  const Work wk = work_of(a, a.own_q, blk, a.H, a.causal != 0);
  if (!wk.any) return;
  const int h = wk.h, hk = h / (a.H / a.Hkv), hd = a.hd, dv = 2 * hd;
  const long long NqP = a.Nq + PAD, NkP = a.Nk + PAD;
  if (wk.b == a.B) {      // rows behind the last session have no gradient
    for (long long r = rows_used(a.cu_q, a.B, a.Nq) + wk.tile; r < a.Nq; r += a.own_q.n_tiles)
      for (int c = tid; c < dv; c += NT) a.dq[r * a.lddq + (long long)h * dv + c] = 0.f;
    return;
  }
  long long qr0, kr0; int nq, nk;
  rows_of(a.cu_q, wk.b, a.Lq, a.Nq, qr0, nq);
  rows_of(a.cu_k, wk.b, a.Lk, a.Nk, kr0, nk);
  const int off = nk - nq;
  const unsigned lds0 = lds_addr(smem);
  const long long krow = hk * NkP + kr0;
  auto issue = [&](int c, int st) {
    const unsigned dst = lds0 + st * STAGE;
    const long long r = krow + c * CH;
    copy_chunk<HD>(a.kp + r * Row<HD>::BYTES, dst, tid);
    copy_chunk<HD>(a.vp + r * Row<HD>::BYTES, dst + Row<HD>::CHUNK, tid);
    const long long at = kr0 + c * CH + i;
    if (wave == 0) dma4(a.ks + (2 * hk + g) * NkP + at, dst + 2 * Row<HD>::CHUNK);
    if (wave == 1) dma4((g == 0 ? a.lvb : a.vs) + hk * NkP + at, dst + 2 * Row<HD>::CHUNK + 256);
  };

  for (int tile = wk.tile; tile * OWN < nq; tile += a.own_q.n_tiles) {
    const int q0 = tile * OWN + 32 * rg, qi = q0 + i;
    const bool qok = qi < nq;
    const long long qrow = qr0 + min(qi, nq - 1);
    P2 Qp[NS], Dp[NS];      // dO: columns mp * HD .. of the padded 2 HD
    load_own<NS>(a.qp + (h * NqP + qrow) * Row<HD>::BYTES + mp * 4 * HD, 0, 2 * HD, g, Qp);
    load_own<NS>(a.dp + (h * NqP + qrow) * Row<HD>::BYTES, mp * HD, 4 * HD, g, Dp);
    const long long at = (2 * h + mp) * NqP + qrow;
    const float qsc = a.qs[at] * (a.scale * LOG2E), lse = a.lse[at], dl = a.delta[at], dc = a.dc[at];
    f32x16 dQ[NB];
#pragma unroll
    for (int cb = 0; cb < NB; ++cb) dQ[cb] = zero16();
    float unit = NO_UNIT;
    const int k_end = a.causal ? min(nk, tile * OWN + OWN + off) : nk;
    const int n_ch = k_end > 0 ? (k_end + CH - 1) / CH : 0;
    barrier();
    if (STAGES == 2 && n_ch > 0) issue(0, 0);
    int st = 0;
    for (int c = 0; c < n_ch; ++c, st ^= STAGES - 1) {
      const int t0 = c * CH, left = nk - t0;
      unsigned char* img = smem + st * STAGE;
      float* sc = reinterpret_cast<float*>(img + 2 * Row<HD>::CHUNK);
      if (STAGES == 1) {
        if (c > 0) barrier();      // chunk c - 1 has been read
        issue(c, 0);
      }
      dma_done();
      barrier();
      if (STAGES == 2 && c + 1 < n_ch) issue(c + 1, st ^ 1);
      if (left < CH) {
        clear_rows<HD>(img, left, tid);
        if (tid < 128 && (tid & 31) >= left) sc[tid] = 0.f;
        barrier();
      }
      const bool on = q0 < nq && !(a.causal && t0 > q0 + 31 + off);      // (the same for the two waves of a row group)
      f32x16 S, G;
      if (on) {
        rows_dot<HD, NS>(img + Row<HD>::CHUNK, mp * HD, 4 * HD, Dp, i, g, G);
#pragma unroll
        for (int r = 0; r < 4; ++r) swap[(wave * 4 + r) * 64 + lane] = f32x4{G[4 * r], G[4 * r + 1], G[4 * r + 2], G[4 * r + 3]};
        rows_dot<HD, NS>(img + mp * 4 * HD, 0, 2 * HD, Qp, i, g, S);
      }
      barrier();
      if (!on) continue;
      float x[16];
      const bool edge = left < CH || (a.causal && t0 + 31 > q0 + off);
      const int last = a.causal ? min(qi + off - t0, left - 1) : left - 1;
      if ((a.causal ? min(nk, q0 + 32 + off) : nk) <= CH) {      // the only chunk that these rows see
        float sum = 0.f, mean = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const bool ok = reg_row(r, g) <= last && sc[64 + reg_row(r, g)] != -INFINITY;
          x[r] = ok ? __builtin_amdgcn_exp2f(fmaf(S[r] * sc[32 * mp + reg_row(r, g)], qsc, -lse)) : 0.f;
          G[r] = fmaf(G[r] + swap[((wave ^ 1) * 4 + (r >> 2)) * 64 + lane][r & 3], sc[96 + reg_row(r, g)], -dl);
          sum += x[r];
        }
        sum += __shfl_xor(sum, 32, 64);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if (x[r] > 0.f) mean = fmaf(x[r] / sum, G[r], mean);
          __builtin_amdgcn_sched_barrier(0);      // (one key after the other: few registers)
        }
        mean += __shfl_xor(mean, 32, 64);
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] *= (G[r] - mean) * sc[32 * mp + reg_row(r, g)];
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const f32x4 other = swap[((wave ^ 1) * 4 + r) * 64 + lane];
          const f32x4 k4 = *reinterpret_cast<const f32x4*>(sc + 32 * mp + 8 * r + 4 * g), v4 = *reinterpret_cast<const f32x4*>(sc + 96 + 8 * r + 4 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            x[4 * r + e] = __builtin_amdgcn_exp2f(fmaf(S[4 * r + e] * k4[e], qsc, -lse)) * fmaf(G[4 * r + e] + other[e], v4[e], -dl) * k4[e];
        }
      }
      if (edge) {
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = reg_row(r, g) <= last ? x[r] : 0.f;
      }
      if (a.key_ids != nullptr) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const f32x4 b4 = *reinterpret_cast<const f32x4*>(sc + 64 + 8 * r + 4 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[4 * r + e] = b4[e] == -INFINITY ? 0.f : x[4 * r + e];
        }
      }
      P2 w[2];
      split16_scaled<NB>(x, unit, dQ, w);
      cols_dot<HD, NB>(img + mp * 4 * HD, 0, 2 * HD, w, lane, dQ);
    }
    if (qok) {
      const int n = fresh(hd), vec = fresh(a.vec_q);
      float* o = a.dq + (qr0 + qi) * a.lddq + (long long)(2 * h + mp) * n;
      const float f = a.scale * dc / unit;      // (the row's own factors wait until here)
#pragma unroll
      for (int cb = 0; cb < NB; ++cb)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          put4(o, 32 * cb + 8 * r + 4 * g, n, f32x4{dQ[cb][4 * r], dQ[cb][4 * r + 1], dQ[cb][4 * r + 2], dQ[cb][4 * r + 3]} * f, vec != 0);
    }
  }
}

// ---- backward, dK and dV: the owner is a key; the query heads of its group are summed in a fixed order ---------------------------------------
// The two waves of a row group swap their halves of G and their probabilities: each makes dK of its map and dV of its half of the columns.
template <int HD>
__device__ __forceinline__ void bwd_dkv(const Args& a, unsigned char* smem, int blk) {
  constexpr int NS = HD / 16, NB = HD / 32, STAGE = dkv_stage<HD>(), STAGES = bwd_stages<HD>();
  f32x4* swap = reinterpret_cast<f32x4*>(smem + STAGES * STAGE);      // [wave][8][64]: G halves, probabilities
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_of(tid), mp = wave & 1, rg = wave >> 1, i = lane & 31, g = lane >> 5;
  const Work wk = work_of(a, a.own_k, blk, a.Hkv, false);
  if (!wk.any) return;
  const int hk = wk.h, rep = a.H / a.Hkv, hd = a.hd, dv = 2 * hd;
  const long long NqP = a.Nq + PAD, NkP = a.Nk + PAD;
  if (wk.b == a.B) {
    for (long long r = rows_used(a.cu_k, a.B, a.Nk) + wk.tile; r < a.Nk; r += a.own_k.n_tiles)
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
  const unsigned lds0 = lds_addr(smem);
  const int c_all = (nq + CH - 1) / CH;
  // row values behind the images: scales of the maps' queries | lse | delta | dc, each [2][32]
  auto issue = [&](int h, int c, int st) {
    const unsigned dst = lds0 + st * STAGE;
    const long long r = h * NqP + qr0 + c * CH;
    copy_chunk<HD>(a.qp + r * Row<HD>::BYTES, dst, tid);
    copy_chunk<HD>(a.dp + r * Row<HD>::BYTES, dst + Row<HD>::CHUNK, tid);
    const long long at = (2 * h + g) * NqP + qr0 + c * CH + i;
    const float* src = wave == 0 ? a.qs + at : wave == 1 ? a.lse + at : wave == 2 ? a.delta + at : a.dc + at;
    dma4(src, dst + 2 * Row<HD>::CHUNK + wave * 256);
  };

  for (int tile = wk.tile; tile * OWN < nk; tile += a.own_k.n_tiles) {
    const int k0 = tile * OWN + 32 * rg, ki = k0 + i;
    const bool kin = ki < nk;
    const long long krow = kr0 + min(ki, nk - 1);
    const bool kok = kin && a.lvb[hk * NkP + krow] != -INFINITY;
    P2 Kp[NS], Vp[NS];
    load_own<NS>(a.kp + (hk * NkP + krow) * Row<HD>::BYTES + mp * 4 * HD, 0, 2 * HD, g, Kp);
    load_own<NS>(a.vp + (hk * NkP + krow) * Row<HD>::BYTES, mp * HD, 4 * HD, g, Vp);
    const float ksc = a.ks[(2 * hk + mp) * NkP + krow] * (a.scale * LOG2E), vsc = a.vs[hk * NkP + krow];
    f32x16 dK[NB], dV[NB];
#pragma unroll
    for (int cb = 0; cb < NB; ++cb) { dK[cb] = zero16(); dV[cb] = zero16(); }
    float unit_k = NO_UNIT, unit_v = NO_UNIT;
    const int c_lo = a.causal ? min(c_all, max(0, tile * OWN - off) / CH) : 0, n_ch = c_all - c_lo, n_all = n_ch * rep;      // chunks of the heads one after another
    barrier();
    if (STAGES == 2 && n_all > 0) issue(hk * rep, c_lo, 0);
    int st = 0;
    for (int n = 0; n < n_all; ++n, st ^= STAGES - 1) {
      const int h = hk * rep + n / n_ch, c = c_lo + n % n_ch, t0 = c * CH, left = nq - t0;
      unsigned char* img = smem + st * STAGE;
      float* sc = reinterpret_cast<float*>(img + 2 * Row<HD>::CHUNK);
      if (STAGES == 1) {
        if (n > 0) barrier();
        issue(h, c, 0);
      }
      dma_done();
      barrier();
      if (STAGES == 2 && n + 1 < n_all) issue(hk * rep + (n + 1) / n_ch, c_lo + (n + 1) % n_ch, st ^ 1);
      if (left < CH) {      // rows behind the session's end have no probabilities
        clear_rows<HD>(img, left, tid);
        if ((tid & 31) >= left) sc[tid] = 0.f;
        barrier();
      }
      const bool on = k0 < nk && !(a.causal && t0 + 31 + off < k0);
      f32x16 S, G;
      float p[16];
      if (on) {
        rows_dot<HD, NS>(img + mp * 4 * HD, 0, 2 * HD, Kp, i, g, S);
        rows_dot<HD, NS>(img + Row<HD>::CHUNK, mp * HD, 4 * HD, Vp, i, g, G);
        const bool edge = a.causal && t0 + off < k0 + 31;
        const int first = a.causal ? ki - off - t0 : -1;      // the first row of the chunk that sees this key
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const f32x4 q4 = *reinterpret_cast<const f32x4*>(sc + 32 * mp + 8 * r + 4 * g), l4 = *reinterpret_cast<const f32x4*>(sc + 64 + 32 * mp + 8 * r + 4 * g),
                      c4 = *reinterpret_cast<const f32x4*>(sc + 192 + 32 * mp + 8 * r + 4 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e) p[4 * r + e] = __builtin_amdgcn_exp2f(fmaf(S[4 * r + e] * q4[e], ksc, -l4[e])) * c4[e];
        }
        if (edge) {
#pragma unroll
          for (int r = 0; r < 16; ++r) p[r] = reg_row(r, g) >= first ? p[r] : 0.f;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          swap[(wave * 8 + r) * 64 + lane] = f32x4{G[4 * r], G[4 * r + 1], G[4 * r + 2], G[4 * r + 3]};
          swap[(wave * 8 + 4 + r) * 64 + lane] = f32x4{p[4 * r], p[4 * r + 1], p[4 * r + 2], p[4 * r + 3]};
        }
      }
      barrier();
      if (!on) continue;
      float x[16];
      P2 w[2];
      const bool few = (a.causal ? min(nk, t0 + 32 + off) : nk) <= CH;      // rows that see no other keys than the wave's
      if (few) {
        const float* own = reinterpret_cast<const float*>(swap + wave * 8 * 64 + lane);
        const float* other = reinterpret_cast<const float*>(swap + (wave ^ 1) * 8 * 64 + lane);
#pragma unroll 1
        for (int r = 0; r < 16; ++r) {      // (a loop: unrolled it costs the kernel registers that it has not got)
          const int at = (r >> 2) * 256 + (r & 3), row = 32 * mp + reg_row(r, g);
          const bool ok = kok && (!a.causal || t0 + reg_row(r, g) + off >= ki);
          const float pr = ok ? own[1024 + at] : 0.f, sum = group_sum<32>(pr), gr = fmaf(own[at] + other[at], vsc, -sc[128 + row]);
          const float mean = group_sum<32>(ok && sum != 0.f ? pr / sum * gr : 0.f);
          if (i == 0) sc[64 + row] = mean;      // (where the exponents were: read above, by this wave alone)
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x4 og = swap[((wave ^ 1) * 8 + r) * 64 + lane];
        const f32x4 q4 = *reinterpret_cast<const f32x4*>(sc + 32 * mp + 8 * r + 4 * g), dl = *reinterpret_cast<const f32x4*>(sc + 128 + 32 * mp + 8 * r + 4 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) G[4 * r + e] = fmaf(G[4 * r + e] + og[e], vsc, -dl[e]);
        if (few) {
          const f32x4 m4 = *reinterpret_cast<const f32x4*>(sc + 64 + 32 * mp + 8 * r + 4 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e) G[4 * r + e] -= m4[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * r + e] = p[4 * r + e] * G[4 * r + e] * q4[e];
      }
      split16_scaled<NB>(x, unit_k, dK, w);
      cols_dot<HD, NB>(img + mp * 4 * HD, 0, 2 * HD, w, lane, dK);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x4 op = swap[((wave ^ 1) * 8 + 4 + r) * 64 + lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * r + e] = p[4 * r + e] + op[e];
      }
      split16_scaled<NB>(x, unit_v, dV, w);
      cols_dot<HD, NB>(img + Row<HD>::CHUNK, mp * HD, 4 * HD, w, lane, dV);
    }
    if (kin) {      // a masked key's lane holds whatever its zeroed row made of the probabilities: its gradients are zero
      const int n = fresh(hd), vec = fresh(a.vec_kv);
      float* ok = a.dk + (kr0 + ki) * a.lddk + (long long)(2 * hk + mp) * n;
      float* ov = a.dv + (kr0 + ki) * a.lddv + (long long)hk * 2 * n;
      const float fk = a.scale / unit_k, fv = 1.f / unit_v;
#pragma unroll
      for (int cb = 0; cb < NB; ++cb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int col = 32 * cb + 8 * r + 4 * g;
          f32x4 tk = f32x4{dK[cb][4 * r], dK[cb][4 * r + 1], dK[cb][4 * r + 2], dK[cb][4 * r + 3]} * fk;
          f32x4 tv = f32x4{dV[cb][4 * r], dV[cb][4 * r + 1], dV[cb][4 * r + 2], dV[cb][4 * r + 3]} * fv;
          if (!kok) tk = tv = f32x4{0.f, 0.f, 0.f, 0.f};
          put4(ok, col, n, tk, vec != 0);
          put4(ov, mp * HD + col, 2 * n, tv, vec != 0);
        }
    }
  }
}

// Both passes in one launch, the dK/dV workgroups (one and a half times the work of the others) first: they share no data, and each alone ends with
// a few of its longest workgroups on an empty machine.  Two sessions of 4,096, 4 heads of hd 64, causal: 466 us = 3.6e11 flops (three terms a product) at
// 775 TFLOP/s; one launch after the other 309 + 445 us before the later steps, together 562.  The column sums of dlam and dw ride along between the two.
template <int HD>
__global__ __launch_bounds__(NT, 2) void diff_bwd_kernel(Args a, Sums m) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int blk = blockIdx.x;
  if (blk < a.own_k.blocks) bwd_dkv<HD>(a, smem, blk);
  else if (blk < a.own_k.blocks + m.blocks) bwd_sums(a, m, blk - a.own_k.blocks);
  else bwd_dq<HD>(a, smem, blk - a.own_k.blocks - m.blocks);
}

// ---- few query rows: the products are matrix-vector products, the keys and values are read once and the loads are the work ---------------------
// A workgroup takes the R queries (rows x heads) that share a key head through its share of the keys.  A wave reads TK keys at a time straight
// into registers: a key's two maps (and its value row) lie across 2 HD / 4 lanes, four columns each, so every load is whole cache lines; a
// dot product is four multiply-adds and a sum over the lanes of its map (cross-lane adds, no LDS), the two maps' lanes swap their probabilities, the value
// sums stay with the lanes' columns.  Every lane group keeps its own running maximum and sum until the end; no barrier in the loop, and the
// next TK keys are read while these are taken.  1,024 sessions of up to 200 keys, 4 heads of hd 32, one query each: 43 us = 6.1 TB/s (memory bound);
// 8 sessions of up to 65,536, 4 queries to each of 2 key heads of hd 64: 130 us = 5.0 TB/s; 8 of 65,536 each 186 us = 5.8 TB/s with one query, 194 with
// four.  R is the next power of two: instances for 1, 2, 4, 8, so that one query pays for one.
constexpr int MAXR = 8;

template <int HD> __device__ __forceinline__ float other_map(float v) {
  if (HD == 32) return dpp<0x128>(v);      // rotated by 8 in 16 lanes
  return lane_xor16(v);
}
template <int HD> __device__ __forceinline__ float keys_max(float v) {      // over the keys of one load
  if (HD == 32) v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
template <int HD> __device__ __forceinline__ float keys_sum(float v) {
  if (HD == 32) v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}
constexpr int decode_keys(int HDP) { return HDP == 32 ? 16 : 8; }      // TK

template <int HD, int MODE, int R>
__global__ __launch_bounds__(NT, R > 4 ? 1 : 2) void diff_decode_kernel(Args a) {
  constexpr int DV = 2 * HD, LPK = HD / 2, KPL = 64 / LPK, NL = 4, TK = KPL * NL;
  __shared__ float wstat[4][R][2][2], wacc[4][R][2][DV];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, kk = lane / LPK, c4 = lane % LPK, mp = c4 / (HD / 4), cm = c4 % (HD / 4), col = cm * 4;
  const int id = blockIdx.x, nbh = gridDim.x / a.n_split, split = a.share > 0 ? id % a.n_split : id / nbh, bh = a.share > 0 ? id / a.n_split : id % nbh, b = bh / a.Hkv, hk = bh % a.Hkv, rep = a.H / a.Hkv, hd = a.hd, dv = 2 * hd;
  if (b == a.B) {      // rows behind the last session: zeros
    if (split != 0) return;
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
    f32x4 qv[R], acc[R][2];                        // acc: value columns 4 c4 .. + 3 under the two maps
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
    const int n_t = (k_end + TK - 1) / TK, each = max(a.share, (n_t + a.n_split - 1) / a.n_split), t_lo = min(n_t, split * each), t_hi = min(n_t, t_lo + each);
    if (a.share > 0 && split > 0 && t_lo >= n_t) {      // nothing left: an empty share (diff_combine_kernel does not read its sums)
      for (int u = tid; u < 2 * rows * rep; u += NT) {
        const int w = u >> 1;
        const long long at = (((long long)split * a.Nq + qr0 + first + w / rep) * a.H + hk * rep + w % rep) * 2 + (u & 1);
        a.ml[2 * at] = -INFINITY;
        a.ml[2 * at + 1] = 0.f;
      }
      continue;
    }
    const float* kbase = a.k + kr0 * a.ldk + (long long)(2 * hk + mp) * hd;
    const float* vbase = a.v + kr0 * a.ldv + (long long)hk * dv;
    struct Tile { f32x4 k[NL], v[NL]; unsigned live; };
    auto read = [&](int t, Tile& x) {
      x.live = 0u;
#pragma unroll
      for (int u = 0; u < NL; ++u) {
        const int key = t * TK + u * KPL + kk;
        x.k[u] = x.v[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (t < t_hi && key < k_end && (a.key_ids == nullptr || a.key_ids[kr0 + key] != 0)) {
          x.live |= 1u << u;
          x.k[u] = get4<MODE>(kbase + (long long)key * a.ldk, col, hd);
          x.v[u] = get4<MODE>(vbase + (long long)key * a.ldv, 4 * c4, dv);
        }
      }
    };
    auto take = [&](int t, const Tile& x) {
      const bool edge = __any(x.live != (1u << NL) - 1u) || (a.causal && t * TK + TK - 1 > first + off);
#pragma unroll
      for (int w = 0; w < R; ++w) {
        if (w >= rows * rep) break;
        float s[NL], mx = m[w];
#pragma unroll
        for (int u = 0; u < NL; ++u)
          s[u] = group_sum<HD / 4>(fmaf(qv[w][0], x.k[u][0], qv[w][1] * x.k[u][1]) + fmaf(qv[w][2], x.k[u][2], qv[w][3] * x.k[u][3]));
        if (edge) {
          const int last = a.causal ? first + w / rep + off : 0x7FFFFFFF;
#pragma unroll
          for (int u = 0; u < NL; ++u) s[u] = (((x.live >> u) & 1u) == 0u || t * TK + u * KPL + kk > last) ? -INFINITY : s[u];
        }
#pragma unroll
        for (int u = 0; u < NL; ++u) mx = fmaxf(mx, s[u]);
        if (__any(mx != m[w])) {
          const float alpha = __builtin_amdgcn_exp2f(m[w] - (mx == -INFINITY ? 0.f : mx));
          const float other = other_map<HD>(alpha);
          m[w] = mx;
          l[w] *= alpha;
          acc[w][0] *= mp == 0 ? alpha : other;
          acc[w][1] *= mp == 0 ? other : alpha;
        }
        const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll
        for (int u = 0; u < NL; ++u) {
          const float p = __builtin_amdgcn_exp2f(s[u] - base), po = other_map<HD>(p), p0 = mp == 0 ? p : po, p1 = mp == 0 ? po : p;
          l[w] += p;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            acc[w][0][e] = fmaf(p0, x.v[u][e], acc[w][0][e]);
            acc[w][1][e] = fmaf(p1, x.v[u][e], acc[w][1][e]);
          }
        }
      }
    };
    Tile x, y;      // one is read while the other is taken
    read(t_lo + wave, x);
    for (int t = t_lo + wave; t < t_hi; t += 8) {
      read(t + 4, y);
      take(t, x);
      if (t + 4 >= t_hi) break;
      read(t + 8, x);
      take(t + 4, y);
    }
    __syncthreads();      // (the previous pass's readers are done)
#pragma unroll
    for (int w = 0; w < R; ++w) {                  // the lane groups of the wave meet
      const float mx = keys_max<HD>(m[w]), e = __builtin_amdgcn_exp2f(m[w] - (mx == -INFINITY ? 0.f : mx)), lt = keys_sum<HD>(l[w] * e);
      const float eo = other_map<HD>(e);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        acc[w][0][k] = keys_sum<HD>(acc[w][0][k] * (mp == 0 ? e : eo));
        acc[w][1][k] = keys_sum<HD>(acc[w][1][k] * (mp == 0 ? eo : e));
      }
      if (kk == 0) {
        if (cm == 0) { wstat[wave][w][mp][0] = mx; wstat[wave][w][mp][1] = lt; }
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
          const long long at = (((long long)split * a.Nq + row) * a.H + h) * 2 + q;
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
// In 64 bits: the difference of the two exponentials is all that is left of them (a head of few columns lost 2e-7 of lam).  1.8 us, 4.6 behind a kernel that has emptied the caches
__device__ __forceinline__ double wave_dot(const float* x, const float* y, int n, int lane) {
  double s = 0.0;
  for (int c = lane; c < n; c += 64) s += (double)x[c] * (double)y[c];
  return wave_sum_d(s);
}
__global__ __launch_bounds__(64) void diff_lambda_fwd_kernel(const float* q1, const float* k1, const float* q2, const float* k2, float init, int hd, float* lam) {
  const long long o = (long long)blockIdx.x * hd;
  const double e1 = exp(wave_dot(q1 + o, k1 + o, hd, threadIdx.x)), e2 = exp(wave_dot(q2 + o, k2 + o, hd, threadIdx.x));
  if (threadIdx.x == 0) lam[blockIdx.x] = (float)(e1 - e2 + (double)init);
}
__global__ __launch_bounds__(64) void diff_lambda_bwd_kernel(const float* dlam, const float* q1, const float* k1, const float* q2, const float* k2, int hd,
                                                             float* dq1, float* dk1, float* dq2, float* dk2) {
  const long long o = (long long)blockIdx.x * hd;
  const float g = dlam[blockIdx.x];
  const float e1 = (float)(g * exp(wave_dot(q1 + o, k1 + o, hd, threadIdx.x))), e2 = (float)(-g * exp(wave_dot(q2 + o, k2 + o, hd, threadIdx.x)));
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

struct Plan { bool decode; int n_split, share; };
// Training keeps the outputs of both maps and always takes the matrix kernels.  Otherwise few queries to a key head (rows x heads of its group) go
// through diff_decode_kernel, up to twelve of them, in two passes over the keys behind eight.  Decode against matrix, causal, hd 64, 2 key heads:
//   1 query   8 x 65,536 keys 185 | 763 us   256 x 200 19 | 62     1 x 8,192 17 | 29
//   8         8 x 65,536      370 | 1158     256 x 200 60 | 128    1 x 8,192 30 | 35
//   10        8 x 65,536      555 | 837      256 x 200 84 | 88     1 x 8,192 39 | 31
//   16        8 x 65,536      729 | 837      256 x 200 114 | 89    1 x 8,192 48 | 31
// Keys are split over workgroups until the launch has what the machine holds at once, two per CU (decode of more than four queries: its registers
// leave one), with 2 (decode) or 4 chunks each at least.  Decode, 64 sessions of 2,048 keys: 4 queries 52 us (1 per CU: 68, 4 per CU: 58), 8 queries
// 105 (2: 114, 4: 133); matrix, 8 x 1,024 rows of 4 heads: 82 (1: 84, 4: 134).
// Decode over sessions of different lengths (their keys are below nine tenths of B x Lk): shares of one size instead of one number, so that a long session
// has more workgroups and not longer ones, an eighth fewer than fit (a session's last share counts as one), a session's shares on different
// dies.  Lengths of a long tail, one size | one number: 8 of up to 65,536 keys, 8 heads on 2 of hd 64 155 | 183 us; 300 of up to 1,000, one head of
// hd 50 86 | 105; 100 of up to 2,000, 8 heads on 2 of hd 32 40 | 45; 32 of up to 8,192, 4 heads of hd 64 154 | 142.  Sessions of one length keep the order that
// leaves a session's shares on one die (8 of 65,536: 194 us, spread out 204).
Plan plan_of(int B, int H, int Hkv, int hd, int Lq, int Lk, long long Nk, bool train) {
  Plan p;
  const int rep = H / Hkv;
  const long long queries = (long long)rep * Lq;
  p.decode = !train && rep <= MAXR && queries <= MAXR + MAXR / 2;
  const long long wgs = p.decode ? (long long)B * Hkv : (long long)B * H * ((Lq + OWN - 1) / OWN);
  const int tile = decode_keys(pad_hd(hd)), chunk = p.decode ? 4 * tile : CH;      // keys a workgroup takes at once
  const long long want = (long long)rt_num_cus() * (p.decode && queries > 4 ? 1 : 2);
  const bool ragged = p.decode && 10 * Nk < 9 * (long long)B * Lk && Nk > 0;
  long long s = ragged ? want * 7 / 8 * Lk / (Nk * Hkv) : (wgs > 0 ? want / wgs : 1);
  const long long most = Lk / (p.decode ? 2 * chunk : 4 * chunk);
  if (s > most) s = most;
  if (s > 64) s = 64;
  p.n_split = s > 1 ? (int)s : 1;
  p.share = ragged && p.n_split > 1 ? ((Lk + tile - 1) / tile + p.n_split - 1) / p.n_split : 0;
  return p;
}
size_t part_floats(const Plan& p, long long Nq, int H, int hd) {
  return p.n_split > 1 ? (size_t)p.n_split * (size_t)Nq * H * 2 * (2 * (size_t)hd + 2) : 0;
}

constexpr long long MAX_ROWS = 0x3FFFFFFF;      // rows within a session are counted in 32 bits; offsets into q, k, v are 64 bits everywhere
int check(int B, int H, int Hkv, int hd, int Lq, int Lk, long long Nq, long long Nk, const void* cu_q, const void* cu_k) {
  if (B < 0 || H <= 0 || Hkv <= 0 || hd <= 0 || Lq < 0 || Lk < 0 || Nq < 0 || Nk < 0 || H % Hkv != 0) return RT_ERR_INVALID_ARG;
  if (hd > 64 || Nq > MAX_ROWS || Nk > MAX_ROWS) return RT_ERR_UNSUPPORTED;
  if (cu_q == nullptr && Nq != (long long)B * Lq) return RT_ERR_INVALID_ARG;
  if (cu_k == nullptr && Nk != (long long)B * Lk) return RT_ERR_INVALID_ARG;
  return RT_OK;
}
// a launch dimension holds less than 2^32 threads
bool grid_ok(long long blocks) { return blocks > 0 && blocks <= 0xFFFFFFFFLL / NT; }
// work of B sessions x H heads x tiles of L owner rows (tail: and the rows behind the last session)
bool plan_grid(Grid& g, int B, int H, int L, bool tail) {
  const long long bhs = (long long)B * H, counted = bhs >= 64 ? (bhs + 7) / 8 * 8 : (bhs > 0 ? bhs : 1), tiles = L > 0 ? (L + OWN - 1) / OWN : 1;
  const long long blocks = (counted + (tail ? H : 0)) * tiles;
  g = Grid{(int)tiles, (int)counted, (int)blocks};
  return grid_ok(blocks);
}


// consecutive 256-byte aligned pieces of a buffer (base null: sizes only)
struct Carve {
  unsigned char* base; size_t at = 0;
  template <typename T> void take(T*& p, size_t n) {
    if (base != nullptr) p = reinterpret_cast<T*>(base + at);
    at += (n * sizeof(T) + 255) & ~(size_t)255;
  }
};
size_t carve_planes(Args& a, void* base, bool train) {      // what diff_planes_kernel writes; train: and what the forward keeps for the backward
  Carve c{static_cast<unsigned char*>(base)};
  const size_t row = 8 * (size_t)pad_hd(a.hd) + 48, nq = (size_t)a.Nq + PAD, nk = (size_t)a.Nk + PAD, H = a.H, G = a.Hkv;
  c.take(a.qp, H * nq * row);
  c.take(a.kp, G * nk * row);
  c.take(a.vp, G * nk * row);
  c.take(a.qs, 2 * H * nq);
  c.take(a.ks, 2 * G * nk);
  c.take(a.vs, G * nk);
  c.take(a.ivs, G * nk);
  c.take(a.lvb, G * nk);
  if (train) {
    c.take(a.lse, 2 * H * nq);
    c.take(a.lsf, 2 * H * nq);
    c.take(a.o12, (size_t)a.Nq * H * 4 * a.hd);
  }
  return c.at;
}
size_t carve_backward(Args& a, void* base, double*& part) {
  Carve c{static_cast<unsigned char*>(base)};
  const size_t row = 8 * (size_t)pad_hd(a.hd) + 48, nq = (size_t)a.Nq + PAD, H = a.H;
  c.take(a.dp, H * nq * row);
  c.take(a.delta, 2 * H * nq);
  c.take(a.dc, 2 * H * nq);
  c.take(part, (size_t)PRE_WG * (H + 2 * a.hd));
  return c.at;
}
Args sizes(int H, int Hkv, int hd, long long Nq, long long Nk) {
  Args a{};
  a.H = H; a.Hkv = Hkv; a.hd = hd; a.Nq = Nq; a.Nk = Nk;
  return a;
}

template <typename K, typename... A>
int start(K kernel, dim3 grid, int threads, size_t lds, hipStream_t stream, const A&... a) {
  if (lds > 65536) RT_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  kernel<<<grid, threads, lds, stream>>>(a...);
  RT_CHECK_LAUNCH();
  return RT_OK;
}
// mode: 0 the head fills its tile and rows are 16-byte aligned, 1 aligned, columns checked, 2 single columns, checked
int mode_of(bool vec, int hd) { return !vec ? 2 : (hd == pad_hd(hd) ? 0 : 1); }

template <int HD, int R>
int start_decode(int mode, dim3 grid, hipStream_t stream, const Args& a) {
  return mode == 0 ? start(diff_decode_kernel<HD, 0, R>, grid, NT, 0, stream, a) : mode == 1 ? start(diff_decode_kernel<HD, 1, R>, grid, NT, 0, stream, a)
                                                                                         : start(diff_decode_kernel<HD, 2, R>, grid, NT, 0, stream, a);
}
template <int HD>
int start_decode(long long queries, int mode, dim3 grid, hipStream_t stream, const Args& a) {
  return queries <= 1 ? start_decode<HD, 1>(mode, grid, stream, a) : queries <= 2 ? start_decode<HD, 2>(mode, grid, stream, a)
         : queries <= 4 ? start_decode<HD, 4>(mode, grid, stream, a) : start_decode<HD, 8>(mode, grid, stream, a);
}
template <int HD>
int start_planes(const Args& a, int mode, hipStream_t stream) {
  constexpr int GROUPS = NT / (HD / 2);
  const long long qb = (a.Nq * a.H + GROUPS - 1) / GROUPS, kb = (a.Nk * a.Hkv + GROUPS - 1) / GROUPS, n = qb + 2 * kb;
  if (!grid_ok(n)) return RT_ERR_UNSUPPORTED;
  if (mode == 0) diff_planes_kernel<HD, 0><<<(unsigned)n, NT, 0, stream>>>(a, (unsigned)qb, (unsigned)kb);
  else if (mode == 1) diff_planes_kernel<HD, 1><<<(unsigned)n, NT, 0, stream>>>(a, (unsigned)qb, (unsigned)kb);
  else diff_planes_kernel<HD, 2><<<(unsigned)n, NT, 0, stream>>>(a, (unsigned)qb, (unsigned)kb);
  RT_CHECK_LAUNCH();
  return RT_OK;
}
template <int HD>
int start_pre(const Args& a, int mode, unsigned n, const float* dy, long long lddy, double* part, hipStream_t stream) {
  if (mode == 0) diff_bwd_pre_kernel<HD, 0><<<n, NT, 0, stream>>>(a, dy, lddy, part);
  else if (mode == 1) diff_bwd_pre_kernel<HD, 1><<<n, NT, 0, stream>>>(a, dy, lddy, part);
  else diff_bwd_pre_kernel<HD, 2><<<n, NT, 0, stream>>>(a, dy, lddy, part);
  RT_CHECK_LAUNCH();
  return RT_OK;
}
#define RT_TRY(call)                 \
  do {                               \
    const int rc__ = (call);         \
    if (rc__ != RT_OK) return rc__;  \
  } while (0)

}  // namespace

extern "C" {

size_t rt_diffattn_saved_bytes(int32_t H, int32_t Hkv, int32_t hd, int64_t Nq, int64_t Nk) {
  if (H <= 0 || Hkv <= 0 || hd <= 0 || hd > 64 || Nq < 0 || Nk < 0) return 0;
  Args a = sizes(H, Hkv, hd, Nq, Nk);
  return carve_planes(a, nullptr, true);
}

size_t rt_diffattn_fwd_workspace_bytes(int32_t B, int32_t H, int32_t Hkv, int32_t hd, int32_t Lq, int32_t Lk, int64_t Nq, int64_t Nk, int32_t train) {
  if (B < 0 || H <= 0 || Hkv <= 0 || hd <= 0 || hd > 64 || Lq < 0 || Lk < 0 || Nq <= 0 || Nk < 0 || H % Hkv != 0) return 0;
  const Plan p = plan_of(B > 0 ? B : 1, H, Hkv, hd, Lq, Lk, Nk, train != 0);
  Args a = sizes(H, Hkv, hd, Nq, Nk);
  return part_floats(p, Nq, H, hd) * sizeof(float) + (train == 0 && !p.decode ? carve_planes(a, nullptr, false) + 256 : 0);
}

int rt_diffattn_fwd(const float* q, int64_t ldq, const float* k, int64_t ldk, const float* v, int64_t ldv, const float* lam, const int64_t* cu_q,
                    const int64_t* cu_k, const int64_t* key_ids, int32_t B, int32_t H, int32_t Hkv, int32_t hd, int32_t Lq, int32_t Lk, int64_t Nq,
                    int64_t Nk, float scale, int32_t causal, const float* norm_w, float out_scale, float eps, float* y, int64_t ldy, void* saved,
                    size_t saved_bytes, void* ws, size_t ws_bytes, hipStream_t stream) {
  RT_TRY(check(B, H, Hkv, hd, Lq, Lk, Nq, Nk, cu_q, cu_k));
  const long long wq = 2LL * H * hd, wk = 2LL * Hkv * hd;
  if (lam == nullptr || (norm_w != nullptr && !(eps > 0.f)) || (Nq > 0 && (q == nullptr || y == nullptr || ldq < wq || ldy < wq))) return RT_ERR_INVALID_ARG;
  if (Nk > 0 && (k == nullptr || v == nullptr || ldk < wk || ldv < wk)) return RT_ERR_INVALID_ARG;
  if (saved != nullptr && (saved_bytes < rt_diffattn_saved_bytes(H, Hkv, hd, Nq, Nk) || ((uintptr_t)saved & 15u) != 0)) return RT_ERR_WORKSPACE;
  if (Nq == 0) return RT_OK;
  Args a = sizes(H, Hkv, hd, Nq, Nk);
  a.q = q; a.k = k; a.v = v; a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.lam = lam;
  a.cu_q = (const long long*)cu_q; a.cu_k = (const long long*)cu_k; a.key_ids = (const long long*)key_ids;
  a.B = B; a.Lq = Lq; a.Lk = Lk;
  a.scale = scale > 0.f ? scale : 1.f / sqrtf((float)hd); a.causal = causal;
  a.norm_w = norm_w; a.out_scale = out_scale; a.eps = eps; a.y = y; a.ldy = ldy;
  const Plan p = plan_of(B > 0 ? B : 1, H, Hkv, hd, Lq, Lk, Nk, saved != nullptr);
  a.n_split = p.n_split; a.share = p.share;
  const size_t part_bytes = part_floats(p, Nq, H, hd) * sizeof(float);
  const size_t need = part_bytes + (saved == nullptr && !p.decode ? carve_planes(a, nullptr, false) + 256 : 0);
  if (need > 0 && (ws == nullptr || ws_bytes < need || ((uintptr_t)ws & 15u) != 0)) return RT_ERR_WORKSPACE;
  if (p.n_split > 1) {
    a.part = (float*)ws;
    a.ml = a.part + (size_t)p.n_split * Nq * H * 4 * hd;
  }
  const int HDP = pad_hd(hd);
  const int mode = mode_of(hd % 4 == 0 && vec_ok(q, ldq) && vec_ok(k, ldk) && vec_ok(v, ldv), hd);
  a.vec_y = hd % 2 == 0 && vec_ok(y, ldy);
  const long long B1 = B + (cu_q != nullptr ? 1 : 0);
  if (p.decode) {
    if (!grid_ok(B1 * Hkv * p.n_split)) return RT_ERR_UNSUPPORTED;
    const long long queries = (long long)(H / Hkv) * (Lq > 0 ? Lq : 1);
    const dim3 grid((unsigned)(B1 * Hkv * p.n_split));
    RT_TRY(HDP == 32 ? start_decode<32>(queries, mode, grid, stream, a) : start_decode<64>(queries, mode, grid, stream, a));
  } else {
    if (!plan_grid(a.own_q, B, H, Lq, cu_q != nullptr)) return RT_ERR_UNSUPPORTED;
    // One workgroup of eight waves per CU, two chunks at a time, where all the workgroups of four would be resident at once: a CU keeps the two it is given
    // then, and a causal session's heavy one ends alone; as one workgroup the tiles are dealt out one after the other, the light ones behind the
    // heavy ones.  4 heads, planes included: 2 x 4,096 rows, hd 64 267 -> 219 us, hd 32 174 -> 134; 1 x 4,096 (keys in two splits) 197 -> 148.  Short shares of
    // the keys lose by the join of the two halves (1 x 1,024, eight splits: 36 -> 42 us; 100 x 128, hd 32: 22.5 -> 25.8), and where there are more tiles
    // than that, two independent workgroups overlap better (64 x 512, hd 64: 205 -> 248).
    const bool wide = causal && Lk / p.n_split > 256 && (long long)B * H * a.own_q.n_tiles * p.n_split <= 2LL * rt_num_cus();
    carve_planes(a, saved != nullptr ? saved : (unsigned char*)ws + ((part_bytes + 255) & ~(size_t)255), saved != nullptr);
    RT_TRY(HDP == 32 ? start_planes<32>(a, mode, stream) : start_planes<64>(a, mode, stream));
    const dim3 grid((unsigned)a.own_q.blocks, p.n_split);
    const int lds = HDP == 32 ? 2 * fwd_stage<32>() : 2 * fwd_stage<64>();
    if (wide) RT_TRY(HDP == 32 ? start(diff_fwd_kernel<32, 2>, grid, 2 * NT, 2 * lds, stream, a) : start(diff_fwd_kernel<64, 2>, grid, 2 * NT, 2 * lds, stream, a));
    else RT_TRY(HDP == 32 ? start(diff_fwd_kernel<32, 1>, grid, NT, lds, stream, a) : start(diff_fwd_kernel<64, 1>, grid, NT, lds, stream, a));
  }
  if (p.n_split > 1) {
    if (!grid_ok(Nq * H)) return RT_ERR_UNSUPPORTED;
    diff_combine_kernel<<<(unsigned)(Nq * H), NT, 0, stream>>>(a);
    RT_CHECK_LAUNCH();
  }
  return RT_OK;
}

size_t rt_diffattn_bwd_workspace_bytes(int32_t H, int32_t hd, int64_t Nq) {
  if (H <= 0 || hd <= 0 || hd > 64 || Nq < 0) return 0;
  Args a = sizes(H, 1, hd, Nq, 0);
  double* part = nullptr;
  return carve_backward(a, nullptr, part);
}

int rt_diffattn_bwd(const void* saved, size_t saved_bytes, const float* lam, const int64_t* cu_q, const int64_t* cu_k, const int64_t* key_ids, int32_t B,
                    int32_t H, int32_t Hkv, int32_t hd, int32_t Lq, int32_t Lk, int64_t Nq, int64_t Nk, float scale, int32_t causal, const float* norm_w,
                    float out_scale, float eps, const float* dy, int64_t lddy, float* dq, int64_t lddq, float* dk, int64_t lddk, float* dv, int64_t lddv,
                    float* dlam, float* dw, void* ws, size_t ws_bytes, hipStream_t stream) {
  RT_TRY(check(B, H, Hkv, hd, Lq, Lk, Nq, Nk, cu_q, cu_k));
  const long long wq = 2LL * H * hd, wk = 2LL * Hkv * hd;
  if (lam == nullptr || dlam == nullptr || (norm_w != nullptr) != (dw != nullptr)) return RT_ERR_INVALID_ARG;
  if (Nq > 0 && (dy == nullptr || dq == nullptr || lddy < wq || lddq < wq)) return RT_ERR_INVALID_ARG;
  if (Nk > 0 && (dk == nullptr || dv == nullptr || lddk < wk || lddv < wk)) return RT_ERR_INVALID_ARG;
  if (saved == nullptr || saved_bytes < rt_diffattn_saved_bytes(H, Hkv, hd, Nq, Nk) || ((uintptr_t)saved & 15u) != 0) return RT_ERR_WORKSPACE;
  if (ws == nullptr || ws_bytes < rt_diffattn_bwd_workspace_bytes(H, hd, Nq) || ((uintptr_t)ws & 15u) != 0) return RT_ERR_WORKSPACE;
  Args a = sizes(H, Hkv, hd, Nq, Nk);
  a.lam = lam; a.cu_q = (const long long*)cu_q; a.cu_k = (const long long*)cu_k; a.key_ids = (const long long*)key_ids;
  a.B = B; a.Lq = Lq; a.Lk = Lk;
  a.scale = scale > 0.f ? scale : 1.f / sqrtf((float)hd); a.causal = causal;
  a.norm_w = norm_w; a.out_scale = out_scale; a.eps = eps;
  a.dq = dq; a.dk = dk; a.dv = dv; a.lddq = lddq; a.lddk = lddk; a.lddv = lddv;
  a.vec_q = hd % 4 == 0 && vec_ok(dq, lddq);
  a.vec_kv = hd % 4 == 0 && vec_ok(dk, lddk) && vec_ok(dv, lddv);
  double* part = nullptr;
  carve_planes(a, const_cast<void*>(saved), true);
  carve_backward(a, ws, part);

  const int HDP = pad_hd(hd), groups = NT / (HDP / 2);
  const long long least = (H + groups - 1) / groups;      // (one lane group per head at least)
  long long n_pre = (Nq * H + groups - 1) / groups;
  n_pre = n_pre > PRE_WG ? PRE_WG : n_pre;
  n_pre = n_pre < least ? least : n_pre;
  if (n_pre > PRE_WG) return RT_ERR_UNSUPPORTED;
  const int mode = mode_of(hd % 2 == 0 && vec_ok(dy, lddy) && (norm_w == nullptr || vec_ok(norm_w, 4)), hd);
  RT_TRY(HDP == 32 ? start_pre<32>(a, mode, (unsigned)n_pre, dy, lddy, part, stream) : start_pre<64>(a, mode, (unsigned)n_pre, dy, lddy, part, stream));
  if ((Nq > 0 && !plan_grid(a.own_q, B, H, Lq, cu_q != nullptr)) || (Nk > 0 && !plan_grid(a.own_k, B, Hkv, Lk, cu_k != nullptr))) return RT_ERR_UNSUPPORTED;
  const Sums m{part, (int)n_pre, (H + 2 * hd + NT / 64 - 1) / (NT / 64), dlam, dw};
  const long long blocks = (long long)a.own_q.blocks + a.own_k.blocks + m.blocks;
  if (!grid_ok(blocks)) return RT_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)blocks);
  RT_TRY(HDP == 32 ? start(diff_bwd_kernel<32>, grid, NT, bwd_lds<32>(), stream, a, m) : start(diff_bwd_kernel<64>, grid, NT, bwd_lds<64>(), stream, a, m));
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
