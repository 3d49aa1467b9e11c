// Rotary positions: the pairs of a head's first `rot` columns turn by the angle position * frequency.
//
//   (a, b) -> gain * (a cos phi - b sin phi, a sin phi + b cos phi),  phi = t f_j,  j = 0 .. rot / 2 - 1
//
// half layout: (a, b) = (x[j], x[j + rot / 2]); interleaved: (x[2 j], x[2 j + 1]); columns from `rot` on are copied.  The backward pass is the
// transposed map: the same kernel with the angle's sign turned.  The angle is formed and reduced to a fraction of a turn in 64 bits — at
// position 10^6 an fp32 product is off by 0.06 rad — and only the reduced fraction goes to fp32 (sincospif).
//
// Memory bound: every column is read and written once.  The sine and cosine of a (row, pair) are shared by all heads of q AND k: a thread
// keeps them for up to 4 heads of its pairs (64-bit product, reduction and sincos are about 50 operations a pair; at one head per thread
// they cost as much issue time as the memory traffic: half as long again).  65,536 rows, 16 + 4 heads of 64 columns, 32 of them turned, interleaved: 122 us
// = 5.5 TB/s; heads of 63 columns, which no wide load divides: 164 us = 4.0 TB/s, all of them turned 135.  With few rows the heads go to threads of their own instead: latency counts there.
#include "rt_common.h"

namespace {

struct Seg { const float* x; float* y; long long ldx, ldy; int heads; };
struct RotArgs {
  Seg s[2];
  const long long* pos; const double* freq;
  long long M;
  int hd, rot, groups, units, rows_per_wg;      // groups: head groups; units: work units of a head
  float gain, sign;
};

// V pairs (rotated part) or V columns (the rest) per unit
template <int V, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(RotArgs a) {
  const int T = a.groups * a.units, half = a.rot / 2, turn_units = (half + V - 1) / V, heads = a.s[0].heads + a.s[1].heads;
  const int in_row = T <= 256 ? (int)threadIdx.x / T : 0;
  if (in_row >= a.rows_per_wg) return;
  for (long long row = (long long)blockIdx.x * a.rows_per_wg + in_row; row < a.M; row += (long long)gridDim.x * a.rows_per_wg) {
    for (int t = T <= 256 ? (int)threadIdx.x % T : (int)threadIdx.x; t < T; t += 256) {
      const int unit = t % a.units, hg = t / a.units;
      const bool turns = unit < turn_units;
      float cs[V], sn[V];
      const int j0 = unit * V;
      if (turns) {
        const double p = (double)a.pos[row];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const double rev = (p * a.freq[min(j0 + e, half - 1)]) * 0.15915494309189533577;      // 1 / (2 pi)
          float s, c;
          sincospif(2.f * (float)(rev - rint(rev)), &s, &c);
          cs[e] = c * a.gain;
          sn[e] = s * a.gain * a.sign;
        }
      }
      auto in = [&](int h) { return h < a.s[0].heads ? a.s[0].x + row * a.s[0].ldx + (long long)h * a.hd : a.s[1].x + row * a.s[1].ldx + (long long)(h - a.s[0].heads) * a.hd; };
      auto out = [&](int h) { return h < a.s[0].heads ? a.s[0].y + row * a.s[0].ldy + (long long)h * a.hd : a.s[1].y + row * a.s[1].ldy + (long long)(h - a.s[0].heads) * a.hd; };
      if (V == 1) {      // single columns: a thread's heads are read in front of the first one's store (one after the other: two
        // 4-byte loads in flight, 65,536 rows of 20 heads of 63 columns 294 us instead of 164)
        const int ia = turns ? (INTER ? 2 * j0 : j0) : a.rot + unit - turn_units, ib = INTER ? 2 * j0 + 1 : half + j0;
        for (int h0 = hg; h0 < heads; h0 += 4 * a.groups) {
          float u[4], v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int h = h0 + j * a.groups;
            if (h < heads) {
              u[j] = in(h)[ia];
              v[j] = turns ? in(h)[ib] : 0.f;
            }
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int h = h0 + j * a.groups;
            if (h < heads) {
              float* y = out(h);
              y[ia] = turns ? u[j] * cs[0] - v[j] * sn[0] : u[j];
              if (turns) y[ib] = u[j] * sn[0] + v[j] * cs[0];
            }
          }
        }
        continue;
      }
      for (int h = hg; h < heads; h += a.groups) {
        const float* x = in(h);
        float* y = out(h);
        if (!turns) {
          const int c0 = a.rot + (unit - turn_units) * V;
          *reinterpret_cast<f32x4*>(y + c0) = *reinterpret_cast<const f32x4*>(x + c0);
          continue;
        }
        if (INTER) {
          const f32x4 u = *reinterpret_cast<const f32x4*>(x + 2 * j0), v = *reinterpret_cast<const f32x4*>(x + 2 * j0 + 4);
          *reinterpret_cast<f32x4*>(y + 2 * j0) = f32x4{u[0] * cs[0] - u[1] * sn[0], u[0] * sn[0] + u[1] * cs[0],
                                                        u[2] * cs[1 % V] - u[3] * sn[1 % V], u[2] * sn[1 % V] + u[3] * cs[1 % V]};
          *reinterpret_cast<f32x4*>(y + 2 * j0 + 4) = f32x4{v[0] * cs[2 % V] - v[1] * sn[2 % V], v[0] * sn[2 % V] + v[1] * cs[2 % V],
                                                            v[2] * cs[3 % V] - v[3] * sn[3 % V], v[2] * sn[3 % V] + v[3] * cs[3 % V]};
        } else {
          const f32x4 u = *reinterpret_cast<const f32x4*>(x + j0), v = *reinterpret_cast<const f32x4*>(x + half + j0);
          f32x4 p, q;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            p[e] = u[e] * cs[e % V] - v[e] * sn[e % V];
            q[e] = u[e] * sn[e % V] + v[e] * cs[e % V];
          }
          *reinterpret_cast<f32x4*>(y + j0) = p;
          *reinterpret_cast<f32x4*>(y + half + j0) = q;
        }
      }
    }
  }
}

}  // namespace

extern "C" int rt_rotary(const float* q, int64_t ldq, float* q_out, int64_t ldq_out, int32_t n_heads, const float* k, int64_t ldk, float* k_out,
                         int64_t ldk_out, int32_t n_kv_heads, const int64_t* pos, const double* freq, int64_t M, int32_t hd, int32_t rot,
                         int32_t interleaved, float gain, int32_t backward, hipStream_t stream) {
  if (M < 0 || hd <= 0 || rot <= 0 || rot % 2 != 0 || rot > hd || n_heads < 0 || n_kv_heads < 0) return RT_ERR_INVALID_ARG;
  const int heads = n_heads + n_kv_heads;
  if (M == 0 || heads == 0) return RT_OK;
  if (pos == nullptr || freq == nullptr) return RT_ERR_INVALID_ARG;
  const long long wq = (long long)n_heads * hd, wk = (long long)n_kv_heads * hd;
  if (n_heads > 0 && (q == nullptr || q_out == nullptr || ldq < wq || ldq_out < wq)) return RT_ERR_INVALID_ARG;
  if (n_kv_heads > 0 && (k == nullptr || k_out == nullptr || ldk < wk || ldk_out < wk)) return RT_ERR_INVALID_ARG;
  RotArgs a{};
  a.s[0] = Seg{q, q_out, ldq, ldq_out, n_heads};
  a.s[1] = Seg{k, k_out, ldk, ldk_out, n_kv_heads};
  a.pos = (const long long*)pos; a.freq = freq; a.M = M; a.hd = hd; a.rot = rot; a.gain = gain; a.sign = backward ? -1.f : 1.f;
  bool vec = hd % 4 == 0 && rot % 8 == 0;
  for (const Seg& s : a.s)
    if (s.heads > 0) vec = vec && (((uintptr_t)s.x | (uintptr_t)s.y) & 15u) == 0 && s.ldx % 4 == 0 && s.ldy % 4 == 0;
  const int V = vec ? 4 : 1;
  a.units = rot / 2 / V + (hd - rot) / V;
  // up to 4 heads per thread where one per thread would be more threads than the machine holds (2,048 per CU): 17,920 rows of 8 + 8 heads of 32 14.4 us
  // (one: 15.4), 64 such rows 4.2 us (one: 3.6)
  a.groups = M * a.units * heads > 2048LL * rt_num_cus() ? (heads + 3) / 4 : heads;
  const long long T = (long long)a.groups * a.units;
  if (T > 0x7FFFFFFF) return RT_ERR_INVALID_ARG;
  a.rows_per_wg = T <= 256 ? (int)(256 / T) : 1;
  const long long blocks = (M + a.rows_per_wg - 1) / a.rows_per_wg;
  const unsigned n = (unsigned)(blocks < (1LL << 23) ? blocks : 1LL << 23);      // (a launch holds less than 2^32 threads; workgroups loop)
  if (vec) {
    if (interleaved) rotary_kernel<4, true><<<n, 256, 0, stream>>>(a);
    else rotary_kernel<4, false><<<n, 256, 0, stream>>>(a);
  } else {
    if (interleaved) rotary_kernel<1, true><<<n, 256, 0, stream>>>(a);
    else rotary_kernel<1, false><<<n, 256, 0, stream>>>(a);
  }
  RT_CHECK_LAUNCH();
  return RT_OK;
}
