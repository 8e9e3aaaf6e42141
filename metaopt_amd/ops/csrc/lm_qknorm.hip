// Query / key head norms with the position rotation, and the split of a QKV activation into heads
// (ops/heads.py qk_norm_rope, qk_norm_rope_cached).
//
//   y = x rsqrt(mean_D(x^2) + eps) w[trial],  z = R(position) y      for every query and key head
//   v heads are copied.
// Backward, from the saved activation (the norm is formed again from the x that is read anyway):
//   dy = R^T dz,  u = w dy,  x^ = x r,  dx = r (u - x^ mean(u x^)),  dw[trial] = sum dy x^
//
// x: [rows][(H + 2 KV) D], rows ordered (trial, sequence, token).  A head of one row is held by
// D / 8 lanes, 16 bytes each; the mean is a butterfly over those lanes, the pairs of an
// interleaved rotation lie within a lane and those of a rotate-half one in lane ^ (D / 16).
// Everything is bound by memory: each value is read once and written once.  32768 rows of 36 heads
// of 64: forward 51 us (6.0 TB/s), backward 81 us and 4 for the weights (5.0 TB/s); 12003 rows of 28
// heads of 128: 34 (5.1 TB/s) and 57 + 6 us.
#include "elt.h"

using namespace mopt;

namespace {

struct QkArgs {
  const uint16_t* x;
  int64_t x_ld;               // row stride of x (elements)
  const uint16_t *wq, *wk;    // [P][D]
  const float *cosT, *sinT;   // [reach][D / 2]
  const int32_t* start;       // per sequence position of its first token (cached form), or null
  uint16_t *q, *k, *v;        // q [B][H][T][D]; k, v with the strides below
  int64_t k_sb, k_sh, k_st, v_sb, v_sh, v_st;
  int rows, T, H, KV, rpt, reach, cap;   // cap: rows of the cache
  float eps;
};

template <int LPR>
__device__ __forceinline__ float sum_lanes(float v) {
#pragma unroll
  for (int o = 1; o < LPR; o <<= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// f rotated by +angle (sgn = 1) or -angle (sgn = -1); col = first column of this lane's 8
template <int D, bool IL>
__device__ __forceinline__ void rotate8(float (&f)[8], const float* cs, const float* sn, int col,
                                        float sgn) {
  if constexpr (IL) {
    const f32x4 c = *(const f32x4*)(cs + (col >> 1)), s = *(const f32x4*)(sn + (col >> 1));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a = f[2 * j], b = f[2 * j + 1], si = sgn * s[j];
      f[2 * j] = a * c[j] - b * si;
      f[2 * j + 1] = b * c[j] + a * si;
    }
  } else {
    const bool low = col < D / 2;
    const int at = low ? col : col - D / 2;
    const float side = low ? -sgn : sgn;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 c = *(const f32x4*)(cs + at + 4 * h), s = *(const f32x4*)(sn + at + 4 * h);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float own = f[4 * h + j], other = __shfl_xor(own, D / 16, 64);
        f[4 * h + j] = own * c[j] + side * other * s[j];
      }
    }
  }
}

template <class E, int D, bool IL>
__global__ __launch_bounds__(256) void qk_norm_rope_fwd_kernel(QkArgs a) {
  constexpr int LPR = D / 8, UPB = 256 / LPR;    // lanes per head row, head rows per block
  const int nh = a.H + 2 * a.KV;
  const int64_t unit = (int64_t)blockIdx.x * UPB + threadIdx.x / LPR;
  const int col = (threadIdx.x % LPR) * 8;
  // whole head rows drop out together, and a row's lanes only exchange among themselves
  if (unit >= (int64_t)a.rows * nh) return;
  const int r = (int)(unit / nh), hh = (int)(unit - (int64_t)r * nh);
  const int b = r / a.T, t = r - b * a.T;
  const int64_t pos = a.start ? (int64_t)a.start[b] + t : t;
  const bool in = pos >= 0 && pos < a.reach && pos < a.cap;
  const u32x4 raw = *(const u32x4*)(a.x + (int64_t)r * a.x_ld + hh * D + col);
  const int64_t at = a.start ? pos : t;
  if (hh >= a.H + a.KV) {
    if (in) *(u32x4*)(a.v + b * a.v_sb + (hh - a.H - a.KV) * a.v_sh + at * a.v_st + col) = raw;
    return;
  }
  const bool isq = hh < a.H;
  float f[8], w[8];
  up8<E>(raw, f);
  up8<E>(*(const u32x4*)((isq ? a.wq : a.wk) + (int64_t)(r / a.rpt) * D + col), w);
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) ss = fmaf(f[j], f[j], ss);
  const float rstd = rsqrtf(sum_lanes<LPR>(ss) * (1.f / D) + a.eps);
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] *= rstd * w[j];
  const int64_t ang = in ? pos * (D / 2) : 0;
  rotate8<D, IL>(f, a.cosT + ang, a.sinT + ang, col, 1.f);
  u32x4 out = down8<E>(f);
  if (isq) {
    if (!in) out = u32x4{0, 0, 0, 0};      // a token behind the cache: no position, no query
    *(u32x4*)(a.q + (((int64_t)b * a.H + hh) * a.T + t) * D + col) = out;
  } else if (in) {
    *(u32x4*)(a.k + b * a.k_sb + (hh - a.H) * a.k_sh + at * a.k_st + col) = out;
  }
}

struct QkBwdArgs {
  const uint16_t* x;
  int64_t x_ld;
  const uint16_t *wq, *wk;
  const float *cosT, *sinT;
  const uint16_t *dq, *dk, *dv;      // [B][H | KV][T][D]
  uint16_t* dx;                      // [rows][(H + 2 KV) D]
  float* part;                       // [P][blocks][2][D]
  int rows, T, H, KV, rpt, per;      // per: rows of one block
  float eps;
};

// `heads` query or key heads of rows [r0, r0 + n), the first at column c0 of x: their dx, and this
// thread's terms of dw
template <class E, int D, bool IL>
__device__ __forceinline__ void heads_bwd(const QkBwdArgs& a, int r0, int n, int c0, int heads, const uint16_t* dz,
                                          const uint16_t* wg, float (&acc)[8]) {
  constexpr int LPR = D / 8, UPB = 256 / LPR;
  const int nh = a.H + 2 * a.KV, col = (threadIdx.x % LPR) * 8;
  float w[8];
  up8<E>(*(const u32x4*)(wg + col), w);
  const int units = n * heads;
#pragma unroll 2
  for (int u = threadIdx.x / LPR; u < units; u += UPB) {
    const int rl = u / heads, hh = u - rl * heads, r = r0 + rl;
    const int b = r / a.T, t = r - b * a.T;
    float x[8], d[8];
    up8<E>(*(const u32x4*)(a.x + (int64_t)r * a.x_ld + c0 + hh * D + col), x);
    up8<E>(*(const u32x4*)(dz + (((int64_t)b * heads + hh) * a.T + t) * D + col), d);
    rotate8<D, IL>(d, a.cosT + (int64_t)t * (D / 2), a.sinT + (int64_t)t * (D / 2), col, -1.f);
    float ss = 0.f, dot = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ss = fmaf(x[j], x[j], ss);
      dot = fmaf(d[j] * w[j], x[j], dot);
    }
    ss = sum_lanes<LPR>(ss);
    dot = sum_lanes<LPR>(dot);
    const float rstd = rsqrtf(ss * (1.f / D) + a.eps), m = dot * rstd * rstd * (1.f / D);
    float o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      o[j] = rstd * (d[j] * w[j] - x[j] * m);
      acc[j] += d[j] * x[j] * rstd;
    }
    *(u32x4*)(a.dx + ((int64_t)r * nh) * D + c0 + hh * D + col) = down8<E>(o);
  }
}

// One block: rows [per * blockIdx.x, ...) of trial blockIdx.y; its sums of dw over rows and heads
// go to part in a fixed order (no atomics), qk_norm_dw_kernel adds the blocks.
template <class E, int D, bool IL>
__global__ __launch_bounds__(256) void qk_norm_rope_bwd_kernel(QkBwdArgs a) {
  constexpr int LPR = D / 8, UPB = 256 / LPR;
  __shared__ float red[UPB][2 * D + 4];
  const int col = (threadIdx.x % LPR) * 8, slot = threadIdx.x / LPR, p = blockIdx.y;
  const int lo = blockIdx.x * a.per, n = min(lo + a.per, a.rpt) - lo, r0 = p * a.rpt + lo;
  float aq[8] = {}, ak[8] = {};
  heads_bwd<E, D, IL>(a, r0, n, 0, a.H, a.dq, a.wq + (int64_t)p * D, aq);
  heads_bwd<E, D, IL>(a, r0, n, a.H * D, a.KV, a.dk, a.wk + (int64_t)p * D, ak);
  const int units = n * a.KV, nh = a.H + 2 * a.KV;
#pragma unroll 2
  for (int u = slot; u < units; u += UPB) {            // values: copied
    const int rl = u / a.KV, hh = u - rl * a.KV, r = r0 + rl, b = r / a.T, t = r - b * a.T;
    *(u32x4*)(a.dx + ((int64_t)r * nh + a.H + a.KV + hh) * D + col) =
        *(const u32x4*)(a.dv + (((int64_t)b * a.KV + hh) * a.T + t) * D + col);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    red[slot][col + j] = aq[j];
    red[slot][D + col + j] = ak[j];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * D; c += 256) {
    float s = 0.f;
    for (int i = 0; i < UPB; ++i) s += red[i][c];
    a.part[((int64_t)p * gridDim.x + blockIdx.x) * 2 * D + c] = s;
  }
}

// dwq, dwk [P][D] = sums of part over its blocks: 16 of the 2 D columns a workgroup, 64 slices of the
// blocks (one trial with 1024 blocks: 6 us, with 4 slices of 64 columns 122)
template <class E, int D>
__global__ __launch_bounds__(1024) void qk_norm_dw_kernel(const float* __restrict__ part, int blocks,
                                                          uint16_t* dwq, uint16_t* dwk) {
  __shared__ float red[64][17];
  const int p = blockIdx.y, l = threadIdx.x & 15, c = blockIdx.x * 16 + l, s = threadIdx.x >> 4;
  float v = 0.f;
#pragma unroll 8
  for (int i = s; i < blocks; i += 64) v += part[((int64_t)p * blocks + i) * 2 * D + c];
  red[s][l] = v;
  __syncthreads();
  if (s == 0) {
    v = 0.f;
    for (int i = 0; i < 64; ++i) v += red[i][l];
    uint16_t* dst = c < D ? dwq + (int64_t)p * D + c : dwk + (int64_t)p * D + c - D;
    *dst = (uint16_t)(E::pack2(v, v) & 0xFFFF);
  }
}

template <class E, int D>
int fwd(const QkArgs& a, int il, hipStream_t st) {
  const int64_t units = (int64_t)a.rows * (a.H + 2 * a.KV), upb = 2048 / D;
  const dim3 grid((unsigned)((units + upb - 1) / upb));
  if (il)
    hipLaunchKernelGGL((qk_norm_rope_fwd_kernel<E, D, true>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((qk_norm_rope_fwd_kernel<E, D, false>), grid, dim3(256), 0, st, a);
  return (int)hipGetLastError();
}

template <class E, int D>
int bwd(const QkBwdArgs& a, int P, int blocks, int il, uint16_t* dwq, uint16_t* dwk,
        hipStream_t st) {
  const dim3 grid(blocks, P);
  if (il)
    hipLaunchKernelGGL((qk_norm_rope_bwd_kernel<E, D, true>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((qk_norm_rope_bwd_kernel<E, D, false>), grid, dim3(256), 0, st, a);
  hipLaunchKernelGGL((qk_norm_dw_kernel<E, D>), dim3(2 * D / 16, P), dim3(1024), 0, st, a.part,
                     blocks, dwq, dwk);
  return (int)hipGetLastError();
}

}  // namespace

extern "C" {

// dtype 0: bf16, 1: fp16.  D is 64 or 128; every address and stride of a row is a multiple of 16
// bytes (checked by the caller).  start null: T tokens a sequence at positions 0 ... T - 1.
int mopt_qk_norm_rope_fwd(const void* x, int64_t x_ld, const void* wq, const void* wk,
                          const void* cosT, const void* sinT, const void* start, void* q, void* k,
                          void* v, const int64_t* kv_strides, int rows, int T, int H, int KV, int rpt,
                          int D, int reach, int cap, float eps, int il, int dtype, void* stream) {
  if (rows <= 0 || T <= 0 || H <= 0 || KV <= 0 || rpt <= 0 || (D != 64 && D != 128)) return 1;
  if (cap <= 0 || reach <= 0) return 1;      // (row 0 of the tables is read for a token without a position)
  if (!start && (cap < T || reach < T)) return 1;
  if (((int64_t)rows * (H + 2 * KV) * D) / 2048 >= (1ll << 31) - 1) return 1;
  const QkArgs a{(const uint16_t*)x, x_ld, (const uint16_t*)wq, (const uint16_t*)wk,
                 (const float*)cosT, (const float*)sinT, (const int32_t*)start, (uint16_t*)q,
                 (uint16_t*)k, (uint16_t*)v, kv_strides[0], kv_strides[1], kv_strides[2],
                 kv_strides[3], kv_strides[4], kv_strides[5], rows, T, H, KV, rpt, reach, cap, eps};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == 0) return D == 64 ? fwd<Bf16, 64>(a, il, st) : fwd<Bf16, 128>(a, il, st);
  return D == 64 ? fwd<Fp16, 64>(a, il, st) : fwd<Fp16, 128>(a, il, st);
}

// blocks: workgroups of each trial's rows; part: workspace of [P][blocks][2][D] floats
int mopt_qk_norm_rope_bwd(const void* x, int64_t x_ld, const void* wq, const void* wk,
                          const void* cosT, const void* sinT, const void* dq, const void* dk,
                          const void* dv, void* dx, void* part, void* dwq, void* dwk, int rows, int T,
                          int H, int KV, int rpt, int D, int blocks, float eps, int il, int dtype,
                          void* stream) {
  if (rows <= 0 || T <= 0 || H <= 0 || KV <= 0 || rpt <= 0 || rows % rpt || blocks <= 0 || blocks > rpt || (D != 64 && D != 128)) return 1;
  const int P = rows / rpt;
  const int per = (rpt + blocks - 1) / blocks;
  if ((int64_t)per * (H + 2 * KV) >= (1ll << 31) - 256) return 1;
  const QkBwdArgs a{(const uint16_t*)x, x_ld, (const uint16_t*)wq, (const uint16_t*)wk,
                    (const float*)cosT, (const float*)sinT, (const uint16_t*)dq, (const uint16_t*)dk,
                    (const uint16_t*)dv, (uint16_t*)dx, (float*)part, rows, T, H, KV, rpt, per, eps};
  hipStream_t st = (hipStream_t)stream;
  uint16_t *gq = (uint16_t*)dwq, *gk = (uint16_t*)dwk;
  if (dtype == 0)
    return D == 64 ? bwd<Bf16, 64>(a, P, blocks, il, gq, gk, st) : bwd<Bf16, 128>(a, P, blocks, il, gq, gk, st);
  return D == 64 ? bwd<Fp16, 64>(a, P, blocks, il, gq, gk, st) : bwd<Fp16, 128>(a, P, blocks, il, gq, gk, st);
}

}  // extern "C"
