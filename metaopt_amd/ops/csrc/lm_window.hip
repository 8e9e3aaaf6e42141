// Causal attention with a sliding window and sink tokens, forward and backward (ops/heads.py
// window_attention).
//
// Query t of sequence b stands at position i = start[b] + t and sees key j when
//   j <= i < len[b]  and  (i - j < W  or  j < S);
// o_i = sum_j p_ij v_j, p = softmax_j(scale q_i . k_j); a query that sees nothing gives zeros.
// Backward: D_i = do_i . o_i, dS = p (do_i . v_j - D_i), dq = scale dS k, dk = scale dS^T q,
// dv = p^T do; the G = H / KV query heads of a key head add to one dk, dv.
//
// Matrix products are 32x32x16 MFMAs.  Lane l of such a product holds A[l & 31][8 (l >> 5) ..+7],
// B[8 (l >> 5) ..+7][l & 31] and, in register r, C[8 (r >> 2) + 4 (l >> 5) + (r & 3)][l & 31].
// Scores are formed transposed (S^T = K Q^T, a lane is one query) with the K rows fed in an order
// that exchanges bits 2 and 3 of the row: register r of lane half h is then key
// 16 (r >> 3) + 8 h + (r & 7), so registers 8 s ... 8 s + 7 are, converted and packed, the B
// operand of step s of the product with V -- P never leaves its lane.  V^T is read with the
// transposing LDS read.  dK / dV do the same with queries in the place of keys.
#include "elt.h"

using namespace mopt;

namespace {

constexpr int BM = 128;        // queries (forward, dQ) or keys (dK / dV) of a workgroup, 32 a wave
constexpr int BN = 64;         // keys (queries) of a staged tile

struct WinArgs {
  const uint16_t *q, *k, *v;
  int64_t q_sb, q_sh, q_st, k_sb, k_sh, k_st, v_sb, v_sh, v_st;   // strides (elements)
  const int32_t *start, *lengths;   // per sequence, or null: start0 / start + Tq
  int start0, B, H, KV, Tq, Tk, W, S;
  float c;                          // scale log2(e)
};

// positions of a sequence: query t is at st + t, valid t are [t0, t1), keys are [0, len)
struct Seq {
  int st, len, t0, t1;
};

__device__ __forceinline__ Seq seq_of(const WinArgs& a, int b) {
  Seq s;
  // (a start that leaves no query among the keys is as good as the nearest such one)
  const int st = max(-a.Tq, min(a.Tk, a.start ? a.start[b] : a.start0));
  s.st = st;
  s.len = max(0, min(a.lengths ? a.lengths[b] : st + a.Tq, a.Tk));
  s.t0 = max(0, -st);
  s.t1 = max(s.t0, min(a.Tq, s.len - st));
  return s;
}

// LDS tiles [rows][D]: the 16-byte chunk c of row r is kept at c ^ f(r).  Of the 16 rows of a
// b128 fragment read no two share a bank; of the 4 rows of a transposing read neither.
template <int D>
__device__ __forceinline__ int swz(int r) {
  return D == 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : ((r & 2) << 1) | ((r >> 2) & 3);
}
template <int D>
__device__ __forceinline__ int at(int r, int c) {      // element offset of (row, column)
  return r * D + (((c >> 3) ^ swz<D>(r)) << 3) + (c & 7);
}

__device__ __forceinline__ u32x4 lds16(const uint16_t* p) { return *(const u32x4*)p; }

__device__ __forceinline__ int swap23(int r) { return (r & 19) | ((r & 4) << 1) | ((r & 8) >> 1); }

// A operand of rows [r0, r0 + 32) in the exchanged order, columns 16 ks ... + 15
template <int D>
__device__ __forceinline__ u32x4 frag(const uint16_t* s, int r0, int ks, int lane) {
  return lds16(s + at<D>(r0 + swap23(lane & 31), 16 * ks + 8 * (lane >> 5)));
}

// A operand of the transpose: rows = columns [32 dn, 32 dn + 32) of the tile, k = rows r0 ... + 15
template <int D>
__device__ __forceinline__ u32x4 frag_t(const uint16_t* s, int r0, int dn, int lane) {
  const int g = lane >> 4, i = lane & 15;
  const int row = r0 + 8 * (g >> 1) + (i >> 2), col = 32 * dn + 16 * (g & 1) + 4 * (i & 3);
  return __builtin_bit_cast(u32x4, cat_frag(lds_tr4((const bf16_t*)s + at<D>(row, col)),
                                            lds_tr4((const bf16_t*)s + at<D>(row + 4, col))));
}

// registers 8 s ... 8 s + 7 of an accumulator as the B operand of step s
template <class E>
__device__ __forceinline__ u32x4 pack(const f32x16& x, int s) {
  return u32x4{E::pack2(x[8 * s], x[8 * s + 1]), E::pack2(x[8 * s + 2], x[8 * s + 3]),
               E::pack2(x[8 * s + 4], x[8 * s + 5]), E::pack2(x[8 * s + 6], x[8 * s + 7])};
}
// the key (query) within a 32-row group that register r of this lane holds
__device__ __forceinline__ int row_of(int r, int lane) {
  return 16 * (r >> 3) + 8 * (lane >> 5) + (r & 7);
}

__device__ __forceinline__ float other_half(float v, bool mx) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const float a = __uint_as_float(p[0]), b = __uint_as_float(p[1]);
  return mx ? fmaxf(a, b) : a + b;
}

__device__ __forceinline__ f32x16 zero16() {
  return f32x16{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
}

// ------------------------------------------------------------------------------------ staging
// Tiles come from memory straight into LDS (global_load_lds: lane l of a wave fills bytes
// 16 l ... of 1 KB), so the exchange of chunks is applied to the addresses that are read.  A ring of
// NS tiles is filled NS - 1 ahead with one barrier a tile: the fills go through inline asm, where
// the compiler does not see them and would wait for all of them before every transposing read, and
// tile_wait waits for those of the next tile itself.  Rows outside [lo, hi) are read as the nearest
// row inside (values of the sequence, finite as the others; the masks leave them out): what padding
// holds is never read.
typedef __attribute__((address_space(3))) void lds_void;

__device__ __forceinline__ uint32_t lds_at(const void* p) {
  return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)((lds_void*)p));
}
__device__ __forceinline__ void fill16(const void* src, const void* dst) {
  asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds_at(dst)) : "memory", "m0");
}
__device__ __forceinline__ void fill4(const void* src, const void* dst) {
  asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(lds_at(dst)) : "memory", "m0");
}

// until at most N of this wave's loads are under way, then until every wave is there
template <int N>
__device__ __forceinline__ void wait_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

template <int D>
constexpr int kFills = BN * D * 2 / 1024 / 4;          // 1 KB fills of a tile by each of 4 waves

template <int D>
__device__ __forceinline__ void fill_tile(const uint16_t* g, int64_t ld, int row0, int lo, int hi, uint16_t* img,
                                          int wave, int lane) {
  constexpr int CH = D / 8, PER = 64 / CH;             // chunks of a row, rows of a fill
#pragma unroll
  for (int j = 0; j < kFills<D>; ++j) {
    const int blk = wave * kFills<D> + j, r = blk * PER + lane / CH, c = (lane % CH) ^ swz<D>(r);
    const int row = max(lo, min(hi - 1, row0 + r));
    fill16(g + row * ld + c * 8, img + blk * 512);
  }
}

// waves a SIMD: the registers that a kernel may use (512 / waves)
#ifndef MOPT_WINDOW_WAVES
#define MOPT_WINDOW_WAVES 3, 2, 3, 2, 3, 2
#endif
constexpr int kWaves[6] = {MOPT_WINDOW_WAVES};
template <int D> constexpr int kFwdWaves = kWaves[D == 128];
template <int D> constexpr int kDqWaves = kWaves[2 + (D == 128)];
template <int D> constexpr int kDkvWaves = kWaves[4 + (D == 128)];

// ring of a kernel: tiles of two matrices
template <int D>
constexpr int kRing = D == 64 ? 3 : 2;

// 4 + 4 consecutive columns of lanes l and l ^ 32 exchanged so that each lane holds 8: register
// pairs (lo, hi) of column groups 8 a + 4 h (a = 0, 1) -> columns 8 h ... 8 h + 7
template <class E>
__device__ __forceinline__ u32x4 join_halves(const float* a0, const float* a1) {
  const uint32_t x0 = E::pack2(a0[0], a0[1]), x1 = E::pack2(a0[2], a0[3]);
  const uint32_t y0 = E::pack2(a1[0], a1[1]), y1 = E::pack2(a1[2], a1[3]);
  const auto p = __builtin_amdgcn_permlane32_swap(x0, y0, false, false);
  const auto q = __builtin_amdgcn_permlane32_swap(x1, y1, false, false);
  return u32x4{p[0], q[0], p[1], q[1]};
}

// rows = lanes (l & 31), columns 32 dn + ...: store an accumulator [D][32] transposed into a row;
// with `rest`, what its rounding left off goes there, rounded
template <class E, int D>
__device__ __forceinline__ void put_rows(uint16_t* row, bool ok, const f32x16 (&acc)[D / 32], float f,
                                         int lane, uint16_t* rest = nullptr) {
#pragma unroll
  for (int dn = 0; dn < D / 32; ++dn)
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      float x[2][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[0][j] = acc[dn][8 * a + j] * f;
        x[1][j] = acc[dn][8 * a + 4 + j] * f;
      }
      const u32x4 w = join_halves<E>(x[0], x[1]);
      if (ok) *(u32x4*)(row + 32 * dn + 16 * a + 8 * (lane >> 5)) = w;
      if (rest) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float v = x[j >> 2][j & 3];
          x[j >> 2][j & 3] = v - E::up(E::pack2(v, v) & 0xFFFF);
        }
        const u32x4 lo = join_halves<E>(x[0], x[1]);
        if (ok) *(u32x4*)(rest + 32 * dn + 16 * a + 8 * (lane >> 5)) = lo;
      }
    }
}

// The key tiles of queries [i0, i1] (positions): first the sink tiles in front of the window,
// then the window's.  Tiles are 64 keys, aligned, so none comes twice.
struct Tiles {
  int sinks, lo, n;
  __device__ __forceinline__ Tiles(int i0, int i1, int W, int S) {
    lo = max(0, i0 - W + 1) / BN;
    sinks = min((S + BN - 1) / BN, lo);
    n = sinks + i1 / BN - lo + 1;
  }
  __device__ __forceinline__ int key(int it) const { return BN * (it < sinks ? it : lo + it - sinks); }
};

// What 32 keys k0 ... are to the queries at positions [i0, i1]: 0 not seen, 1 partly, 2 by all
__device__ __forceinline__ int sight(int k0, int i0, int i1, int W, int S) {
  if (k0 > i1 || (k0 + 31 <= i0 - W && k0 >= S)) return 0;
  if (k0 + 31 <= i0 && (k0 > i1 - W || k0 + 31 < S)) return 2;
  return 1;
}

template <class E, int D>
__global__ __launch_bounds__(256, kFwdWaves<D>) void window_fwd_kernel(WinArgs a, uint16_t* o, uint16_t* rest, float* lse) {
  constexpr int DK = D / 16, DN = D / 32;
  constexpr int NS = kRing<D>;
  __shared__ __attribute__((aligned(16))) uint16_t ring[NS][2][BN * D];
  const int nqb = (a.Tq + BM - 1) / BM;
  const int item = xcd_remap((int)blockIdx.x, (int)gridDim.x);
  const int qb = item % nqb, bh = item / nqb, b = bh / a.H, hq = bh - b * a.H;
  const int hk = hq / (a.H / a.KV);
  const Seq s = seq_of(a, b);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int t = qb * BM + wave * 32 + (lane & 31);        // this lane's query
  const bool valid = t >= s.t0 && t < s.t1;
  const int i = s.st + t;
  // valid queries of the block and of the wave
  const int bt0 = max(s.t0, qb * BM), bt1 = min(s.t1, qb * BM + BM) - 1;
  const int wt0 = max(s.t0, qb * BM + wave * 32), wt1 = min(s.t1, qb * BM + wave * 32 + 32) - 1;

  f32x16 acc[DN];
#pragma unroll
  for (int dn = 0; dn < DN; ++dn) acc[dn] = zero16();
  float m = -3e38f, l = 0.f;
  if (bt0 <= bt1) {
    u32x4 qf[DK];
#pragma unroll
    for (int ks = 0; ks < DK; ++ks) {
      qf[ks] = u32x4{0, 0, 0, 0};
      if (valid)
        qf[ks] = *(const u32x4*)(a.q + b * a.q_sb + hq * a.q_sh + (int64_t)t * a.q_st + 16 * ks + 8 * (lane >> 5));
    }
    const uint16_t* kg = a.k + b * a.k_sb + hk * a.k_sh;
    const uint16_t* vg = a.v + b * a.v_sb + hk * a.v_sh;
    const Tiles tiles(s.st + bt0, s.st + bt1, a.W, a.S);
    auto fetch = [&](int it) {
      fill_tile<D>(kg, a.k_st, tiles.key(it), 0, s.len, ring[it % NS][0], wave, lane);
      fill_tile<D>(vg, a.v_st, tiles.key(it), 0, s.len, ring[it % NS][1], wave, lane);
    };
    for (int it = 0; it < min(NS - 1, tiles.n); ++it) fetch(it);
    for (int it = 0; it < tiles.n; ++it) {
      if (it + NS - 1 <= tiles.n) wait_barrier<2 * kFills<D> * (NS - 2)>();
      else wait_barrier<0>();
      if (it + NS - 1 < tiles.n) fetch(it + NS - 1);
      const uint16_t *Ks = ring[it % NS][0], *Vs = ring[it % NS][1];
      if (wt0 > wt1) continue;
#pragma unroll 1
      for (int sub = 0; sub < 2; ++sub) {
        const int k0 = tiles.key(it) + 32 * sub;
        const int see = sight(k0, s.st + wt0, s.st + wt1, a.W, a.S);
        if (see == 0) continue;
        f32x16 x = zero16();
#pragma unroll
        for (int ks = 0; ks < DK; ++ks) x = E::mfma32(frag<D>(Ks, 32 * sub, ks, lane), qf[ks], x);
        if (see == 1) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int j = k0 + row_of(r, lane);
            if (j > i || (i - j >= a.W && j >= a.S)) x[r] = -INFINITY;
          }
        }
        float mx = x[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, x[r]);
        mx = other_half(mx, true) * a.c;
        // the reference of the exponents moves only when a row's maximum has grown past 2^8 of it:
        // sums and products stay far inside 32 bits, and most tiles need no rescaling
        if (__any(mx > m + 8.f)) {
          const float mn = fmaxf(m, mx), f = __builtin_amdgcn_exp2f(m - mn);
          m = mn;
          l *= f;
#pragma unroll
          for (int dn = 0; dn < DN; ++dn) acc[dn] *= f;
        }
        float part = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          x[r] = __builtin_amdgcn_exp2f(fmaf(x[r], a.c, -m));
          part += x[r];
        }
        l += part;
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          const u32x4 p = pack<E>(x, st);
#pragma unroll
          for (int dn = 0; dn < DN; ++dn)
            acc[dn] = E::mfma32(frag_t<D>(Vs, 32 * sub + 16 * st, dn, lane), p, acc[dn]);
        }
      }
    }
  }
  l = other_half(l, false);
  const bool some = valid && l > 0.f;
  const int64_t row = (((int64_t)b * a.Tq + t) * a.H + hq) * D;
  put_rows<E, D>(o + row, t < a.Tq, acc, some ? 1.f / l : 0.f, lane, rest ? rest + row : nullptr);
  if (lse && lane < 32) lse[(int64_t)bh * nqb * BM + t] = some ? m + log2f(l) : INFINITY;
}

// dQ, and D of its rows for the dK / dV kernel.  D is formed from o and what o's rounding left off
// (`rest`, written by the forward): with o alone its error adds to that of the rounded dS, and where
// few keys are seen it is the larger one (a window of 4: 1.8 times the error of a once rounded dq
// instead of 1.5).
template <class E, int D>
__global__ __launch_bounds__(256, kDqWaves<D>) void window_dq_kernel(WinArgs a, const uint16_t* o, const uint16_t* rest,
                                                        const uint16_t* dout, const float* lse, float* dsum, uint16_t* dq,
                                                        float scale) {
  constexpr int DK = D / 16, DN = D / 32;
  constexpr int NS = kRing<D>;
  __shared__ __attribute__((aligned(16))) uint16_t ring[NS][2][BN * D];
  const int nqb = (a.Tq + BM - 1) / BM;
  const int item = xcd_remap((int)blockIdx.x, (int)gridDim.x);
  const int qb = item % nqb, bh = item / nqb, b = bh / a.H, hq = bh - b * a.H;
  const int hk = hq / (a.H / a.KV);
  const Seq s = seq_of(a, b);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int t = qb * BM + wave * 32 + (lane & 31);
  const bool valid = t >= s.t0 && t < s.t1;
  const int i = s.st + t;
  const int bt0 = max(s.t0, qb * BM), bt1 = min(s.t1, qb * BM + BM) - 1;
  const int wt0 = max(s.t0, qb * BM + wave * 32), wt1 = min(s.t1, qb * BM + wave * 32 + 32) - 1;

  f32x16 acc[DN];
#pragma unroll
  for (int dn = 0; dn < DN; ++dn) acc[dn] = zero16();
  float ds = 0.f;
  if (bt0 <= bt1) {
    u32x4 qf[DK], df[DK];
    const int64_t row = (((int64_t)b * a.Tq + t) * a.H + hq) * D;
#pragma unroll
    for (int ks = 0; ks < DK; ++ks) {
      qf[ks] = df[ks] = u32x4{0, 0, 0, 0};
      if (valid) {
        const int col = 16 * ks + 8 * (lane >> 5);
        qf[ks] = *(const u32x4*)(a.q + b * a.q_sb + hq * a.q_sh + (int64_t)t * a.q_st + col);
        df[ks] = *(const u32x4*)(dout + row + col);
        float x[8], y[8], z[8];
        up8<E>(df[ks], x);
        up8<E>(*(const u32x4*)(o + row + col), y);
        up8<E>(*(const u32x4*)(rest + row + col), z);
#pragma unroll
        for (int j = 0; j < 8; ++j) ds = fmaf(x[j], y[j] + z[j], ds);
      }
    }
    ds = other_half(ds, false);
    const float ls = lse[(int64_t)bh * nqb * BM + t];
    const uint16_t* kg = a.k + b * a.k_sb + hk * a.k_sh;
    const uint16_t* vg = a.v + b * a.v_sb + hk * a.v_sh;
    const Tiles tiles(s.st + bt0, s.st + bt1, a.W, a.S);
    auto fetch = [&](int it) {
      fill_tile<D>(kg, a.k_st, tiles.key(it), 0, s.len, ring[it % NS][0], wave, lane);
      fill_tile<D>(vg, a.v_st, tiles.key(it), 0, s.len, ring[it % NS][1], wave, lane);
    };
    for (int it = 0; it < min(NS - 1, tiles.n); ++it) fetch(it);
    for (int it = 0; it < tiles.n; ++it) {
      if (it + NS - 1 <= tiles.n) wait_barrier<2 * kFills<D> * (NS - 2)>();
      else wait_barrier<0>();
      if (it + NS - 1 < tiles.n) fetch(it + NS - 1);
      const uint16_t *Ks = ring[it % NS][0], *Vs = ring[it % NS][1];
      if (wt0 > wt1) continue;
#pragma unroll 1
      for (int sub = 0; sub < 2; ++sub) {
        const int k0 = tiles.key(it) + 32 * sub;
        const int see = sight(k0, s.st + wt0, s.st + wt1, a.W, a.S);
        if (see == 0) continue;
        f32x16 x = zero16(), y = zero16();
#pragma unroll
        for (int ks = 0; ks < DK; ++ks) {
          x = E::mfma32(frag<D>(Ks, 32 * sub, ks, lane), qf[ks], x);
          y = E::mfma32(frag<D>(Vs, 32 * sub, ks, lane), df[ks], y);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float p = __builtin_amdgcn_exp2f(fmaf(x[r], a.c, -ls));
          if (see == 1) {
            const int j = k0 + row_of(r, lane);
            if (j > i || (i - j >= a.W && j >= a.S)) p = 0.f;
          }
          x[r] = p * (y[r] - ds);
        }
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          const u32x4 p = pack<E>(x, st);
#pragma unroll
          for (int dn = 0; dn < DN; ++dn)
            acc[dn] = E::mfma32(frag_t<D>(Ks, 32 * sub + 16 * st, dn, lane), p, acc[dn]);
        }
      }
    }
  }
  put_rows<E, D>(dq + ((int64_t)bh * a.Tq + t) * D, t < a.Tq, acc, valid ? scale : 0.f, lane);
  if (lane < 32) dsum[(int64_t)bh * nqb * BM + t] = valid ? ds : 0.f;
}

// dK, dV.  Two kinds of items:
// near: 128 keys, 32 a wave, with the queries that have them in their window;
// far: 32 keys, those of sinks, with `span` of the queries that have left their window behind (j < S,
// i - j >= W) -- pairs that would leave a few workgroups with the whole length.  The four waves take
// turns at the groups of 32 queries and their sums are added up in the end.
// The sums of rows j < S go to `part` [slot][b, hk][S][2][D] in 32 bits (slot 0: the near ones, then a
// slot for each span); window_sink_kernel adds the slots.
template <class E, int D>
struct Dkv {
  static constexpr int DK = D / 16, DN = D / 32, NS = kRing<D>;
  struct Lds {
    uint16_t ring[NS][2][BN * D];
    float stat[NS][2][BN];                             // log-sums, D
  };
  static constexpr float kUnshift = 1.f / (1 << E::kShift);   // (elt.h: p is 2^kShift times its value)
  const WinArgs& a;
  const uint16_t* dout;
  const float *lse, *dsum;
  Lds& lds;
  const Seq& s;
  int b, hk, tq_pad, tid, lane, wave;
  u32x4 kf[DK], vf[DK];
  f32x16 ak[DN], av[DN];

  // keys kw ... kw + 31 as B operands (zeros behind the sequence), accumulators cleared
  __device__ __forceinline__ void begin(int kw) {
    const int j = kw + (lane & 31);
#pragma unroll
    for (int dn = 0; dn < DN; ++dn) ak[dn] = av[dn] = zero16();
#pragma unroll
    for (int ks = 0; ks < DK; ++ks) {
      kf[ks] = vf[ks] = u32x4{0, 0, 0, 0};
      if (j < s.len) {
        const int col = 16 * ks + 8 * (lane >> 5);
        kf[ks] = *(const u32x4*)(a.k + b * a.k_sb + hk * a.k_sh + (int64_t)j * a.k_st + col);
        vf[ks] = *(const u32x4*)(a.v + b * a.v_sb + hk * a.v_sh + (int64_t)j * a.v_st + col);
      }
    }
  }

  // query tile it of `per` tiles a head, the first at row tb
  __device__ __forceinline__ void fetch(int it, int per, int tb) {
    const int G = a.H / a.KV, hq = hk * G + it / per, row0 = tb + (it % per) * BN, slot = it % NS;
    fill_tile<D>(a.q + b * a.q_sb + hq * a.q_sh, a.q_st, row0, s.t0, s.t1, lds.ring[slot][0], wave, lane);
    fill_tile<D>(dout + ((int64_t)b * a.Tq * a.H + hq) * D, (int64_t)a.H * D, row0, s.t0, s.t1,
                 lds.ring[slot][1], wave, lane);
    // (waves 2 and 3 write what waves 0 and 1 do: each has the same number of loads under way)
    fill4(((wave & 1) ? dsum : lse) + ((int64_t)b * a.H + hq) * tq_pad + row0 + lane, lds.stat[slot][wave & 1]);
  }

  // queries 32 sub ... of the tile against this wave's keys; ALL: every pair counts
  template <bool FAR>
  __device__ __forceinline__ void step(int slot, int sub, int p0, int kw, bool all) {
    const uint16_t *Qs = lds.ring[slot][0], *Os = lds.ring[slot][1];
    const float *ls = lds.stat[slot][0], *ds = lds.stat[slot][1];
    f32x16 x = zero16(), y = zero16();
#pragma unroll
    for (int ks = 0; ks < DK; ++ks) {
      x = E::mfma32(frag<D>(Qs, 32 * sub, ks, lane), kf[ks], x);
      y = E::mfma32(frag<D>(Os, 32 * sub, ks, lane), vf[ks], y);
    }
    const int j = kw + (lane & 31);
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const int q0 = row_of(4 * r4, lane);
      const f32x4 l4 = *(const f32x4*)(ls + 32 * sub + q0), d4 = *(const f32x4*)(ds + 32 * sub + q0);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 4 * r4 + e;
        float p = __builtin_amdgcn_exp2f(fmaf(x[r], a.c, (float)E::kShift - l4[e]));
        if (!all) {
          const int d = p0 + q0 + e - j;               // i - j
          if (FAR ? (j >= a.S || d < a.W) : (d < 0 || d >= a.W)) p = 0.f;
        }
        x[r] = p;
        y[r] = p * fmaf(d4[e], -kUnshift, y[r] * kUnshift);
      }
    }
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const u32x4 p = pack<E>(x, st), d = pack<E>(y, st);
#pragma unroll
      for (int dn = 0; dn < DN; ++dn) {
        av[dn] = E::mfma32(frag_t<D>(Os, 32 * sub + 16 * st, dn, lane), p, av[dn]);
        ak[dn] = E::mfma32(frag_t<D>(Qs, 32 * sub + 16 * st, dn, lane), d, ak[dn]);
      }
    }
  }

  // all tiles of rows [t0, t1) of every query head
  template <bool FAR>
  __device__ __forceinline__ void run(int kw, int t0, int t1) {
    const int tb = t0 & ~(BN - 1), per = (t1 - 1 - tb) / BN + 1, n = per * (a.H / a.KV);
    for (int it = 0; it < min(NS - 1, n); ++it) fetch(it, per, tb);
    for (int it = 0; it < n; ++it) {
      if (it + NS - 1 <= n) wait_barrier<(2 * kFills<D> + 1) * (NS - 2)>();
      else wait_barrier<0>();
      if (it + NS - 1 < n) fetch(it + NS - 1, per, tb);
      const int row0 = tb + (it % per) * BN;
      if (FAR) {
        if ((it & 1) != (wave >> 1)) continue;
        const int sub = wave & 1, p0 = s.st + row0 + 32 * sub;
        if (p0 + 31 - kw >= a.W) step<true>(it % NS, sub, p0, kw, kw + 31 < a.S && p0 - (kw + 31) >= a.W);
      } else {
#pragma unroll 1
        for (int sub = 0; sub < 2; ++sub) {
          const int p0 = s.st + row0 + 32 * sub;
          if (p0 + 31 < kw || p0 - (kw + 31) >= a.W) continue;
          step<false>(it % NS, sub, p0, kw, p0 >= kw + 31 && p0 + 31 - kw < a.W);
        }
      }
    }
  }

  __device__ __forceinline__ void put_part(float* dst) const {
#pragma unroll
    for (int dn = 0; dn < DN; ++dn)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const int col = 32 * dn + 8 * r4 + 4 * (lane >> 5);
        *(f32x4*)(dst + col) = f32x4{ak[dn][4 * r4], ak[dn][4 * r4 + 1], ak[dn][4 * r4 + 2], ak[dn][4 * r4 + 3]};
        *(f32x4*)(dst + D + col) = f32x4{av[dn][4 * r4], av[dn][4 * r4 + 1], av[dn][4 * r4 + 2], av[dn][4 * r4 + 3]};
      }
  }

  // x of the four waves added up in wave 0, in their order
  __device__ __forceinline__ void join(f32x16 (&x)[DN]) {
    float* buf = (float*)&lds;                         // 3 waves, 16 DN registers, 64 lanes
    __syncthreads();
    if (wave)
#pragma unroll
      for (int dn = 0; dn < DN; ++dn)
#pragma unroll
        for (int r = 0; r < 16; ++r) buf[(((wave - 1) * DN + dn) * 16 + r) * 64 + lane] = x[dn][r];
    __syncthreads();
    if (!wave)
      for (int w = 0; w < 3; ++w)
#pragma unroll
        for (int dn = 0; dn < DN; ++dn)
#pragma unroll
          for (int r = 0; r < 16; ++r) x[dn][r] += buf[((w * DN + dn) * 16 + r) * 64 + lane];
  }
};

template <class E, int D>
__global__ __launch_bounds__(256, kDkvWaves<D>) void window_dkv_kernel(WinArgs a, const uint16_t* dout, const float* lse,
                                                         const float* dsum, uint16_t* dk, uint16_t* dv,
                                                         float* part, int spans, int span, float scale) {
  using K = Dkv<E, D>;
  static_assert(sizeof(typename K::Lds) >= 3 * 64 * D / 2 * 4, "room to join the waves");
  __shared__ __attribute__((aligned(16))) typename K::Lds lds;
  const int nkb = (a.Tk + BM - 1) / BM;
  const int nst = spans ? (a.S + 31) / 32 : 0, items = nkb + nst * spans;
  const int item = xcd_remap((int)blockIdx.x, (int)gridDim.x);
  const int bk = item / items, it0 = item - bk * items, b = bk / a.KV, hk = bk - b * a.KV;
  const Seq s = seq_of(a, b);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  K k{a, dout, lse, dsum, lds, s, b, hk, (a.Tq + BM - 1) / BM * BM, tid, lane, wave};
  if (it0 < nst * spans) {
    const int c = it0 % spans, kw = it0 / spans * 32, j = kw + (lane & 31);
    const int t0 = (int)max((int64_t)max(s.t0, c * span), (int64_t)a.W + kw - s.st);
    const int t1 = (int)min((int64_t)s.t1, (int64_t)(c + 1) * span);
    k.begin(kw);
    if (t0 < t1 && kw < s.len) k.template run<true>(kw, t0, t1);
    k.join(k.ak);
    k.join(k.av);
    if (!wave && j < a.S) k.put_part(part + (((int64_t)(1 + c) * a.B * a.KV + bk) * a.S + j) * 2 * D);
    return;
  }
  const int kb = it0 - nst * spans, kw = kb * BM + wave * 32, j = kw + (lane & 31);
  // positions [kb BM, last key + W)
  const int t0 = max(s.t0, kb * BM - s.st);
  const int t1 = (int)min((int64_t)s.t1, (int64_t)kb * BM + BM - 1 + a.W - s.st);
  k.begin(kw);
  if (t0 < t1 && kb * BM < s.len) k.template run<false>(kw, t0, t1);
  const bool sink = spans && j < a.S;
  const int64_t row = ((int64_t)bk * a.Tk + j) * D;
  put_rows<E, D>(dk + row, j < a.Tk && !sink, k.ak, scale, lane);
  put_rows<E, D>(dv + row, j < a.Tk && !sink, k.av, K::kUnshift, lane);
  if (sink) k.put_part(part + ((int64_t)bk * a.S + j) * 2 * D);
}

// dk, dv rows j < min(S, Tk) from the slots of window_dkv_kernel, in their order
template <class E, int D>
__global__ __launch_bounds__(256) void window_sink_kernel(const float* part, int slots, int bks, int S, int Tk,
                                                          uint16_t* dk, uint16_t* dv, float scale) {
  constexpr int PER = D / 4;                           // threads of one row of one of dk, dv
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int c = (int)(u % PER) * 4, which = (int)(u / PER) & 1;
  const int64_t row = u / (2 * PER);
  if (row >= (int64_t)bks * S) return;
  const int bk = (int)(row / S), j = (int)(row - (int64_t)bk * S);
  if (j >= Tk) return;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < slots; ++i)
    v += *(const f32x4*)(part + (((int64_t)i * bks + bk) * S + j) * 2 * D + which * D + c);
  v *= which ? 1.f / (1 << E::kShift) : scale;
  *(uint2*)((which ? dv : dk) + ((int64_t)bk * Tk + j) * D + c) =
      make_uint2(E::pack2(v[0], v[1]), E::pack2(v[2], v[3]));
}

template <class E, int D>
int fwd(const WinArgs& a, void* o, void* rest, void* lse, hipStream_t st) {
  const int64_t n = (int64_t)((a.Tq + BM - 1) / BM) * a.B * a.H;
  if (n >= (1ll << 31)) return 1;
  hipLaunchKernelGGL((window_fwd_kernel<E, D>), dim3((unsigned)n), dim3(256), 0, st, a, (uint16_t*)o, (uint16_t*)rest,
                     (float*)lse);
  return (int)hipGetLastError();
}

template <class E, int D>
int bwd(const WinArgs& a, const void* o, const void* rest, const void* dout, const void* lse, void* dsum, void* dq, void* dk,
        void* dv, void* part, int spans, int span, float scale, hipStream_t st) {
  const int64_t n = (int64_t)((a.Tq + BM - 1) / BM) * a.B * a.H;
  const int64_t nk = ((int64_t)(a.Tk + BM - 1) / BM + (int64_t)((a.S + 31) / 32) * spans) *
                     a.B * a.KV;
  if (n >= (1ll << 31) || nk >= (1ll << 31)) return 1;
  hipLaunchKernelGGL((window_dq_kernel<E, D>), dim3((unsigned)n), dim3(256), 0, st, a, (const uint16_t*)o,
                     (const uint16_t*)rest, (const uint16_t*)dout, (const float*)lse, (float*)dsum, (uint16_t*)dq,
                     scale);
  hipLaunchKernelGGL((window_dkv_kernel<E, D>), dim3((unsigned)nk), dim3(256), 0, st, a, (const uint16_t*)dout,
                     (const float*)lse, (const float*)dsum, (uint16_t*)dk, (uint16_t*)dv, (float*)part, spans,
                     span, scale);
  if (spans) {
    const int64_t threads = (int64_t)a.B * a.KV * a.S * 2 * (D / 4);
    if ((threads + 255) / 256 >= (1ll << 31)) return 1;
    hipLaunchKernelGGL((window_sink_kernel<E, D>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st,
                       (const float*)part, 1 + spans, a.B * a.KV, a.S, a.Tk, (uint16_t*)dk, (uint16_t*)dv, scale);
  }
  return (int)hipGetLastError();
}

bool good(const WinArgs& a, int D) {
  return a.B > 0 && a.H > 0 && a.KV > 0 && a.H % a.KV == 0 && a.Tq > 0 && a.Tk > 0 && a.W > 0 && a.S >= 0 &&
         (D == 64 || D == 128) && a.Tq <= (1 << 29) && a.Tk <= (1 << 29) && a.W <= (1 << 30) &&
         a.S <= a.Tk && a.c > 0.f;
}

WinArgs args(const void* q, const void* k, const void* v, const int64_t* s, const void* start, const void* lengths,
             int start0, int B, int H, int KV, int Tq, int Tk, int W, int S, float scale) {
  return WinArgs{(const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v, s[0], s[1], s[2], s[3], s[4], s[5],
                 s[6], s[7], s[8], (const int32_t*)start, (const int32_t*)lengths, start0, B, H, KV, Tq, Tk, W, S,
                 scale * 1.4426950408889634f};
}

}  // namespace

extern "C" {

// dtype 0: bf16, 1: fp16.  strides: (batch, head, row) of q, k, v in elements; rows are contiguous
// and 16-byte aligned (checked by the caller).  o, rest: [B][Tq][H][D]; lse: [B][H][Tq rounded
// up to 128]; rest and lse (for the backward) or null.
int mopt_window_fwd(const void* q, const void* k, const void* v, const int64_t* strides, const void* start,
                    const void* lengths, int start0, void* o, void* rest, void* lse, int B, int H, int KV, int Tq, int Tk,
                    int D, int W, int S, float scale, int dtype, void* stream) {
  const WinArgs a = args(q, k, v, strides, start, lengths, start0, B, H, KV, Tq, Tk, W, S, scale);
  if (!good(a, D)) return 1;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == 0) return D == 64 ? fwd<Bf16, 64>(a, o, rest, lse, st) : fwd<Bf16, 128>(a, o, rest, lse, st);
  return D == 64 ? fwd<Fp16, 64>(a, o, rest, lse, st) : fwd<Fp16, 128>(a, o, rest, lse, st);
}

// dq [B][H][Tq][D], dk, dv [B][KV][Tk][D]; dsum: floats of workspace; part: workspace of
// (1 + spans) B KV S 2 D floats, spans * span >= Tq (spans 0: no sink is seen out of its window);
// lse, dsum: rows of Tq rounded up to 128
int mopt_window_bwd(const void* q, const void* k, const void* v, const int64_t* strides, const void* start,
                    const void* lengths, int start0, const void* o, const void* rest, const void* dout, const void* lse, void* dsum,
                    void* dq, void* dk, void* dv, void* part, int spans, int span, int B, int H, int KV, int Tq,
                    int Tk, int D, int W, int S, float scale, int dtype, void* stream) {
  const WinArgs a = args(q, k, v, strides, start, lengths, start0, B, H, KV, Tq, Tk, W, S, scale);
  if (!good(a, D) || spans < 0 || span <= 0 || span % BN || (spans && (!part || S == 0))) return 1;
  if (S && Tk > W && (int64_t)spans * span < Tq) return 1;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == 0)
    return D == 64 ? bwd<Bf16, 64>(a, o, rest, dout, lse, dsum, dq, dk, dv, part, spans, span, scale, st)
                   : bwd<Bf16, 128>(a, o, rest, dout, lse, dsum, dq, dk, dv, part, spans, span, scale, st);
  return D == 64 ? bwd<Fp16, 64>(a, o, rest, dout, lse, dsum, dq, dk, dv, part, spans, span, scale, st)
                 : bwd<Fp16, 128>(a, o, rest, dout, lse, dsum, dq, dk, dv, part, spans, span, scale, st);
}

}  // extern "C"
