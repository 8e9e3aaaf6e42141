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
// operands (two: see split8) of step s of the product with V -- P never leaves its lane.  V^T is read with the
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
__device__ __forceinline__ int lds_off(int r, int c) {      // element offset of (row, column)
  return r * D + (((c >> 3) ^ swz<D>(r)) << 3) + (c & 7);
}

__device__ __forceinline__ u32x4 lds16(const uint16_t* p) { return *(const u32x4*)p; }

__device__ __forceinline__ int swap23(int r) { return (r & 19) | ((r & 4) << 1) | ((r & 8) >> 1); }

typedef __attribute__((address_space(3))) void lds_void;
__device__ __forceinline__ uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)((lds_void*)p); }

// Fragments of a tile at LDS address `tile` (a multiple of 256).  A lane's place in the tile is kept
// in one register; columns change it by an exclusive or, rows by an offset of the instruction.
template <int D>
struct Place {
  uint32_t f, t, b;
  __device__ __forceinline__ explicit Place(int lane) {
    const int r = swap23(lane & 31), g = lane >> 4, i = lane & 15, q = 8 * (g >> 1) + (i >> 2);
    f = r * D * 2 + (((lane >> 5) ^ swz<D>(r)) << 4);
    b = (lane & 31) * D * 2 + (((lane >> 5) ^ swz<D>(lane & 31)) << 4);
    t = q * D * 2 + (((2 * (g & 1) + ((i & 3) >> 1)) ^ swz<D>(q)) << 4) + (i & 1) * 8;
  }
  // A operand of rows [r0, r0 + 32) (r0 a multiple of 32) in the exchanged order, columns 16 ks ...
  __device__ __forceinline__ u32x4 frag(uint32_t tile, int r0, int ks) const {
    typedef __attribute__((address_space(3))) const u32x4 vec;
    return *(vec*)(uintptr_t)(((tile + f) ^ (ks << 5)) + r0 * D * 2);
  }
  // B operand of step ks of the 32 rows of an image: this lane's row, columns 16 ks + 8 (l >> 5) ...
  __device__ __forceinline__ u32x4 frag_b(uint32_t image, int ks) const {
    typedef __attribute__((address_space(3))) const u32x4 vec;
    return *(vec*)(uintptr_t)((image + b) ^ (ks << 5));
  }
  // A operand of the transpose: rows = columns [32 dn, 32 dn + 32) of the tile, k = rows r0 ... + 15
  // (r0 a multiple of 16); rows 4 further have bit 0 of their exchange turned
  __device__ __forceinline__ u32x4 frag_t(uint32_t tile, int r0, int dn) const {
    const uint32_t p = (tile + t) ^ (dn << 6);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(p + r0 * D * 2));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)((p ^ 16) + (r0 + 4) * D * 2));
    return __builtin_bit_cast(u32x4, cat_frag(lo, hi));
  }
};

// Probabilities and score gradients, held in 32 bits, enter their products as two 16-bit pieces: rounded,
// and what that rounding left off.  One piece alone made o, dq, dk and dv up to 1.45 times as far from 64
// bits as outputs that are only rounded in the end; with two they are as near as these.  The price is a
// product more for each of P V, dS K, P^T dO and dS^T Q: forward 51 -> 64 us (4 x 12 heads of 64, 4096 tokens,
// window 512), 8192 tokens of 16 / 4 heads of 128, window 1024: 89 -> 112, dQ 123 -> 146, dK / dV 158 -> 206;
// 125M step (64 x 12 heads of 64, 512 tokens, window 128): 57 -> 60, 78 -> 82, 81 -> 92; a single token over
// a cache 14.8 -> 15.0, memory bounds that.  (Medians of 300 passes by the profiler, as all times here.)
struct Two {
  u32x4 hi, lo;
};
template <class E>
__device__ __forceinline__ Two split8(float a, float b, float c, float d, float e, float f, float g, float h) {
  Two t;
  t.hi = u32x4{E::pack2(a, b), E::pack2(c, d), E::pack2(e, f), E::pack2(g, h)};
  const f32x2_t r0 = E::less2(a, b, t.hi[0]), r1 = E::less2(c, d, t.hi[1]);
  const f32x2_t r2 = E::less2(e, f, t.hi[2]), r3 = E::less2(g, h, t.hi[3]);
  t.lo = u32x4{E::pack2(r0[0], r0[1]), E::pack2(r1[0], r1[1]), E::pack2(r2[0], r2[1]), E::pack2(r3[0], r3[1])};
  return t;
}
// registers 8 s ... 8 s + 7 of an accumulator as the B operand of step s
template <class E>
__device__ __forceinline__ Two pack(const f32x16& x, int s) {
  return split8<E>(x[8 * s], x[8 * s + 1], x[8 * s + 2], x[8 * s + 3], x[8 * s + 4], x[8 * s + 5], x[8 * s + 6],
                   x[8 * s + 7]);
}
template <class E>
__device__ __forceinline__ f32x16 mfma_both(const u32x4& a, const Two& b, f32x16 c) {
  return E::mfma32(a, b.lo, E::mfma32(a, b.hi, c));
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
// wait_barrier waits for those of the next tile itself.  Rows outside [lo, hi) are read as the nearest
// row inside (values of the sequence, finite as the others; the masks leave them out): what padding
// holds is never read.
__device__ __forceinline__ uint32_t lds_at(const void* p) { return __builtin_amdgcn_readfirstlane(lds_addr(p)); }
// base: the same for the whole wave; off: bytes, each lane's own.  (m0 is read a wait state after it is set.)
__device__ __forceinline__ const char* scalar(const void* p) {
  // (readfirstlane gives an int: the low half must not be extended by its sign)
  const uint64_t v = (uint64_t)p;
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)v);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (const char*)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ void fill16(const char* base, uint32_t off, const void* dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds_at(dst))
               : "memory");
}
__device__ __forceinline__ void fill4(const char* base, uint32_t off, const void* dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "s"(lds_at(dst))
               : "memory");
}

// until at most N of this wave's loads are under way, then until every wave is there
template <int N>
__device__ __forceinline__ void wait_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

template <int D, int ROWS = BN>
constexpr int kFills = ROWS * D * 2 / 1024 / 4;        // 1 KB fills of a tile by each of 4 waves

// A tile of rows row0 ... of a matrix.  Where each lane reads is kept for the tiles whose rows all lie
// inside [lo, hi): with the rows clamped one by one for every tile a fill was 25 vector instructions.
template <int D, int ROWS = BN>
struct Fill {
  static constexpr int N = kFills<D, ROWS>, CH = D / 8, PER = 64 / CH;   // chunks of a row, rows of a fill
  uint32_t off[N], row;                                // bytes from row0's start and of a row
  int wave, lane;
  __device__ __forceinline__ Fill(int64_t ld, int wave, int lane) : row((uint32_t)ld * 2), wave(wave), lane(lane) {
#pragma unroll
    for (int j = 0; j < N; ++j) off[j] = r(j) * row + c(j) * 16;
  }
  __device__ __forceinline__ int r(int j) const { return (wave * N + j) * PER + lane / CH; }
  __device__ __forceinline__ int c(int j) const { return (lane % CH) ^ swz<D>(r(j)); }
  __device__ __forceinline__ void tile(const uint16_t* g, int row0, int lo, int hi, uint16_t* img) const {
    const char* base = scalar((const char*)g + (int64_t)row0 * row);
    const int first = lo - row0, last = hi - 1 - row0;   // (last >= 0: a tile starts inside)
    if (first <= 0 && last >= ROWS - 1) {
#pragma unroll
      for (int j = 0; j < N; ++j) fill16(base, off[j], img + (wave * N + j) * 512);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        fill16(base, (uint32_t)max(first, min(last, r(j))) * row + c(j) * 16, img + (wave * N + j) * 512);
    }
  }
};

// waves a SIMD (registers: 512 / waves) and ring of a kernel (tiles of two matrices)
template <int D> constexpr int kDkvWaves = D == 64 ? 3 : 2;
template <int D> constexpr int kFwdWaves = D == 64 ? 4 : 2;
template <int D> constexpr int kDqWaves = D == 64 ? 3 : 2;
template <int D> constexpr int kFwdRing = 2;
template <int D> constexpr int kBwdRing = D == 64 ? 3 : 2;

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

// ------------------------------------------------------------------------------------ a wave's rows
// 32 rows of D values between memory and a wave's fragments go through an image in LDS that is the
// wave's own, so that memory is read and written in whole rows: fragments straight from memory touch
// 32 lines for 32 bytes each (125M step, dQ without any products: 94 us so, with a window of 1).
template <int D>
struct Rows {
  static constexpr int CH = D / 8, PER = 64 / CH, N = 32 / PER;   // chunks a row, rows a pass, passes
  static constexpr int SIZE = 32 * D;                              // elements of an image

  // rows row0 ... of a matrix; those outside [lo, hi) as the nearest inside
  static __device__ __forceinline__ void fill(const uint16_t* g, int64_t ld, int row0, int lo, int hi,
                                              uint16_t* img, int lane) {
    row0 = min(row0, hi - 1);                          // (a wave without a row inside)
    const char* base = scalar(g + row0 * ld);
    const int first = lo - row0, last = hi - 1 - row0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int r = j * PER + lane / CH, c = (lane % CH) ^ swz<D>(r);
      fill16(base, (uint32_t)max(first, min(last, r)) * ((uint32_t)ld * 2) + c * 16, img + j * 512);
    }
  }
  // the B operand of step ks: this lane's row, columns 16 ks + 8 (l >> 5) ...
  static __device__ __forceinline__ void read(const uint16_t* img, u32x4 (&f)[D / 16], int lane) {
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) f[ks] = lds16(img + lds_off<D>(lane & 31, 16 * ks + 8 * (lane >> 5)));
  }
  // acc * f, rounded, into rows row0 ... < hi of a matrix; with REST, what the rounding left off
  template <class E, bool REST>
  static __device__ __forceinline__ void put(const f32x16 (&acc)[D / 32], float f, uint16_t* g, int64_t ld,
                                             int row0, int lo, int hi, uint16_t* img, int lane) {
#pragma unroll
    for (int dn = 0; dn < D / 32; ++dn)
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        float x[2][4];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float v = acc[dn][8 * a + j] * f;
          x[j >> 2][j & 3] = REST ? v - E::up(E::pack2(v, v) & 0xFFFF) : v;
        }
        *(u32x4*)(img + lds_off<D>(lane & 31, 32 * dn + 16 * a + 8 * (lane >> 5))) = join_halves<E>(x[0], x[1]);
      }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int r = j * PER + lane / CH, c = lane % CH, row = row0 + r;
      const u32x4 w = lds16(img + lds_off<D>(r, c * 8));
      if (row >= lo && row < hi) *(u32x4*)(g + row * ld + c * 8) = w;
    }
  }
};

template <int N>
__device__ __forceinline__ void wait_own() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
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

// x of the keys k0 ... that the query at position i does not see: `with`
template <class E>
__device__ __forceinline__ void hide(f32x16& x, float with, int i, int k0, int lane, int W, int S) {
  const int d0 = i - k0 - 8 * (lane >> 5);
  if (k0 >= S) {
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = (uint32_t)(d0 - row_of(r, 0)) < (uint32_t)W ? x[r] : with;
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r)
      x[r] = (uint32_t)(d0 - row_of(r, 0)) < (k0 + row_of(r, lane) < S ? 1u << 31 : (uint32_t)W) ? x[r] : with;
  }
}

// Score gradients dS on their way into fp16.  Those of a mean loss over many tokens are far below 2^-14,
// where fp16 has multiples of 2^-24 only, and a fixed factor that lifts these lets others overflow.  So
// each row of a product (dQ: a query, dK: a key) carries a power of two of its own: dS comes multiplied by
// it, and where a row's largest passes 2^15 the factor, this group and the sums so far are brought down to
// put it at 2^7 ... 2^8.  A pair is then off by 2^-11 of itself or 2^-32 of its row's largest.  It starts at
// 2^60: products of fp16 rows (below 2^39) stay inside 32 bits with it.  It costs dQ 3 - 6 %, dK / dV 8 %.
constexpr float kFirstLift = (float)(1ull << 60);

// the factor that `x`, its row's sums and its lift take now (1, mostly)
template <class E>
__device__ __forceinline__ float settle(f32x16& x) {
  float mx = fabsf(x[0]);
#pragma unroll
  for (int r = 1; r < 16; ++r) mx = fmaxf(mx, fabsf(x[r]));
  mx = other_half(mx, true);
  if (!__any(mx > 32768.f)) return 1.f;
  const float f = mx > 32768.f ? __uint_as_float((261u - (__float_as_uint(mx) >> 23)) << 23) : 1.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) x[r] *= f;
  return f;
}

// Forward: one pass over the keys with a running reference and sum.  Bound by the vector work on the scores
// and the products, which hardly overlap: heads of 64 (4 sequences of 12 heads, 4096 tokens, window 512: 64
// us, passes back to back 57) keep the vector pipe busy for 47 % of the time and the matrix pipe for 27 %,
// heads of 128 (8192 tokens of 16 / 4 heads, window 1024: 112 us) both for 37 %.
template <class E, int D>
__global__ __launch_bounds__(256, kFwdWaves<D>) void window_fwd_kernel(WinArgs a, uint16_t* o, uint16_t* rest,
                                                                       float* lse) {
  constexpr int DK = D / 16, DN = D / 32, NS = kFwdRing<D>;
  __shared__ __attribute__((aligned(256))) uint16_t ring[NS][2][BN * D];
  const int nqb = (a.Tq + BM - 1) / BM;
  const int item = xcd_remap((int)blockIdx.x, (int)gridDim.x);
  const int qb = item % nqb, bh = item / nqb, b = bh / a.H, hq = bh - b * a.H;
  const int hk = hq / (a.H / a.KV);
  const Seq s = seq_of(a, b);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tw = qb * BM + wave * 32, t = tw + (lane & 31);   // the wave's first query, this lane's
  const bool valid = t >= s.t0 && t < s.t1;
  const int i = s.st + t;
  // valid queries of the block and of the wave
  const int bt0 = max(s.t0, qb * BM), bt1 = min(s.t1, qb * BM + BM) - 1;
  const int wt0 = max(s.t0, tw), wt1 = min(s.t1, tw + 32) - 1;

  const Place<D> at(lane);
  f32x16 acc[DN];
#pragma unroll
  for (int dn = 0; dn < DN; ++dn) acc[dn] = zero16();
  float m = -3e38f, l = 0.f;
  // the wave's image, in the slot that is filled last
  uint16_t* img = ring[0][0] + wave * Rows<D>::SIZE;
  if (bt0 <= bt1) {
    const uint16_t* kg = a.k + b * a.k_sb + hk * a.k_sh;
    const uint16_t* vg = a.v + b * a.v_sb + hk * a.v_sh;
    const Tiles tiles(s.st + bt0, s.st + bt1, a.W, a.S);
    // (slot of tile 0: 1)
    const Fill<D> kfill(a.k_st, wave, lane), vfill(a.v_st, wave, lane);
    auto fetch = [&](int it) {
      kfill.tile(kg, tiles.key(it), 0, s.len, ring[(it + 1) % NS][0]);
      vfill.tile(vg, tiles.key(it), 0, s.len, ring[(it + 1) % NS][1]);
    };
    Rows<D>::fill(a.q + b * a.q_sb + hq * a.q_sh, a.q_st, tw, s.t0, s.t1, img, lane);
    for (int it = 0; it < min(NS - 1, tiles.n); ++it) fetch(it);
    if (tiles.n >= NS - 1) wait_own<2 * kFills<D> * (NS - 1)>();
    else wait_own<0>();
    u32x4 qf[DK];
    Rows<D>::read(img, qf, lane);
    for (int it = 0; it < tiles.n; ++it) {
      if (it + NS - 1 <= tiles.n) wait_barrier<2 * kFills<D> * (NS - 2)>();
      else wait_barrier<0>();
      if (it + NS - 1 < tiles.n) fetch(it + NS - 1);
      const uint32_t Ks = lds_at(ring[(it + 1) % NS][0]), Vs = lds_at(ring[(it + 1) % NS][1]);
      if (wt0 > wt1) continue;
      // products of the scores of a group of 32 keys, their maximum, their exponentials and P V
      auto scores = [&](int sub) {
        f32x16 x = zero16();
#pragma unroll
        for (int ks = 0; ks < DK; ++ks) x = E::mfma32(at.frag(Ks + sub * 64 * D, 0, ks), qf[ks], x);
        return x;
      };
      auto most = [&](const f32x16& x) {
        float mx = x[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, x[r]);
        return mx;
      };
      // the reference of the exponents moves only when a row's maximum has grown past 2^8 of it:
      // sums and products stay far inside 32 bits, and most tiles need no rescaling
      auto refer = [&](float mx) {
        mx = other_half(mx, true) * a.c;
        if (__any(mx > m + 8.f)) {
          const float mn = fmaxf(m, mx), f = __builtin_amdgcn_exp2f(m - mn);
          m = mn;
          l *= f;
#pragma unroll
          for (int dn = 0; dn < DN; ++dn) acc[dn] *= f;
        }
      };
      auto weigh = [&](f32x16& x, int sub) {
        float part = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          x[r] = __builtin_amdgcn_exp2f(fmaf(x[r], a.c, -m));
          part += x[r];
        }
        l += part;
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          const Two p = pack<E>(x, st);
#pragma unroll
          for (int dn = 0; dn < DN; ++dn)
            acc[dn] = mfma_both<E>(at.frag_t(Vs + sub * 64 * D, 16 * st, dn), p, acc[dn]);
        }
      };
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        const int k0 = tiles.key(it) + 32 * sub, see = sight(k0, s.st + wt0, s.st + wt1, a.W, a.S);
        if (see == 0) continue;
        f32x16 x = scores(sub);
        if (see == 1) hide<E>(x, -INFINITY, i, k0, lane, a.W, a.S);
        refer(most(x));
        weigh(x, sub);
      }
    }
  }
  l = other_half(l, false);
  const bool some = valid && l > 0.f;
  const float f = some ? 1.f / l : 0.f;
  const int64_t ld = (int64_t)a.H * D, base = ((int64_t)b * a.Tq * a.H + hq) * D;
  __syncthreads();                                     // (the tiles have been read)
  Rows<D>::template put<E, false>(acc, f, o + base, ld, tw, 0, a.Tq, img, lane);
  if (rest) Rows<D>::template put<E, true>(acc, f, rest + base, ld, tw, 0, a.Tq, img, lane);
  if (lse && lane < 32) lse[(int64_t)bh * nqb * BM + t] = some ? m + log2f(l) : INFINITY;
}

// dQ, and D of its rows for the dK / dV kernel.  D is formed from o and what o's rounding left off
// (`rest`, written by the forward): with o alone its error adds to that of the rounded dS, and where
// few keys are seen it is the larger one (a window of 4: 1.8 times the error of a once rounded dq
// instead of 1.5, with dS in one piece).  125M step (64 x 12 heads, 512 tokens, window 128): 82 us, of which
// reading and writing 356 MB is 66; heads of 128, 8192 tokens, window 1024: 146 us, the matrix pipe busy for
// 38 % of it, the vector pipe for 31 %.
template <class E, int D>
__global__ __launch_bounds__(256, kDqWaves<D>) void window_dq_kernel(WinArgs a, const uint16_t* o,
                                                                     const uint16_t* rest, const uint16_t* dout,
                                                                     const float* lse, float* dsum, uint16_t* dq,
                                                                     float scale) {
  constexpr int DK = D / 16, DN = D / 32, NS = kBwdRing<D>, CH = Rows<D>::CH, PER = Rows<D>::PER;
  __shared__ __attribute__((aligned(256))) uint16_t ring[NS][2][BN * D];
  __shared__ float ds_s[BM];
  const int nqb = (a.Tq + BM - 1) / BM;
  const int item = xcd_remap((int)blockIdx.x, (int)gridDim.x);
  const int qb = item % nqb, bh = item / nqb, b = bh / a.H, hq = bh - b * a.H;
  const int hk = hq / (a.H / a.KV);
  const Seq s = seq_of(a, b);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tw = qb * BM + wave * 32, t = tw + (lane & 31);
  const bool valid = t >= s.t0 && t < s.t1;
  const int i = s.st + t;
  const int bt0 = max(s.t0, qb * BM), bt1 = min(s.t1, qb * BM + BM) - 1;
  const int wt0 = max(s.t0, tw), wt1 = min(s.t1, tw + 32) - 1;

  const Place<D> at(lane);
  f32x16 acc[DN];
#pragma unroll
  for (int dn = 0; dn < DN; ++dn) acc[dn] = zero16();
  float ds = 0.f, lift = E::kShift ? kFirstLift : 1.f;
  uint16_t* img = ring[0][0] + wave * Rows<D>::SIZE;
  if (bt0 <= bt1) {
    const uint16_t* kg = a.k + b * a.k_sb + hk * a.k_sh;
    const uint16_t* vg = a.v + b * a.v_sb + hk * a.v_sh;
    const Tiles tiles(s.st + bt0, s.st + bt1, a.W, a.S);
    const Fill<D> kfill(a.k_st, wave, lane), vfill(a.v_st, wave, lane);
    auto fetch = [&](int it) {
      kfill.tile(kg, tiles.key(it), 0, s.len, ring[(it + 1) % NS][0]);
      vfill.tile(vg, tiles.key(it), 0, s.len, ring[(it + 1) % NS][1]);
    };
    Rows<D>::fill(a.q + b * a.q_sb + hq * a.q_sh, a.q_st, tw, s.t0, s.t1, img, lane);
    const float ls = lse[(int64_t)bh * nqb * BM + t];
    // D of the wave's rows, from whole rows of do, o and its rest; do goes into the image behind q
    const int64_t ld = (int64_t)a.H * D, base = ((int64_t)b * a.Tq * a.H + hq) * D;
    u32x4 dr[Rows<D>::N];
#pragma unroll
    for (int j = 0; j < Rows<D>::N; ++j) {
      const int r = j * PER + lane / CH;
      const int64_t e = base + max(s.t0, min(s.t1 - 1, tw + r)) * ld + (lane % CH) * 8;
      dr[j] = *(const u32x4*)(dout + e);
      float x[8], y[8], z[8], part = 0.f;
      up8<E>(dr[j], x);
      up8<E>(*(const u32x4*)(o + e), y);
      up8<E>(*(const u32x4*)(rest + e), z);
#pragma unroll
      for (int n = 0; n < 8; ++n) part = fmaf(x[n], y[n] + z[n], part);
#pragma unroll
      for (int m = 1; m < CH; m <<= 1) part += __shfl_xor(part, m, 64);
      if (lane % CH == 0) ds_s[wave * 32 + r] = part;
    }
    for (int it = 0; it < min(NS - 1, tiles.n); ++it) fetch(it);
    // (the q rows and everything before them: the loads of D above have waited for later ones)
    u32x4 qf[DK], df[DK];
    if (tiles.n >= NS - 1) wait_own<2 * kFills<D> * (NS - 1)>();
    else wait_own<0>();
    Rows<D>::read(img, qf, lane);
#pragma unroll
    for (int j = 0; j < Rows<D>::N; ++j)
      *(u32x4*)(img + lds_off<D>(j * PER + lane / CH, (lane % CH) * 8)) = dr[j];
    Rows<D>::read(img, df, lane);
    ds = ds_s[wave * 32 + (lane & 31)];
    for (int it = 0; it < tiles.n; ++it) {
      if (it + NS - 1 <= tiles.n) wait_barrier<2 * kFills<D> * (NS - 2)>();
      else wait_barrier<0>();
      if (it + NS - 1 < tiles.n) fetch(it + NS - 1);
      const uint32_t Ks = lds_at(ring[(it + 1) % NS][0]), Vs = lds_at(ring[(it + 1) % NS][1]);
      if (wt0 > wt1) continue;
      auto scores = [&](int sub, f32x16& x, f32x16& y) {
        x = y = zero16();
#pragma unroll
        for (int ks = 0; ks < DK; ++ks) {
          x = E::mfma32(at.frag(Ks + sub * 64 * D, 0, ks), qf[ks], x);
          y = E::mfma32(at.frag(Vs + sub * 64 * D, 0, ks), df[ks], y);
        }
      };
      auto slope = [&](f32x16& x, const f32x16& y) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          x[r] = __builtin_amdgcn_exp2f(fmaf(x[r], a.c, -ls)) * (E::kShift ? fmaf(y[r], lift, -ds * lift) : y[r] - ds);
      };
      auto add = [&](const f32x16& x, int sub) {
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          const Two p = pack<E>(x, st);
#pragma unroll
          for (int dn = 0; dn < DN; ++dn)
            acc[dn] = mfma_both<E>(at.frag_t(Ks + sub * 64 * D, 16 * st, dn), p, acc[dn]);
        }
      };
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        const int k0 = tiles.key(it) + 32 * sub, see = sight(k0, s.st + wt0, s.st + wt1, a.W, a.S);
        if (see == 0) continue;
        f32x16 x, y;
        scores(sub, x, y);
        slope(x, y);
        if (see == 1) hide<E>(x, 0.f, i, k0, lane, a.W, a.S);
        if constexpr (E::kShift) {
          const float f = settle<E>(x);
          if (__any(f != 1.f)) {
            lift *= f;
#pragma unroll
            for (int dn = 0; dn < DN; ++dn) acc[dn] *= f;
          }
        }
        add(x, sub);
      }
    }
  }
  __syncthreads();
  Rows<D>::template put<E, false>(acc, valid ? scale / lift : 0.f, dq + (int64_t)bh * a.Tq * D, D, tw, 0, a.Tq, img, lane);
  if (lane < 32) dsum[(int64_t)bh * nqb * BM + t] = valid ? ds : 0.f;
}

// v in three bf16 pieces (24 bits), as the row of an A operand that holds them in its first columns and
// zeros behind; lanes l >= 32, later columns, all zeros
__device__ __forceinline__ u32x4 pieces(float v, int lane) {
  v = lane < 32 ? fminf(fmaxf(v, -3e38f), 3e38f) : 0.f;
  const uint32_t a = Bf16::pack2(v, 0.f);
  const float v1 = v - Bf16::up(a);
  const uint32_t b = Bf16::pack2(v1, 0.f);
  return u32x4{a | b << 16, Bf16::pack2(v1 - Bf16::up(b), 0.f), 0, 0};
}

// dK, dV.  Two kinds of items:
// near: 128 keys, 32 a wave, with the queries that have them in their window, or one of `parts` shares
// of these;
// far: 32 keys, those of sinks, with `span` of the queries that have left their window behind (j < S,
// i - j >= W) -- pairs that would leave a few workgroups with the whole length.  The four waves take
// turns at the groups of 32 queries.
// What is not a key's whole sum is left in 32 bits: the near sums of all rows (parts > 1) or of rows
// j < S, [part][b, hk][rows][2][D], and the far ones behind them, [span][wave][b, hk][S][2][D];
// window_sum_kernel adds them.  125M step (64 x 12 heads, 512 tokens, window 128, 4 sinks): 92 us, of which
// reading and writing 397 MB is 74; 8192 tokens of 16 / 4 heads, window 1024: heads of 64 124 us, of 128 206
// us, the matrix pipe busy for 42 % of it, the vector pipe for 29 % (six such sequences 1171: 195 each).
// (Two waves for each key, 8 a workgroup, were nearly 3 times slower.)
template <class E, int D>
struct Dkv {
  // heads of 128: 64 registers of key and value fragments beside 128 of sums leave too few for the
  // rest; the values stay in LDS, and tiles of 32 queries make room for them
  static constexpr bool kValuesInLds = D == 128;
  static constexpr int DK = D / 16, DN = D / 32, NS = kBwdRing<D>, QN = D == 128 ? 32 : BN, SUBS = QN / 32;
  struct Lds {
    uint16_t ring[NS][2][QN * D];
    uint16_t values[kValuesInLds ? BM * D : 8];
    float stat[NS][2][64];                             // log-sums, D
  };
  static constexpr float kUnshift = 1.f / (1 << E::kShift);   // (elt.h: p is 2^kShift times its value)
  const WinArgs& a;
  const uint16_t* dout;
  const float *lse, *dsum;
  Lds& lds;
  const Seq& s;
  float rc;                                            // 1 / c
  int b, hk, tq_pad, lane, wave;
  Place<D> at;
  Fill<D, QN> qfill, ofill;
  u32x4 kf[DK], vf[kValuesInLds ? 1 : DK];
  f32x16 ak[DN], av[DN];
  float lift;                                          // of this lane's key, over 2^kShift; fp16

  __device__ __forceinline__ void clear() {
    lift = kFirstLift * kUnshift;
#pragma unroll
    for (int dn = 0; dn < DN; ++dn) ak[dn] = av[dn] = zero16();
  }

  // Where the next tile is read from: its row, and the first head's matrices and rows of statistics;
  // kept and moved on tile by tile (a division by the tiles of a head, twice a tile, and 64-bit
  // products were as many scalar instructions as the step has vector ones)
  const uint16_t *qn, *on;
  const float* sn;
  int row_n, slot_n;

  __device__ __forceinline__ void fetch(int tb, int te) {
    qfill.tile(qn, row_n, s.t0, s.t1, lds.ring[slot_n][0]);
    ofill.tile(on, row_n, s.t0, s.t1, lds.ring[slot_n][1]);
    // (waves 2 and 3 write what waves 0 and 1 do: each has the same number of loads under way)
    fill4(scalar(sn + row_n), 4 * (lane & (QN - 1)), lds.stat[slot_n][wave & 1]);
    slot_n = slot_n + 1 == NS ? 0 : slot_n + 1;
    row_n += QN;
    if (row_n >= te) {                                 // the next head's first tile
      row_n = tb;
      qn += a.q_sh;
      on += D;
      sn += tq_pad;
    }
  }

  // what takes the lift off ak
  __device__ __forceinline__ float plain() const { return E::kShift ? kUnshift / lift : 1.f; }

  // Tiles [it0, it1) of those of rows [tb, te) of each query head, for the pairs with
  // lo <= i - j < lo + n: the window's (0, W), or far ones (W, as many as there may be; j < S)
  __device__ __forceinline__ void run(bool far, int kw, int tb, int te, int it0, int it1) {
    constexpr int kTile = 2 * kFills<D, QN> + 1;
    const int per = (te - 1 - tb) / QN + 1, skip = it0 / per, hq = hk * (a.H / a.KV) + skip;
    int row0 = tb + (it0 - skip * per) * QN, slot = NS == 3 ? 2 : 0;
    row_n = row0;
    slot_n = slot;
    qn = a.q + b * a.q_sb + hq * a.q_sh;
    on = dout + ((int64_t)b * a.Tq * a.H + hq) * D;
    sn = ((wave & 1) ? dsum : lse) + ((int64_t)b * a.H + hq) * tq_pad;
    // the wave's keys and values: slots 0 and 1 of three; heads of 128: both slots, and the
    // values' place
    uint16_t* img = lds.ring[0][0] + wave * Rows<D>::SIZE;
    uint16_t* vimg = kValuesInLds ? lds.values + wave * Rows<D>::SIZE : img + 4 * Rows<D>::SIZE;
    Rows<D>::fill(a.k + b * a.k_sb + hk * a.k_sh, a.k_st, kw, 0, s.len, img, lane);
    Rows<D>::fill(a.v + b * a.v_sb + hk * a.v_sh, a.v_st, kw, 0, s.len, vimg, lane);
    int issued = it0;
    if (NS == 3) {                                     // (a tile goes into the third slot)
      fetch(tb, te), ++issued;
      wait_own<kTile>();
    } else {
      wait_own<0>();
    }
    Rows<D>::read(img, kf, lane);
    if constexpr (!kValuesInLds) Rows<D>::read(vimg, vf, lane);
    if (NS == 2) {
      wait_barrier<0>();
      fetch(tb, te), ++issued;
    }
    const int j = kw + (lane & 31), lo = far ? a.W : 0;
    const uint32_t n = far ? 1u << 30 : (uint32_t)a.W, mine = far && j >= a.S ? 0 : n;
    for (int it = it0; it < it1; ++it) {
      if (issued - it - 1 == NS - 2) wait_barrier<kTile * (NS - 2)>();
      else wait_barrier<0>();
      while (issued < min(it1, it + NS)) fetch(tb, te), ++issued;
#pragma unroll 1
      for (int sub = 0; sub < SUBS; ++sub) {
        if (far && ((it * SUBS + sub) & 3) != wave) continue;
        const int least = s.st + row0 + 32 * sub - kw - 31;   // of i - j; the largest is 62 more
        if (least + 62 < lo || (least >= lo && (uint32_t)(least - lo) >= n)) continue;
        const bool all = least >= lo && (uint32_t)(least + 62 - lo) < n && (!far || kw + 31 < a.S);
        step(slot, sub, all, least + 31 + kw - j - lo, mine);
      }
      slot = slot + 1 == NS ? 0 : slot + 1;
      row0 = row0 + QN >= te ? tb : row0 + QN;
    }
  }

  // queries 32 sub ... of the tile against this wave's keys.  d0: i - j - lo of the first query and
  // this lane's key, pairs with values of [0, mine) count (all: every pair does)
  __device__ __forceinline__ void step(int slot, int sub, bool all, int d0, uint32_t mine) {
    const uint32_t Qs = lds_at(lds.ring[slot][0]) + sub * 64 * D, Os = lds_at(lds.ring[slot][1]) + sub * 64 * D;
    // Both products start at what their rows' sums take off: a value of each row in three pieces, times
    // ones.  (From LDS to the registers that need them the 2 x 16 values would be 8 reads of 1 KB, 12 % of
    // the time of heads of 64.)
    const int own = 32 * sub + swap23(lane & 31);
    const u32x4 ones = {0x3F803F80, 0x3F803F80, 0x3F803F80, 0x3F803F80};
    f32x16 x = Bf16::mfma32(pieces(-lds.stat[slot][0][own] * rc, lane), ones, zero16());
    f32x16 y = Bf16::mfma32(pieces(-lds.stat[slot][1][own], lane), ones, zero16());
#pragma unroll
    for (int ks = 0; ks < DK; ++ks) x = E::mfma32(at.frag(Qs, 0, ks), kf[ks], x);
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = __builtin_amdgcn_exp2f(E::kShift ? fmaf(x[r], a.c, (float)E::kShift) : x[r] * a.c);
    if (!all) {
      const int d = d0 + 8 * (lane >> 5);
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = (uint32_t)(d + row_of(r, 0)) < mine ? x[r] : 0.f;
    }
    if (D == 128) __builtin_amdgcn_sched_barrier(0);
    // (opaque: the places of the values would be kept over the loop, in 8 registers that it needs)
    uint32_t values = lds_at(lds.values) + wave * Rows<D>::SIZE * 2;
    asm volatile("" : "+v"(values));
#pragma unroll
    for (int ks = 0; ks < DK; ++ks)
      y = E::mfma32(at.frag(Os, 0, ks), kValuesInLds ? at.frag_b(values, ks) : vf[kValuesInLds ? 0 : ks], y);
    if constexpr (D == 128) {                          // reads two products ahead, not all at once
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
      for (int ks = 0; ks < DK - 2; ++ks) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x8, 2, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) y[r] *= E::kShift ? x[r] * lift : x[r];
    if constexpr (E::kShift) {
      const float f = settle<E>(y);
      if (__any(f != 1.f)) {
        lift *= f;
#pragma unroll
        for (int dn = 0; dn < DN; ++dn) ak[dn] *= f;
      }
    }
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const Two p = pack<E>(x, st);
#pragma unroll
      for (int dn = 0; dn < DN; ++dn) av[dn] = mfma_both<E>(at.frag_t(Os, 16 * st, dn), p, av[dn]);
    }
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const Two d = pack<E>(y, st);
#pragma unroll
      for (int dn = 0; dn < DN; ++dn) ak[dn] = mfma_both<E>(at.frag_t(Qs, 16 * st, dn), d, ak[dn]);
    }
  }

  __device__ __forceinline__ void put_part(float* dst) const {
    const float f = plain();
#pragma unroll
    for (int dn = 0; dn < DN; ++dn)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const int col = 32 * dn + 8 * r4 + 4 * (lane >> 5);
        const f32x4 k4 = {ak[dn][4 * r4], ak[dn][4 * r4 + 1], ak[dn][4 * r4 + 2], ak[dn][4 * r4 + 3]};
        *(f32x4*)(dst + col) = E::kShift ? k4 * f : k4;
        *(f32x4*)(dst + D + col) = f32x4{av[dn][4 * r4], av[dn][4 * r4 + 1], av[dn][4 * r4 + 2], av[dn][4 * r4 + 3]};
      }
  }
};

template <class E, int D>
__global__ __launch_bounds__(256, kDkvWaves<D>) void window_dkv_kernel(
    WinArgs a, const uint16_t* dout, const float* lse, const float* dsum, uint16_t* dk, uint16_t* dv, float* part,
    int parts, int spans, int span, float scale) {
  using K = Dkv<E, D>;
  constexpr int QN = K::QN;
  __shared__ __attribute__((aligned(256))) typename K::Lds lds;
  const int nkb = (a.Tk + BM - 1) / BM * parts;
  // far items come first and go round the XCDs, near ones lie together by key head (a multiple of 8
  // before them): each XCD gets its share of both
  const int nfar = spans ? (a.S + 31) / 32 * spans : 0, fars = nfar * a.B * a.KV, first = (fars + 7) & ~7;
  if ((int)blockIdx.x >= fars && (int)blockIdx.x < first) return;
  const bool far = (int)blockIdx.x < fars;
  const int item = far ? (int)blockIdx.x : xcd_remap((int)blockIdx.x - first, (int)gridDim.x - first);
  const int bk = item / (far ? nfar : nkb), it0 = item - bk * (far ? nfar : nkb), b = bk / a.KV, hk = bk - b * a.KV;
  const Seq s = seq_of(a, b);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  K k{a, dout, lse, dsum, lds, s, 1.f / a.c, b, hk, (a.Tq + BM - 1) / BM * BM, lane, wave, Place<D>(lane),
      Fill<D, K::QN>(a.q_st, wave, lane), Fill<D, K::QN>((int64_t)a.H * D, wave, lane)};
  const int G = a.H / a.KV, c = it0 % (far ? spans : parts);
  const int kb = it0 / parts, kw = far ? it0 / spans * 32 : kb * BM + wave * 32;
  const int j = kw + (lane & 31);
  // near: queries of positions [kb BM, last key + W)
  int t0 = max(s.t0, kb * BM - s.st);
  int t1 = (int)min((int64_t)s.t1, (int64_t)kb * BM + BM - 1 + a.W - s.st);
  if (far) {
    t0 = max(max(s.t0, c * span), a.W + kw - s.st);
    t1 = (int)min((int64_t)s.t1, (int64_t)(c + 1) * span);
  }
  k.clear();
  if (t0 < t1 && (far ? kw : kb * BM) < s.len) {
    const int tb = t0 & ~(QN - 1), per = (t1 - 1 - tb) / QN + 1, tiles = per * G;
    const int share = far ? tiles : (tiles + parts - 1) / parts, it = far ? 0 : c * share;
    if (it < tiles) k.run(far, kw, tb, t1, it, min(tiles, it + share));
  }
  const int64_t bks = (int64_t)a.B * a.KV, rows = parts > 1 ? a.Tk : a.S;
  if (far) {
    if (j < a.S) k.put_part(part + (parts * bks * rows + ((c * 4 + wave) * bks + bk) * a.S + j) * 2 * D);
    return;
  }
  __syncthreads();
  uint16_t* img = lds.ring[0][0] + wave * Rows<D>::SIZE;
  const bool some = parts > 1 || (spans && j < a.S);    // what window_sum_kernel adds up
  if (parts == 1) {
    const int64_t base = (int64_t)bk * a.Tk * D;
    const int lo = spans ? a.S : 0;
    Rows<D>::template put<E, false>(k.ak, scale * k.plain(), dk + base, D, kw, lo, a.Tk, img, lane);
    Rows<D>::template put<E, false>(k.av, K::kUnshift, dv + base, D, kw, lo, a.Tk, img, lane);
  }
  if (some && j < a.Tk) k.put_part(part + ((c * bks + bk) * rows + j) * 2 * D);
}

// dk, dv of the first `rows` rows of each key head, from what window_dkv_kernel left.  Each of the first
// `wide` rows (the sinks, where they have many sums) takes a workgroup that adds them in slices (256 sums
// of 4 rows: 14 us with the others, one after another 23; 4 sums of 70 rows of 768 heads: 67, so 31), each
// 4 columns of the other rows a thread.
template <class E, int D>
__global__ __launch_bounds__(256) void window_sum_kernel(const float* part, int parts, int spans, int64_t bks, int rows,
                                                         int S, int wide, int Tk, uint16_t* dk, uint16_t* dv,
                                                         float scale) {
  constexpr int PER = 2 * D / 4, SL = 256 / PER;       // threads of a row of both, slices of a workgroup
  __shared__ f32x4 slices[SL][PER];
  const int c = threadIdx.x % PER, sl = threadIdx.x / PER, which = c / (PER / 2), col = c % (PER / 2) * 4;
  const bool slice = blockIdx.x < bks * wide;
  const int64_t u = slice ? blockIdx.x : (blockIdx.x - bks * wide) * SL + sl;
  const int per = slice ? wide : rows - wide, first = slice ? sl : 0, by = slice ? SL : 1;
  if (u >= bks * per) return;                          // (never of a slice)
  const int64_t bk = u / per;
  const int j = (int)(u - bk * per) + (slice ? 0 : wide);
  const float* p = part + c * 4;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = first; i < parts; i += by) v += *(const f32x4*)(p + ((i * bks + bk) * rows + j) * 2 * D);
  if (j < S)
#pragma unroll 8
    for (int i = first; i < 4 * spans; i += by)
      v += *(const f32x4*)(p + (parts * bks * rows + (i * bks + bk) * S + j) * 2 * D);
  if (slice) {
    slices[sl][c] = v;
    __syncthreads();
    if (sl) return;
    for (int i = 1; i < SL; ++i) v += slices[i][c];
  }
  v *= which ? 1.f / (1 << E::kShift) : scale;
  *(uint2*)((which ? dv : dk) + (bk * Tk + j) * D + col) = make_uint2(E::pack2(v[0], v[1]), E::pack2(v[2], v[3]));
}

// ------------------------------------------------------------------------------------ few queries
// Forward for at most 16 rows of (query head of one key head, token): one token of a cache, mostly.
// What counts there is that the keys and values are read once at full rate, so a workgroup is 8 waves
// that go through the keys 32 at a time on their own -- keys from memory into registers as operands,
// values into LDS for the transposing read, both a chunk ahead -- and join their maxima, sums and
// products in the end.  With `splits` > 1 the keys of a head are shared among that many workgroups,
// which leave theirs in `part`, and window_join_kernel joins them.  32768 keys of 8 heads of 128: 25.2 us
// (5.3 TB/s) and 4 for joining.
// Products are 16x16x32: lane l holds A[l & 15][8 (l >> 4) ..], B[8 (l >> 4) ..][l & 15] and
// C[4 (l >> 4) + r][l & 15]; the keys of the two score tiles of a chunk are fed so that a lane's
// 4 + 4 scores are those of keys 8 (l >> 4) ... + 7, the B operand of the product with V.
constexpr int NW = 8;          // (64 sequences of 4 key heads of 64, 1028 keys: 15.0 us, with 16 waves 10 % more)

__device__ __forceinline__ float over_groups(float v, bool mx) {      // lanes l, l ^ 16, l ^ 32, l ^ 48
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const float a = __uint_as_float(p[0]), b = __uint_as_float(p[1]);
  return other_half(mx ? fmaxf(a, b) : a + b, mx);
}

template <class E, int D>
__global__ __launch_bounds__(NW * 64) void window_step_kernel(WinArgs a, uint16_t* o, float* part, int splits) {
  constexpr int DK = D / 32, DT = D / 16;
  __shared__ __attribute__((aligned(256))) uint16_t vs[NW][2][32 * D];
  __shared__ float stat[2][NW][16];
  const int G = a.H / a.KV, rows = G * a.Tq;
  const int bk = blockIdx.x / splits, split = blockIdx.x - bk * splits, b = bk / a.KV, hk = bk - b * a.KV;
  const Seq s = seq_of(a, b);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 15, g = lane >> 4;
  const int t = li % a.Tq, hq = hk * G + li / a.Tq;            // this lane's row
  const bool valid = li < rows && t >= s.t0 && t < s.t1;
  const int i = valid ? s.st + t : -1;

  f32x4 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x4{0, 0, 0, 0};
  float m = -3e38f, l = 0.f;
  if (s.t0 < s.t1) {
    const uint16_t* kg = a.k + b * a.k_sb + hk * a.k_sh;
    const uint16_t* vg = a.v + b * a.v_sb + hk * a.v_sh;
    u32x4 qf[DK];
#pragma unroll
    for (int ks = 0; ks < DK; ++ks) {
      qf[ks] = u32x4{0, 0, 0, 0};
      if (valid) qf[ks] = *(const u32x4*)(a.q + b * a.q_sb + hq * a.q_sh + (int64_t)t * a.q_st + 32 * ks + 8 * g);
    }
    // chunks of 32 keys: sinks in front of the window, then the window; this workgroup's share
    const int low = max(0, s.st + s.t0 - a.W + 1) & ~31, last = s.st + s.t1 - 1;
    const int sinks = (min(a.S, low) + 31) / 32, n = sinks + (last - low) / 32 + 1;
    const int per = (n + splits - 1) / splits, end = min(n, (split + 1) * per);
    auto key = [&](int c) { return 32 * (c < sinks ? c : c - sinks) + (c < sinks ? 0 : low); };
    u32x4 kf[2][DK];
    auto fetch = [&](int c, int buf) {
      const int k0 = key(c);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // (what the buffer held has been read)
      Rows<D>::fill(vg, a.v_st, k0, 0, s.len, vs[wave][buf], lane);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t row = (int64_t)min(s.len - 1, k0 + 8 * (li >> 2) + 4 * h + (li & 3)) * a.k_st;
#pragma unroll
        for (int ks = 0; ks < DK; ++ks) kf[h][ks] = *(const u32x4*)(kg + row + 32 * ks + 8 * g);
      }
    };
    int c = split * per + wave, buf = 0;
    if (c < end) fetch(c, 0);
    for (; c < end; c += NW, buf ^= 1) {
      const int k0 = key(c);
      // (the keys were loaded behind the values: with one of them here, so are the values, and no
      // read of theirs comes before this)
      asm volatile("" : "+v"(kf[0][0]) : : "memory");
      f32x4 x[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        x[h] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int ks = 0; ks < DK; ++ks) x[h] = E::mfma16(kf[h][ks], qf[ks], x[h]);
      }
      if (c + NW < end) fetch(c + NW, buf ^ 1);
      float mx = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = k0 + 8 * g + 4 * h + r;
          const bool see = j <= i && (i - j < a.W || j < a.S);
          x[h][r] = see ? x[h][r] * a.c : -INFINITY;
          mx = fmaxf(mx, x[h][r]);
        }
      const float mn = fmaxf(m, over_groups(mx, true)), f = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      float sum = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          x[h][r] = __builtin_amdgcn_exp2f(x[h][r] - m);
          sum += x[h][r];
        }
      l = l * f + sum;
      const Two p = split8<E>(x[0][0], x[0][1], x[0][2], x[0][3], x[1][0], x[1][1], x[1][2], x[1][3]);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const uint16_t* v = vs[wave][buf];
        const int r = 8 * g + (li >> 2), col = 16 * dt + 4 * (li & 3);
        const bf16x8 vf = cat_frag(lds_tr4((const bf16_t*)v + lds_off<D>(r, col)),
                                   lds_tr4((const bf16_t*)v + lds_off<D>(r + 4, col)));
        acc[dt] *= f;
        acc[dt] = E::mfma16(__builtin_bit_cast(u32x4, vf), p.hi, acc[dt]);
        acc[dt] = E::mfma16(__builtin_bit_cast(u32x4, vf), p.lo, acc[dt]);
      }
    }
    l = over_groups(l, false);
  }
  // the waves' rows are joined relative to the largest of their maxima
  if (lane < 16) {
    stat[0][wave][lane] = m;
    stat[1][wave][lane] = l;
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();
  float* buf = (float*)vs;                             // [NW][16][D]
  float top = -3e38f, total = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) top = fmaxf(top, stat[0][w][li]);
#pragma unroll
  for (int w = 0; w < NW; ++w) total += stat[1][w][li] * __builtin_amdgcn_exp2f(stat[0][w][li] - top);
  const float f = __builtin_amdgcn_exp2f(m - top);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) *(f32x4*)(buf + (wave * 16 + li) * D + 16 * dt + 4 * g) = acc[dt] * f;
  __syncthreads();
  // thread: row e / (D / 4), 4 columns
  for (int e = tid; e < rows * (D / 4); e += NW * 64) {
    const int row = e / (D / 4), col = e % (D / 4) * 4;
    f32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < NW; ++w) v += *(const f32x4*)(buf + (w * 16 + row) * D + col);
    if (splits > 1) {
      *(f32x4*)(part + ((int64_t)blockIdx.x * 16 + row) * (D + 4) + col) = v;
    } else {
      float tm = -3e38f, z = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) tm = fmaxf(tm, stat[0][w][row]);
#pragma unroll
      for (int w = 0; w < NW; ++w) z += stat[1][w][row] * __builtin_amdgcn_exp2f(stat[0][w][row] - tm);
      v *= z > 0.f ? 1.f / z : 0.f;
      const int64_t at = (((int64_t)b * a.Tq + row % a.Tq) * a.H + hk * G + row / a.Tq) * D + col;
      *(uint2*)(o + at) = make_uint2(E::pack2(v[0], v[1]), E::pack2(v[2], v[3]));
    }
  }
  if (splits > 1 && wave == 0 && lane < rows) {
    float* st = part + ((int64_t)blockIdx.x * 16 + lane) * (D + 4) + D;
    st[0] = top;
    st[1] = total;
  }
}

// one row of a key head from the shares of its workgroups: thread (slice, 4 columns)
template <class E, int D>
__global__ __launch_bounds__(256) void window_join_kernel(const float* part, int splits, uint16_t* o, int H, int KV,
                                                          int Tq) {
  constexpr int C = D / 4, SL = 256 / C;
  constexpr int64_t step = 16 * (D + 4);
  __shared__ float tops[4];
  __shared__ f32x4 sums[SL][C];
  __shared__ float zs[SL];
  const int G = H / KV, rows = G * Tq, bk = blockIdx.x / rows, row = blockIdx.x - bk * rows;
  const int b = bk / KV, hk = bk - b * KV, tid = threadIdx.x;
  const float* p = part + ((int64_t)bk * splits * 16 + row) * (D + 4);
  float top = -3e38f;
  for (int i = tid; i < splits; i += 256) top = fmaxf(top, p[i * step + D]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  if ((tid & 63) == 0) tops[tid >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const int sl = tid / C, col = tid % C * 4;
  float z = 0.f;
  f32x4 v = {0, 0, 0, 0};
#pragma unroll 4
  for (int i = sl; i < splits; i += SL) {
    const float f = __builtin_amdgcn_exp2f(p[i * step + D] - top);
    z += p[i * step + D + 1] * f;
    v += *(const f32x4*)(p + i * step + col) * f;
  }
  sums[sl][col / 4] = v;
  if (col == 0) zs[sl] = z;
  __syncthreads();
  if (sl) return;
  for (int i = 1; i < SL; ++i) {
    v += sums[i][col / 4];
    z += zs[i];
  }
  v *= z > 0.f ? 1.f / z : 0.f;
  const int64_t at = (((int64_t)b * Tq + row % Tq) * H + hk * G + row / Tq) * D + col;
  *(uint2*)(o + at) = make_uint2(E::pack2(v[0], v[1]), E::pack2(v[2], v[3]));
}

template <class E, int D>
int step(const WinArgs& a, void* o, void* part, int splits, hipStream_t st) {
  const int64_t n = (int64_t)a.B * a.KV * splits;
  if (n >= (1ll << 31) || (int64_t)a.B * a.H * a.Tq >= (1ll << 31)) return 1;
  hipLaunchKernelGGL((window_step_kernel<E, D>), dim3((unsigned)n), dim3(NW * 64), 0, st, a, (uint16_t*)o,
                     (float*)part, splits);
  if (splits > 1)
    hipLaunchKernelGGL((window_join_kernel<E, D>), dim3((unsigned)((int64_t)a.B * a.H * a.Tq)), dim3(256), 0, st, (const float*)part, splits,
                       (uint16_t*)o, a.H, a.KV, a.Tq);
  return (int)hipGetLastError();
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
int bwd(const WinArgs& a, const void* o, const void* rest, const void* dout, const void* lse, void* dsum, void* dq,
        void* dk, void* dv, void* part, int parts, int spans, int span, float scale, hipStream_t st) {
  const int64_t n = (int64_t)((a.Tq + BM - 1) / BM) * a.B * a.H, bks = (int64_t)a.B * a.KV;
  const int64_t near = (int64_t)((a.Tk + BM - 1) / BM) * parts * bks;
  const int64_t nk = near + (((int64_t)((a.S + 31) / 32) * spans * bks + 7) & ~7ll);
  if (n >= (1ll << 31) || nk >= (1ll << 31)) return 1;
  hipLaunchKernelGGL((window_dq_kernel<E, D>), dim3((unsigned)n), dim3(256), 0, st, a, (const uint16_t*)o,
                     (const uint16_t*)rest, (const uint16_t*)dout, (const float*)lse, (float*)dsum, (uint16_t*)dq,
                     scale);
  hipLaunchKernelGGL((window_dkv_kernel<E, D>), dim3((unsigned)nk), dim3(256), 0, st, a, (const uint16_t*)dout,
                     (const float*)lse, (const float*)dsum, (uint16_t*)dk, (uint16_t*)dv, (float*)part, parts, spans,
                     span, scale);
  if (parts > 1 || spans) {
    const int rows = parts > 1 ? a.Tk : a.S, S = spans ? a.S : 0, wide = spans > 4 ? S : 0, per = 256 / (2 * D / 4);
    const int64_t blocks = bks * wide + (bks * (rows - wide) + per - 1) / per;
    if (blocks >= (1ll << 31)) return 1;
    hipLaunchKernelGGL((window_sum_kernel<E, D>), dim3((unsigned)blocks), dim3(256), 0, st, (const float*)part, parts,
                       spans, bks, rows, S, wide, a.Tk, (uint16_t*)dk, (uint16_t*)dv, scale);
  }
  return (int)hipGetLastError();
}

bool good(const WinArgs& a, int D) {
  return a.B > 0 && a.H > 0 && a.KV > 0 && a.H % a.KV == 0 && a.Tq > 0 && a.Tk > 0 && a.W > 0 && a.S >= 0 &&
         (D == 64 || D == 128) && a.Tq <= (1 << 29) && a.Tk <= (1 << 29) && a.W <= (1 << 30) &&
         a.S <= a.Tk && (int64_t)a.H * D < (1 << 24) && a.c > 0.f;
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

// The same output for H / KV * Tq <= 16; part: workspace of B KV splits 16 (D + 4) floats where splits > 1.
int mopt_window_step(const void* q, const void* k, const void* v, const int64_t* strides, const void* start,
                     const void* lengths, int start0, void* o, void* part, int splits, int B, int H, int KV, int Tq,
                     int Tk, int D, int W, int S, float scale, int dtype, void* stream) {
  const WinArgs a = args(q, k, v, strides, start, lengths, start0, B, H, KV, Tq, Tk, W, S, scale);
  if (!good(a, D) || (int64_t)(H / KV) * Tq > 16 || splits < 1 || (splits > 1 && !part)) return 1;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == 0) return D == 64 ? step<Bf16, 64>(a, o, part, splits, st) : step<Bf16, 128>(a, o, part, splits, st);
  return D == 64 ? step<Fp16, 64>(a, o, part, splits, st) : step<Fp16, 128>(a, o, part, splits, st);
}

// dq [B][H][Tq][D], dk, dv [B][KV][Tk][D]; dsum: floats of workspace; part: workspace of
// (parts R + 4 spans S) B KV 2 D floats, R = Tk where parts > 1, else S; parts: shares of each key
// block's queries; spans * span >= Tq (spans 0: no sink is seen out of its window);
// lse, dsum: rows of Tq rounded up to 128
int mopt_window_bwd(const void* q, const void* k, const void* v, const int64_t* strides, const void* start,
                    const void* lengths, int start0, const void* o, const void* rest, const void* dout, const void* lse, void* dsum,
                    void* dq, void* dk, void* dv, void* part, int parts, int spans, int span, int B, int H, int KV, int Tq,
                    int Tk, int D, int W, int S, float scale, int dtype, void* stream) {
  const WinArgs a = args(q, k, v, strides, start, lengths, start0, B, H, KV, Tq, Tk, W, S, scale);
  if (!good(a, D) || parts < 1 || spans < 0 || span <= 0 || span % BN) return 1;
  if ((parts > 1 || spans) && !part || (spans && S == 0)) return 1;
  if (S && Tk > W && (int64_t)spans * span < Tq) return 1;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == 0)
    return D == 64 ? bwd<Bf16, 64>(a, o, rest, dout, lse, dsum, dq, dk, dv, part, parts, spans, span, scale, st)
                   : bwd<Bf16, 128>(a, o, rest, dout, lse, dsum, dq, dk, dv, part, parts, spans, span, scale, st);
  return D == 64 ? bwd<Fp16, 64>(a, o, rest, dout, lse, dsum, dq, dk, dv, part, parts, spans, span, scale, st)
                 : bwd<Fp16, 128>(a, o, rest, dout, lse, dsum, dq, dk, dv, part, parts, spans, span, scale, st);
}

}  // extern "C"
