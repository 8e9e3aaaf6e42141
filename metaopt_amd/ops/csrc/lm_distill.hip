// Distillation from a teacher's top logits, with the hard labels' cross-entropy (ops/distill.py).
//
// Row of V student logits x, label y (negative: none), K teacher logits t_k at vocabulary indices
// i_k (negative: absent), temperature tau and mix a of the row's trial:
//   q = softmax(t / tau) over the present entries, p1 = softmax(x), ptau = softmax(x / tau)
//   loss = (1 - a) (-log p1[y]) + a tau^2 sum_k q_k (log q_k - log ptau[i_k])
//   dx_j = (1 - a) (p1_j - [j = y]) + a tau (ptau_j - sum_k q_k [i_k = j])
// A row without a label has no first term, one without a teacher no second.
//
// One workgroup per row.  The row is read once, into registers (distill_row_kernel with NCH 16-byte
// chunks a thread): its maximum, then both sums of exponentials, then the gradient come from there,
// so the traffic is one read and one write of the logits, which bounds it (32768 rows of 32000 bf16
// logits, K = 64: 843 - 851 us a pass, 837 of it this kernel, 5 TB/s, as fast as a copy of 4 GiB; before the
// row's floats were kept from being held unpacked, at half the occupancy, 951).  Two exponentials a value in
// each of the two passes just hide behind it (the vector pipe is busy for 92 % of the time): at temperature 1,
// where one would do, the time is the same.  The K + 1 corrected places of
// the gradient are written again after the dense pass with their whole f32 value, so each value
// is rounded once; equal indices are added up by every entry that has them.  Sums of losses are
// taken row by row in a fixed order (no atomics).
#include "elt.h"

using namespace mopt;

namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct F32 {};

// 16-byte chunk of logits -> floats and back
template <class E>
struct Row {
  static constexpr int N = 8, SIZE = 2;
  static __device__ __forceinline__ void get(const u32x4& w, float (&f)[8]) { up8<E>(w, f); }
  static __device__ __forceinline__ u32x4 put(const float (&f)[8]) { return down8<E>(f); }
  static __device__ __forceinline__ float load(const void* p, int64_t i) {
    return E::up(((const uint16_t*)p)[i]);
  }
  static __device__ __forceinline__ void store(void* p, int64_t i, float v) {
    ((uint16_t*)p)[i] = (uint16_t)(E::pack2(v, v) & 0xFFFF);
  }
};
template <>
struct Row<F32> {
  static constexpr int N = 4, SIZE = 4;
  static __device__ __forceinline__ void get(const u32x4& w, float (&f)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = __uint_as_float(w[j]);
  }
  static __device__ __forceinline__ u32x4 put(const float (&f)[4]) {
    return u32x4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                 __float_as_uint(f[3])};
  }
  static __device__ __forceinline__ float load(const void* p, int64_t i) {
    return ((const float*)p)[i];
  }
  static __device__ __forceinline__ void store(void* p, int64_t i, float v) { ((float*)p)[i] = v; }
};

// rows of an odd length start at any element: chunks are moved with the element's alignment
template <int SIZE>
struct Chunk;
template <>
struct Chunk<2> {
  struct __attribute__((packed, aligned(2))) type { u32x4 v; };
};
template <>
struct Chunk<4> {
  struct __attribute__((packed, aligned(4))) type { u32x4 v; };
};

struct DistillArgs {
  const void* x;
  int64_t ld;                // row stride of x (elements); the gradient's is V
  const int32_t* labels;
  const void* top;           // [rows][K] f32, bf16 or fp16 (top_type 2, 0, 1)
  const int32_t* index;      // [rows][K]
  const float *tau, *alpha;  // per trial, or null: the values below
  const float* weight;       // per trial factor of the gradient, or null
  float* row_loss;           // [rows], or null
  void* grad;                // [rows][V], or null
  int rpt, V, K, top_type;
  float tau_v, alpha_v, scale;
};

// sums (or maxima) of N values over the workgroup, given to every thread
template <int NT, int N, bool MAX>
__device__ __forceinline__ void block_all(float (&v)[N], float* red) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const float w = __shfl_xor(v[i], o, 64);
      v[i] = MAX ? fmaxf(v[i], w) : v[i] + w;
    }
  }
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  __syncthreads();
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) red[wave * N + i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float r = red[i];
    for (int w = 1; w < NT / 64; ++w) r = MAX ? fmaxf(r, red[w * N + i]) : r + red[w * N + i];
    v[i] = r;
  }
}

__device__ __forceinline__ float load_top(const void* p, int type, int64_t i) {
  if (type == 2) return ((const float*)p)[i];
  const uint32_t h = ((const uint16_t*)p)[i];
  return type == 0 ? Bf16::up(h) : Fp16::up(h);
}

// The compiler would keep the unpacked floats of the row from one pass to the next, in twice the
// registers: a value that went through this is unpacked anew, chunk after chunk (volatile: in order).
__device__ __forceinline__ void forget(u32x4& v) { asm volatile("" : "+v"(v)); }

// NCH > 0: the row is kept in NCH chunks of NT threads (V <= NT * NCH * N).  NCH = 0: longer rows
// are read again from memory in each pass.  WAVES a SIMD: the registers (512 / WAVES).
template <class E, int NT, int NCH, int WAVES>
__global__ __launch_bounds__(NT, WAVES) void distill_row_kernel(DistillArgs a) {
  using R = Row<E>;
  using C = typename Chunk<R::SIZE>::type;
  constexpr int N = R::N;
  extern __shared__ float lds[];                    // [K] index, [K] exp of the teacher, reductions
  int* s_idx = (int*)lds;
  float* s_e = lds + a.K;
  float* red = lds + 2 * a.K;
  const int tid = threadIdx.x, V = a.V, K = a.K;
  const int64_t row = blockIdx.x;
  const int trial = (int)(row / a.rpt);
  const char* const x = (const char*)a.x + row * a.ld * R::SIZE;
  const float tau = a.tau ? a.tau[trial] : a.tau_v, alpha = a.alpha ? a.alpha[trial] : a.alpha_v;
  const float rtau = 1.f / tau;

  // whole chunks, and the few values behind them: one more of the first threads
  const int full = V / N;
  const float more = tid < V - full * N ? R::load(x, full * N + tid) : -INFINITY;
  float none[N];
#pragma unroll
  for (int j = 0; j < N; ++j) none[j] = -INFINITY;
  u32x4 keep[NCH > 0 ? NCH : 1];
  if constexpr (NCH > 0) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      keep[i] = R::put(none);
      if (i * NT + tid < full) keep[i] = ((const C*)(x + i * NT * 16))[tid].v;   // (scalar base, one offset)
    }
  }
  // every chunk of this thread, in its order: f(first chunk of the group, values)
  auto each = [&](auto f) {
    if constexpr (NCH > 0) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        float v[N];
        forget(keep[i]);
        R::get(keep[i], v);
        f(i * NT, v);
      }
    } else {
      for (int c = 0; c + tid < full; c += NT) {
        float v[N];
        R::get(((const C*)(x + c * 16))[tid].v, v);
        f(c, v);
      }
    }
  };
  float mx[2] = {more, -INFINITY};                  // of the row, of the teacher
  const int y = a.labels[row];
  const bool has_label = y >= 0 && y < V;
  const float xy = has_label ? R::load(x, y) : 0.f;
  for (int k = tid; k < K; k += NT) {
    const int i = a.index[row * K + k];
    const bool ok = i >= 0 && i < V;
    const float t = ok ? load_top(a.top, a.top_type, row * K + k) : -INFINITY;
    s_idx[k] = ok ? i : -1;
    s_e[k] = t;                                      // (each thread reads back its own entries)
    mx[1] = fmaxf(mx[1], t);
  }
  each([&](int, const float (&f)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) mx[0] = fmaxf(mx[0], f[j]);
  });
  block_all<NT, 2, true>(mx, red);
  const float m = mx[0], tm = mx[1];
  // Exponents are formed from v - m itself, the reference that the loss is relative to: with -m k rounded
  // once and added in an fma, all terms are off by one factor that the loss does not take off again (losses
  // of rows with logits of 1000: 4e-5 off; past m / tau = 2^31 the factor is infinite).
  const float kt = kLog2e * rtau;
  const bool hard = has_label && alpha != 1.f, soft = tm > -INFINITY && alpha != 0.f;
  char* const g = (char*)a.grad + row * (int64_t)V * R::SIZE;
  if (!hard && !soft) {                              // no loss and no gradient, whatever the logits are
    if (tid == 0 && a.row_loss) a.row_loss[row] = 0.f;
    if (!a.grad) return;
    u32x4 zero = {0, 0, 0, 0};
    for (int c = tid; c < full; c += NT) ((C*)g)[c].v = zero;
    if (tid < V - full * N) R::store(g, full * N + tid, 0.f);
    return;
  }
  float sums[4] = {0.f, 0.f, 0.f, 0.f};            // z1, ztau, zq, sum e_k (log e_k - x_k / tau)
  auto add = [&](float v) {
    sums[0] += __builtin_amdgcn_exp2f((v - m) * kLog2e);
    sums[1] += __builtin_amdgcn_exp2f((v - m) * kt);
  };
  each([&](int, const float (&f)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) add(f[j]);
  });
  add(more);
  if (soft)
    for (int k = tid; k < K; k += NT) {
      const float d = (s_e[k] - tm) * rtau;
      const int i = s_idx[k];
      const float e = i >= 0 ? __builtin_amdgcn_exp2f(d * kLog2e) : 0.f;
      s_e[k] = e;
      sums[2] += e;
      if (e > 0.f) sums[3] += e * (d - (R::load(x, i) - m) * rtau);
    }
  block_all<NT, 4, false>(sums, red);
  if (tid == 0 && a.row_loss) {
    float loss = 0.f;
    if (hard) loss += (1.f - alpha) * (logf(sums[0]) - (xy - m));
    if (soft) loss += alpha * tau * tau * (sums[3] / sums[2] - logf(sums[2]) + logf(sums[1]));
    a.row_loss[row] = loss;
  }
  if (!a.grad) return;
  const float scale = a.scale * (a.weight ? a.weight[trial] : 1.f);
  const float h1 = hard ? scale * (1.f - alpha) : 0.f, ht = soft ? scale * alpha * tau : 0.f;
  const float c1 = hard ? h1 / sums[0] : 0.f, ct = soft ? ht / sums[1] : 0.f;
  auto dense = [&](float v) {
    return fmaf(c1, __builtin_amdgcn_exp2f((v - m) * kLog2e), ct * __builtin_amdgcn_exp2f((v - m) * kt));
  };
  // The corrected places, each computed by the entries that have it (the teacher's, then the
  // label).  Their logits are read before any gradient is written: it may take the logits' place.
  const int entries = K + 1;
  auto place = [&](int k) { return k < K ? s_idx[k] : (has_label ? y : -1); };
  float late = 0.f;
  float* const lates = lds + 2 * K + 4 * (NT / 64);  // [K] where there are more entries than threads
  for (int k = tid; k < entries; k += NT) {
    const int i = place(k);
    if (i >= 0) {
      float off = has_label && i == y ? h1 : 0.f;
      if (soft) {
        float q = 0.f;
        for (int n = 0; n < K; ++n) q += s_idx[n] == i ? s_e[n] : 0.f;
        off += ht * (q / sums[2]);
      }
      late = dense(R::load(x, i)) - off;
    }
    if (K >= NT && k < K) lates[k] = late;
  }
  __syncthreads();
  // (written past the caches: nothing here reads it again, and what the next rows read stays)
  each([&](int c, const float (&f)[N]) {
    float o[N];
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = dense(f[j]);
    if (c + tid < full) __builtin_nontemporal_store(R::put(o), &((C*)(g + c * 16))[tid].v);
  });
  if (tid < V - full * N) R::store(g, full * N + tid, dense(more));
  __syncthreads();
  for (int k = tid; k < entries; k += NT) {
    const int i = place(k);
    if (i >= 0) R::store(g, i, K >= NT && k < K ? lates[k] : late);
  }
}

// loss[p] = sum of the trial's row losses, one block a trial, in a fixed order
__global__ __launch_bounds__(1024) void distill_sum_kernel(const float* __restrict__ rows, float* loss,
                                                           int rpt) {
  __shared__ double red[16];
  double s = 0.0;
  for (int i = threadIdx.x; i < rpt; i += 1024) s += rows[(int64_t)blockIdx.x * rpt + i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int w = 0; w < 16; ++w) s += red[w];
    loss[blockIdx.x] = (float)s;
  }
}

template <class E, int NT, int NCH, int WAVES>
void launch(const DistillArgs& a, int rows, hipStream_t st) {
  const size_t lds = 4 * (2 * (size_t)a.K + 4 * (NT / 64) + (a.K >= NT ? a.K : 0));
  hipLaunchKernelGGL((distill_row_kernel<E, NT, NCH, WAVES>), dim3(rows), dim3(NT), lds, st, a);
}

// Threads of a row and the chunks that each holds.  Small groups: several rows of a CU then load,
// add up and write at different times (32000 bf16 logits: 16 chunks of 256 threads 874 us, 8 of 512
// 896, 4 of 1024 1929; 49999 f32 logits: 25 of 512 80 us, 16 of 1024 103).  At the steps' edges, 2^28 f32
// logits: 16 of 512 (32768 columns) 441 us, 25 of 512 (33000 to 51200) 433 - 470, 16 of 1024 (51210 to
// 65536) 526 - 584, no chunks kept (65540 to 128256) 619 - 649: that one reads three times and writes once, at
// 6.9 TB/s (the later reads mostly from caches); bf16 338 us at 131072 columns, 388 - 410 past them.
template <class E>
void choose(const DistillArgs& a, int rows, hipStream_t st) {
  const int chunks = (a.V + Row<E>::N - 1) / Row<E>::N;
  if (chunks <= 512) launch<E, 256, 2, 4>(a, rows, st);
  else if (chunks <= 2048) launch<E, 256, 8, 4>(a, rows, st);
  else if (chunks <= 4096) launch<E, 256, 16, 4>(a, rows, st);
  else if (chunks <= 8192) launch<E, 512, 16, 4>(a, rows, st);
  else if (chunks <= 512 * 25) launch<E, 512, 25, 4>(a, rows, st);
  else if (chunks <= 1024 * 16) launch<E, 1024, 16, 4>(a, rows, st);
  else launch<E, 1024, 0, 4>(a, rows, st);
}

}  // namespace

extern "C" {

// dtype (of the logits) and top_type: 0 bf16, 1 fp16, 2 f32.  K <= 1024.  loss and grad may be null.
int mopt_distill(const void* x, int64_t ld, const void* labels, const void* top, const void* index,
                 const void* tau, const void* alpha, const void* weight, void* row_loss, void* loss,
                 void* grad, int rows, int rpt, int V, int K, int top_type, int dtype, float tau_v,
                 float alpha_v, float scale, void* stream) {
  if (rows <= 0 || rpt <= 0 || rows % rpt || V <= 0 || V > (1 << 30) || K < 0 || K > 1024) return 1;
  if ((loss == nullptr) != (row_loss == nullptr)) return 1;
  const DistillArgs a{x, ld, (const int32_t*)labels, top, (const int32_t*)index, (const float*)tau,
                      (const float*)alpha, (const float*)weight, (float*)row_loss, grad, rpt, V, K,
                      top_type, tau_v, alpha_v, scale};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == 0) choose<Bf16>(a, rows, st);
  else if (dtype == 1) choose<Fp16>(a, rows, st);
  else choose<F32>(a, rows, st);
  if (loss)
    hipLaunchKernelGGL(distill_sum_kernel, dim3(rows / rpt), dim3(1024), 0, st,
                       (const float*)row_loss, (float*)loss, rpt);
  return (int)hipGetLastError();
}

}  // extern "C"
