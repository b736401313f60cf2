// Distillation from a teacher's top logits for gfx950: loss and gradient of a student's logits in one launch.
//
//   logits  [N, V] bf16 (row stride ld)        teacher [N, K] fp32 logits (or log-probabilities) of the tokens
//   index   [N, K] int32                       weight  [N] fp32 or null (1)
//   p = softmax(teacher / t) over the K listed tokens, q = softmax(logits / t) over the vocabulary
//   loss_i  = t^2 w_i sum_k p_k (log p_k - log q[index_k])
//   dlogits = t w_i (q - scatter(p))           (d loss_i / d logits; the t^2 keeps its size independent of t)
// An entry whose index is outside [0, V) or whose teacher logit is -inf or NaN is padding (p_k = 0); a row of padding
// has p = 0: loss 0 and gradient 0, as has a row of weight 0. Sums and statistics are fp32.
//
// q_i = 2^((x_i - m) c) / s with c = log2 e / t, m the row's maximum and s the sum of those powers; log2 q_i = (x_i - m) c - log2 s. The
// maximum is subtracted before anything is scaled and never joined to the sum: m c + log2 s as one fp32 number is off by half a
// step of m c, which at low temperatures is percents of q (m = 50: 0.8 % at t = 1e-3), and overflows where logits are masked with
// the type's lowest value.
#include "common.h"
#include "kernels.h"

namespace kop {

namespace {
constexpr float kL2E = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// 8 logits of a row at element i, a multiple of 8 (rows may start off the 16-byte grid: global accesses take any element's
// alignment); 32-bit byte offsets keep the row's base in scalar registers
struct __attribute__((packed, aligned(2))) U16 {
  u32x4 v;
};
__device__ __forceinline__ u32x4 load8(const bf16_t* x, uint32_t i) {
  return reinterpret_cast<const U16*>(reinterpret_cast<const char*>(x) + 2 * i)->v;
}
__device__ __forceinline__ void store8(bf16_t* x, uint32_t i, const float* f) {
  reinterpret_cast<U16*>(reinterpret_cast<char*>(x) + 2 * i)->v = pack8(f);
}
__device__ __forceinline__ float max8(const float* f) {
  return fmaxf(fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])), fmaxf(fmaxf(f[4], f[5]), fmaxf(f[6], f[7])));
}

// The teacher's side of a row and the listed tokens' logits, in LDS.
template <int NT>
struct Teacher {
  int idx[kDistillMaxK];    // -1: padding
  float p[kDistillMaxK];    // logit, then probability
  float x[kDistillMaxK];    // the student's logit of the token
  float red[NT / 64];

  // the row's entries; returns the largest teacher logit (-inf: all padding), in every thread
  __device__ __forceinline__ float load(const bf16_t* xr, int V, const int* index, const float* teacher, int K) {
    float m = -INFINITY;
    for (int k = threadIdx.x; k < K; k += NT) {
      const int i = index[k];
      float v = teacher[k];
      const bool real = i >= 0 && i < V && v > -INFINITY;  // false for NaN
      v = real ? v : -INFINITY;
      idx[k] = real ? i : -1;
      p[k] = v;
      x[k] = real ? bf2f(xr[i]) : 0.f;
      m = fmaxf(m, v);
    }
    return block_max<NT / 64>(m, red);
  }
  // p = softmax; returns the loss in units of log2 without its factors. m, ls2: the student's maximum and log2 of its sum
  __device__ __forceinline__ float finish(int K, float tm, float c, float m, float ls2, bool some) {
    float s = 0.f;
    for (int k = threadIdx.x; k < K; k += NT) s += idx[k] >= 0 ? __builtin_amdgcn_exp2f((p[k] - tm) * c) : 0.f;
    __syncthreads();  // red may still be read
    s = block_sum<NT / 64>(s, red);
    const float ls = __log2f(s);
    float part = 0.f;
    for (int k = threadIdx.x; k < K; k += NT) {
      const float lp = (p[k] - tm) * c - ls;
      const float e = idx[k] >= 0 ? __builtin_amdgcn_exp2f(lp) : 0.f;
      p[k] = e;
      if (e > 0.f) part += e * (lp - (some ? (x[k] - m) * c - ls2 : -INFINITY));
    }
    __syncthreads();
    return block_sum<NT / 64>(part, red);
  }
  // the listed tokens' own elements, once every element of the row has been written. A token listed more than once: its
  // entries' sum, written by the first of them. inv: 1 / the student's sum
  __device__ __forceinline__ void patch(int K, float c, float m, float inv, float gw, bf16_t* gx) {
    __syncthreads();
    for (int k = threadIdx.x; k < K; k += NT) {
      const int i = idx[k];
      if (i < 0) continue;
      float sum = 0.f;
      bool first = true;
#pragma unroll 8
      for (int j = 0; j < K; ++j) {
        const bool same = idx[j] == i;
        sum += same ? p[j] : 0.f;
        first = first && !(same && j < k);
      }
      if (first) gx[i] = f2bf(gw * (__builtin_amdgcn_exp2f((x[k] - m) * c) * inv - sum));
    }
  }
};

struct Args {
  const bf16_t* logits;
  int64_t ld;
  int V, K;
  const int* index;
  const float *teacher, *weight;
  float temp;
  float* loss;
  bf16_t* grad;
  int64_t gld;
};
// rows without a loss: zeros
template <int NT>
__device__ __forceinline__ void no_loss(const Args& a, int64_t row, bf16_t* gx) {
  const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const uint32_t V8 = a.V & ~7u;
  if (threadIdx.x == 0) a.loss[row] = 0.f;
  for (uint32_t i = threadIdx.x * 8; i < V8; i += NT * 8) store8(gx, i, z);
  if (V8 + threadIdx.x < (uint32_t)a.V) gx[V8 + threadIdx.x] = 0;
}

// keeps the compiler from carrying a pass's unpacked floats (twice the registers) over to the next pass
template <int N>
__device__ __forceinline__ void repack(u32x4* v) {
#pragma unroll
  for (int j = 0; j < N; ++j) asm volatile("" : "+v"(v[j]));
}

// One workgroup per row that holds the whole row: CR 16-byte pieces per thread in registers, CL more in LDS, so every
// logit is read once and every gradient element written once. Two plain reductions, no running rescale. Bound by memory: 16384 rows
// of 50304 612 us, 5.4 TB/s (two rows per CU: one loads while the other one reduces); 8192 rows of 128256 830 us, 5.06 TB/s.
template <int NT, int CR, int CL>
__global__ void __launch_bounds__(NT, NT >= 512 && CR + CL > 16 ? 4 : 1) distill_row_kernel(Args a) {
  __shared__ Teacher<NT> s_t;
  __shared__ u32x4 s_w[CL > 0 ? CL * NT : 1];
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x;
  const bf16_t* x = a.logits + row * a.ld;
  bf16_t* gx = a.grad + row * a.gld;
  const float w = a.weight ? a.weight[row] : 1.f;
  const float c = kL2E / a.temp;
  // pieces j * NT + t of 8 logits; the up to 7 logits behind the last whole piece: one each for the first threads
  const uint32_t V8 = a.V & ~7u;
  const bool tail = V8 + t < (uint32_t)a.V;
  constexpr uint32_t kPad = 0xff80ff80u;  // two bf16 -inf
  u32x4 v[CR];
  static_assert(CL % 3 == 0, "LDS pieces are loaded three at a time");
#pragma unroll 1
  for (int j = 0; j < CL; j += 3) {
    u32x4 q[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const uint32_t i = ((CR + j + k) * NT + t) * 8;
      q[k] = u32x4{kPad, kPad, kPad, kPad};
      if (i < V8) q[k] = load8(x, i);
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) s_w[(j + k) * NT + t] = q[k];
  }
#pragma unroll
  for (int j = 0; j < CR; ++j) {
    const uint32_t i = (j * NT + t) * 8;
    v[j] = u32x4{kPad, kPad, kPad, kPad};
    if (i < V8) v[j] = load8(x, i);
  }
  const float xt = tail ? bf2f(x[V8 + t]) : -INFINITY;
  const float tm = s_t.load(x, a.V, a.index + row * a.K, a.teacher + row * a.K, a.K);
  if (!(tm > -INFINITY && w != 0.f)) {
    no_loss<NT>(a, row, gx);
    return;
  }
  float m = xt;
  float f[8];
#pragma unroll 1
  for (int j = 0; j < CL; ++j) {
    unpack8(s_w[j * NT + t], f);
    m = fmaxf(m, max8(f));
  }
#pragma unroll
  for (int j = 0; j < CR; ++j) {
    unpack8(v[j], f);
    m = fmaxf(m, max8(f));
  }
  __syncthreads();
  m = block_max<NT / 64>(m, s_t.red);
  const bool some = m > -INFINITY;  // false: every logit is -inf, q = 0
  m = some ? m : 0.f;
  repack<CR>(v);
  float s = __builtin_amdgcn_exp2f((xt - m) * c);
#pragma unroll 1
  for (int j = 0; j < CL; ++j) {
    unpack8(s_w[j * NT + t], f);
#pragma unroll
    for (int e = 0; e < 8; ++e) s += __builtin_amdgcn_exp2f((f[e] - m) * c);
  }
#pragma unroll
  for (int j = 0; j < CR; ++j) {
    unpack8(v[j], f);
#pragma unroll
    for (int e = 0; e < 8; ++e) s += __builtin_amdgcn_exp2f((f[e] - m) * c);
  }
  __syncthreads();
  s = block_sum<NT / 64>(s, s_t.red);
  const float inv = some ? 1.f / s : 0.f;
  const float part = s_t.finish(a.K, tm, c, m, __log2f(s), some);
  if (t == 0) a.loss[row] = part * kLn2 * a.temp * a.temp * w;
  const float gw = a.temp * w, gq = gw * inv;
  repack<CR>(v);
  auto put = [&](u32x4 q, uint32_t i) {
    unpack8(q, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = gq * __builtin_amdgcn_exp2f((f[e] - m) * c);
    if (i < V8) store8(gx, i, f);
  };
#pragma unroll
  for (int j = 0; j < CR; ++j) put(v[j], (j * NT + t) * 8);
#pragma unroll 1
  for (int j = 0; j < CL; ++j) put(s_w[j * NT + t], ((CR + j) * NT + t) * 8);
  if (tail) gx[V8 + t] = f2bf(gq * __builtin_amdgcn_exp2f((xt - m) * c));
  s_t.patch(a.K, c, m, inv, gw, gx);
}

// Rows longer than that: two passes, running (maximum, sum) in the log2 domain, then the gradient. Bound by memory, with the
// logits read twice: 8192 rows of 128256 (which the form above holds) 1272 us, 5.0 TB/s.
template <int NT>
__global__ void __launch_bounds__(NT) distill_long_kernel(Args a) {
  __shared__ Teacher<NT> s_t;
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x;
  const bf16_t* x = a.logits + row * a.ld;
  bf16_t* gx = a.grad + row * a.gld;
  const float w = a.weight ? a.weight[row] : 1.f;
  const float c = kL2E / a.temp;
  const uint32_t V8 = a.V & ~7u;
  const bool tail = V8 + t < (uint32_t)a.V;
  const float xt = tail ? bf2f(x[V8 + t]) : -INFINITY;
  const float tm = s_t.load(x, a.V, a.index + row * a.K, a.teacher + row * a.K, a.K);
  if (!(tm > -INFINITY && w != 0.f)) {
    no_loss<NT>(a, row, gx);
    return;
  }
  float m = xt, s = xt > -INFINITY ? 1.f : 0.f, f[8];
  for (uint32_t i = t * 8; i < V8; i += NT * 8) {
    unpack8(load8(x, i), f);
    const float nm = fmaxf(m, max8(f));
    if (nm == -INFINITY) continue;
    float add = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) add += __builtin_amdgcn_exp2f((f[e] - nm) * c);
    s = s * __builtin_amdgcn_exp2f((m - nm) * c) + add;  // m = -inf: times 0
    m = nm;
  }
  __syncthreads();
  float M = block_max<NT / 64>(m, s_t.red);
  __syncthreads();
  s = block_sum<NT / 64>(m == -INFINITY ? 0.f : s * __builtin_amdgcn_exp2f((m - M) * c), s_t.red);
  const bool some = M > -INFINITY;
  M = some ? M : 0.f;
  const float inv = some ? 1.f / s : 0.f;
  const float part = s_t.finish(a.K, tm, c, M, __log2f(s), some);
  if (t == 0) a.loss[row] = part * kLn2 * a.temp * a.temp * w;
  const float gw = a.temp * w, gq = gw * inv;
  for (uint32_t i = t * 8; i < V8; i += NT * 8) {
    unpack8(load8(x, i), f);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = gq * __builtin_amdgcn_exp2f((f[e] - M) * c);
    store8(gx, i, f);
  }
  if (tail) gx[V8 + t] = f2bf(gq * __builtin_amdgcn_exp2f((xt - M) * c));
  s_t.patch(a.K, c, M, inv, gw, gx);
}
}  // namespace

int distill_topk(const bf16_t* logits, int64_t ld, int64_t N, int V, const int* index, const float* teacher, int K,
                 const float* weight, float temp, float* loss, bf16_t* grad, int64_t gld, hipStream_t stream) {
  if (K < 1 || K > kDistillMaxK || V < 1 || V > 0x3fffffff || N < 0 || N > 0x7fffffff) return -1;
  if (N == 0) return 0;
  const Args a = {logits, ld, V, K, index, teacher, weight, temp, loss, grad, gld};
  const unsigned n = (unsigned)N;
  // The smallest workgroup that holds a row, so that several rows share a CU. A wave up to 4096 logits (16384 rows of 512 / 2000 /
  // 4000: 20 / 34 / 58 us against 50 / 51 / 60 by 256 threads; 64 rows of 4000 6.9 against 6.5); 512 threads above. Rows that 512
  // threads hold only with LDS's help: with one row per CU or fewer by 1024 in registers (32 rows of 128000: 21.1 us against 22.4;
  // 512 rows: 59 against 50). Rows that no workgroup holds: two passes (8192 rows of 128256 that way: 1272 us against 830).
#define KOP_ROW(NT, CR, CL)                                        \
  if (V < NT * 8 * (CR + CL) + 8) {                                \
    distill_row_kernel<NT, CR, CL><<<n, NT, 0, stream>>>(a);       \
    return hipGetLastError() == hipSuccess ? 0 : -9;               \
  }
  KOP_ROW(64, 1, 0)
  KOP_ROW(64, 2, 0)
  KOP_ROW(64, 4, 0)
  KOP_ROW(64, 8, 0)
  KOP_ROW(256, 4, 0)
  KOP_ROW(512, 8, 0)
  KOP_ROW(512, 16, 0)
  if (N <= 256) {
    KOP_ROW(1024, 16, 0)
  }
  KOP_ROW(512, 23, 9)
#undef KOP_ROW
  distill_long_kernel<512><<<n, 512, 0, stream>>>(a);
  return hipGetLastError() == hipSuccess ? 0 : -9;
}

}  // namespace kop
