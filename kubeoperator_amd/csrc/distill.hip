// Distillation from a teacher's top logits for gfx950: loss and gradient of a student's logits in one launch.
//
//   logits  [N, V] bf16 (row stride ld)        teacher [N, K] fp32 logits (or log-probabilities) of the tokens
//   index   [N, K] int32                       weight  [N] fp32 or null (1)
//   p = softmax(teacher / t) over the K listed tokens, q = softmax(logits / t) over the vocabulary
//   loss_i  = t^2 w_i sum_k p_k (log p_k - log q[index_k])
//   dlogits = t w_i (q - scatter(p))           (d loss_i / d logits; the t^2 keeps its size independent of t)
// An entry whose index is outside [0, V) or whose teacher logit is -inf or NaN is padding (p_k = 0); a row of padding
// has p = 0: loss 0 and gradient 0, as has a row of weight 0. Sums and statistics are fp32.
#include "common.h"
#include "kernels.h"

namespace kop {

namespace {
constexpr float kL2E = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
}  // namespace

// one workgroup per row, two passes: running (max, sum) in the log2 domain, then the gradient
template <int NT, bool VEC>
__global__ void __launch_bounds__(NT) distill_kernel(const bf16_t* logits, int64_t ld, int V,
                                                     const int* __restrict__ index, const float* __restrict__ teacher,
                                                     int K, const float* __restrict__ weight, float temp,
                                                     float* __restrict__ loss, bf16_t* grad, int64_t gld) {
  __shared__ float red[NT / 64];
  __shared__ int s_idx[kDistillMaxK];
  __shared__ float s_p[kDistillMaxK], s_x[kDistillMaxK];
  const int64_t row = blockIdx.x;
  const bf16_t* x = logits + row * ld;
  bf16_t* gx = grad + row * gld;
  const int t = threadIdx.x;
  const float w = weight ? weight[row] : 1.f;
  const float c = kL2E / temp;
  // teacher: the row's maximum over its real entries
  float tm = -INFINITY;
  for (int k = t; k < K; k += NT) {
    const int i = index[row * K + k];
    float v = teacher[row * K + k];
    const bool real = i >= 0 && i < V && v == v && v > -INFINITY;
    if (!real) v = -INFINITY;
    s_idx[k] = real ? i : -1;
    s_p[k] = v;
    s_x[k] = real ? bf2f(x[i]) : 0.f;
    tm = fmaxf(tm, v);
  }
  tm = block_max<NT / 64>(tm, red);
  const bool live = tm > -INFINITY && w != 0.f;  // uniform over the workgroup
  if (!live) {
    if (t == 0) loss[row] = 0.f;
    const int V8 = VEC ? V >> 3 : 0;
    for (int i = t; i < V8; i += NT) reinterpret_cast<u32x4*>(gx)[i] = u32x4{0u, 0u, 0u, 0u};
    for (int i = V8 * 8 + t; i < V; i += NT) gx[i] = 0;
    return;
  }
  float ts = 0.f;
  for (int k = t; k < K; k += NT) {
    const float e = s_idx[k] >= 0 ? __builtin_amdgcn_exp2f((s_p[k] - tm) * c) : 0.f;
    ts += e;
  }
  __syncthreads();
  ts = block_sum<NT / 64>(ts, red);
  const float tl2 = __log2f(ts);  // log2 of the teacher's sum
  // student: running maximum and sum
  const int V8 = VEC ? V >> 3 : 0;
  const u32x4* xv = reinterpret_cast<const u32x4*>(x);
  float m = -INFINITY, s = 0.f;
  for (int i = t; i < V8; i += NT) {
    float f[8];
    unpack8(xv[i], f);
    const float cm = fmaxf(fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])), fmaxf(fmaxf(f[4], f[5]), fmaxf(f[6], f[7])));
    const float nm = fmaxf(m, cm);
    if (nm == -INFINITY) continue;
    const float nb = -nm * c;
    float add = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) add += __builtin_amdgcn_exp2f(fmaf(f[e], c, nb));
    s = (m == -INFINITY ? 0.f : s * __builtin_amdgcn_exp2f((m - nm) * c)) + add;
    m = nm;
  }
  for (int i = V8 * 8 + t; i < V; i += NT) {
    const float f = bf2f(x[i]);
    const float nm = fmaxf(m, f);
    if (nm == -INFINITY) continue;
    s = (m == -INFINITY ? 0.f : s * __builtin_amdgcn_exp2f((m - nm) * c)) + __builtin_amdgcn_exp2f((f - nm) * c);
    m = nm;
  }
  __syncthreads();
  const float M = block_max<NT / 64>(m, red);
  __syncthreads();
  s = block_sum<NT / 64>(m == -INFINITY ? 0.f : s * __builtin_amdgcn_exp2f((m - M) * c), red);
  const bool some = M > -INFINITY;                              // false: every logit is -inf, q = 0
  const float lse2 = some ? fmaf(M, c, __log2f(s)) : INFINITY;  // log2 of the student's sum of exp(logit / t)
  // loss: p_k (log2 p_k - log2 q_k) summed, in nats at the end
  float part = 0.f;
  for (int k = t; k < K; k += NT) {
    if (s_idx[k] < 0) {
      s_p[k] = 0.f;
      continue;
    }
    const float lp = (s_p[k] - tm) * c - tl2;
    const float p = __builtin_amdgcn_exp2f(lp);
    s_p[k] = p;
    const float lq = some ? fmaf(s_x[k], c, -lse2) : -INFINITY;
    if (p > 0.f) part += p * (lp - lq);
  }
  __syncthreads();
  part = block_sum<NT / 64>(part, red);
  if (t == 0) loss[row] = part * kLn2 * temp * temp * w;
  // gradient: t w q for every logit, then the listed tokens' own elements
  const float gw = temp * w;
  u32x4* gv = reinterpret_cast<u32x4*>(gx);
  for (int i = t; i < V8; i += NT) {
    float f[8];
    unpack8(xv[i], f);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = gw * __builtin_amdgcn_exp2f(fmaf(f[e], c, -lse2));
    gv[i] = pack8(f);
  }
  for (int i = V8 * 8 + t; i < V; i += NT) gx[i] = f2bf(gw * __builtin_amdgcn_exp2f(fmaf(bf2f(x[i]), c, -lse2)));
  __syncthreads();  // every element has been written (and the LDS probabilities are complete)
  for (int k = t; k < K; k += NT) {
    const int i = s_idx[k];
    if (i < 0) continue;
    float p = 0.f;  // a token listed more than once: its entries' sum, written by the first of them
    bool first = true;
    for (int j = 0; j < K; ++j) {
      const bool same = s_idx[j] == i;
      p += same ? s_p[j] : 0.f;
      first = first && !(same && j < k);
    }
    if (first) gx[i] = f2bf(gw * (__builtin_amdgcn_exp2f(fmaf(s_x[k], c, -lse2)) - p));
  }
}

int distill_topk(const bf16_t* logits, int64_t ld, int64_t N, int V, const int* index, const float* teacher, int K,
                 const float* weight, float temp, float* loss, bf16_t* grad, int64_t gld, hipStream_t stream) {
  if (K < 1 || K > kDistillMaxK || V < 1 || N < 0 || N > 0x7fffffff) return -1;
  if (N == 0) return 0;
  const bool vec = ld % 8 == 0 && gld % 8 == 0 && reinterpret_cast<uintptr_t>(logits) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(grad) % 16 == 0;
  if (vec)
    distill_kernel<512, true><<<(unsigned)N, 512, 0, stream>>>(logits, ld, V, index, teacher, K, weight, temp, loss, grad,
                                                              gld);
  else
    distill_kernel<512, false><<<(unsigned)N, 512, 0, stream>>>(logits, ld, V, index, teacher, K, weight, temp, loss,
                                                               grad, gld);
  return hipGetLastError() == hipSuccess ? 0 : -9;
}

}  // namespace kop
