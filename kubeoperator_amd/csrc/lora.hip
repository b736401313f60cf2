// Low-rank adapters of many requests beside one shared projection (serving), for gfx950:
//
//   out[i] = y[i] + scale[j] * b[j] (a[j] x[i]),   j = index[i]        (j outside [0, n): out[i] = y[i])
//   x [M, K], y / out [M, N] bf16 rows; a [n, r, K], b [n, N, r] bf16; index [M] int32; scale [n] fp32
//
// Two launches: the rows' products with a (K split over workgroups, fp32 partials), then their products with b added to y.
// A tile holds 16 consecutive rows; the adapters that occur in it are taken one after another (lowest row first) on the
// matrix cores, and each row keeps the result of its own adapter only -- by selection, not by a zero factor, so a
// request's NaN weights stay with its own rows. The low-rank values enter the second product as a bf16 pair (value and
// remainder: 2^-17 relative), so the only rounding that counts is the output's.
#include "common.h"
#include "kernels.h"

namespace kop {

namespace {
constexpr int kT = 256;

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ bf16x8 zero8() { return bf16x8{0, 0, 0, 0, 0, 0, 0, 0}; }
__device__ __forceinline__ bf16x8 ld8(const bf16_t* p) { return *reinterpret_cast<const bf16x8*>(p); }

// K elements of one workgroup's part: enough workgroups for the chip, at least 256 elements (64 per wave) each
inline int k_splits(int64_t M, int K) {
  const int64_t tiles = (M + 15) / 16;
  int s = 1;
  while (s < 16 && tiles * s < 1024 && K / (2 * s) >= 256) s *= 2;
  return s;
}
}  // namespace

// ---- t[split][row][r] = a[index[row]] . x[row] over the split's part of K. Grid (16-row tiles, splits); the 4 waves
// take a quarter of the part each and meet in LDS.
template <int RB>  // 16-row blocks of the rank
__global__ void __launch_bounds__(kT) lora_down_kernel(const bf16_t* __restrict__ x, int64_t xs,
                                                       const bf16_t* __restrict__ a, const int* __restrict__ index,
                                                       float* __restrict__ part, int64_t M, int K, int n, int r, int kpart) {
  __shared__ f32x4 s_acc[3][RB][64];
  const int t = threadIdx.x, lane = t & 63, col = lane & 15, g = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(t >> 6);
  const int64_t row = (int64_t)blockIdx.x * 16 + col;
  const bool in = row < M;
  int j = in ? index[row] : -1;
  if (j >= n) j = -1;
  const bf16_t* xr = x + (in ? row : M - 1) * xs + 8 * g;
  const int k0 = blockIdx.y * kpart, k1 = min(K, k0 + kpart);
  const int per = ((k1 - k0 + 127) / 128) * 32;  // a wave's part, a multiple of the product's 32
  const int w0 = k0 + wv * per, w1 = min(k1, w0 + per);
  f32x4 mine[RB];
#pragma unroll
  for (int i = 0; i < RB; ++i) mine[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  uint64_t todo = __ballot(j >= 0) & 0xffffull;
  while (todo) {
    const int aj = __builtin_amdgcn_readlane(j, __builtin_ctzll(todo));
    const bool match = j == aj;
    todo &= ~__ballot(match);
    const bf16_t* ar = a + ((int64_t)aj * r + col) * K + 8 * g;
    f32x4 acc[RB];
#pragma unroll
    for (int i = 0; i < RB; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k = w0; k < w1; k += 32) {
      const bool kin = k + 8 * g < w1;  // K and the parts' ends are multiples of 8
      const bf16x8 xf = kin ? ld8(xr + k) : zero8();
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        const bf16x8 af = kin && 16 * i + col < r ? ld8(ar + (int64_t)16 * i * K + k) : zero8();
        acc[i] = mfma16(af, xf, acc[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) mine[i][e] = match ? acc[i][e] : mine[i][e];
  }
  if (wv > 0) {
#pragma unroll
    for (int i = 0; i < RB; ++i) s_acc[wv - 1][i][lane] = mine[i];
  }
  __syncthreads();
  if (wv == 0 && j >= 0) {
    float* p = part + ((int64_t)blockIdx.y * M + row) * r + 4 * g;
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      if (16 * i + 4 * g >= r) continue;
      f32x4 v = mine[i];
#pragma unroll
      for (int w = 0; w < 3; ++w) {
        const f32x4 o = s_acc[w][i][lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += o[e];
      }
      *reinterpret_cast<f32x4*>(p + 16 * i) = v;
    }
  }
}

// ---- out[row] = y[row] + scale b[index[row]] . (sum over splits of t). Grid (16-row tiles, ceil(N / 256)), 64 columns per
// wave. The 16 b rows of product c are columns n0 + 16 (i >> 2) + 4 c + (i & 3): over the 4 products a lane ends up with
// 16 consecutive columns of its row.
template <int RS>  // 32-steps of the rank
__global__ void __launch_bounds__(kT) lora_up_kernel(const bf16_t* y, int64_t ys, const bf16_t* __restrict__ b,
                                                     const int* __restrict__ index, const float* __restrict__ scale,
                                                     const float* __restrict__ part, int splits, bf16_t* out, int64_t os,
                                                     int64_t M, int N, int n, int r) {
  const int t = threadIdx.x, lane = t & 63, col = lane & 15, g = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(t >> 6);
  const int64_t row = (int64_t)blockIdx.x * 16 + col;
  const int n0 = blockIdx.y * 256 + wv * 64;
  if (n0 >= N) return;
  const bool in = row < M;
  int j = in ? index[row] : -1;
  if (j >= n) j = -1;
  // the row's low-rank values, scaled, as a bf16 value and its remainder: k = 32 s + 8 g .. +7
  bf16x8 hi[RS], lo[RS];
#pragma unroll
  for (int s = 0; s < RS; ++s) {
    hi[s] = lo[s] = zero8();
    const int k = 32 * s + 8 * g;
    if (j >= 0 && k < r) {
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int c = 0; c < splits; ++c) {
        const f32x4* p = reinterpret_cast<const f32x4*>(part + ((int64_t)c * M + row) * r + k);
        const f32x4 p0 = p[0], p1 = p[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] += p0[e];
          v[4 + e] += p1[e];
        }
      }
      const float sc = scale[j];
      float h[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= sc;
      const u32x4 hp = pack8(v);
      unpack8(hp, h);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = fabsf(h[e]) < INFINITY ? v[e] - h[e] : 0.f;
      hi[s] = __builtin_bit_cast(bf16x8, hp);
      lo[s] = __builtin_bit_cast(bf16x8, pack8(h));
    }
  }
  f32x4 mine[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) mine[c] = f32x4{0.f, 0.f, 0.f, 0.f};
  uint64_t todo = __ballot(j >= 0) & 0xffffull;
  while (todo) {
    const int aj = __builtin_amdgcn_readlane(j, __builtin_ctzll(todo));
    const bool match = j == aj;
    todo &= ~__ballot(match);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int nr = n0 + 16 * (col >> 2) + 4 * c + (col & 3);
      const bf16_t* br = b + ((int64_t)aj * N + nr) * r + 8 * g;
      f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < RS; ++s) {
        const bf16x8 bf = nr < N && 32 * s + 8 * g < r ? ld8(br + 32 * s) : zero8();
        acc = mfma16(bf, lo[s], acc);
        acc = mfma16(bf, hi[s], acc);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) mine[c][e] = match ? acc[e] : mine[c][e];
    }
  }
  if (!in) return;
  const bf16_t* yr = y + row * ys + n0 + 16 * g;
  bf16_t* orow = out + row * os + n0 + 16 * g;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (n0 + 16 * g + 8 * h >= N) continue;
    u32x4 v = *reinterpret_cast<const u32x4*>(yr + 8 * h);
    if (j >= 0) {
      float f[8];
      unpack8(v, f);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[e] += mine[2 * h][e];
        f[4 + e] += mine[2 * h + 1][e];
      }
      v = pack8(f);
    }
    *reinterpret_cast<u32x4*>(orow + 8 * h) = v;
  }
}

int64_t lora_workspace(int64_t M, int K, int r) { return (int64_t)k_splits(M, K) * M * r * 4; }

int lora_add(const bf16_t* y, int64_t ys, const bf16_t* x, int64_t xs, const bf16_t* a, const bf16_t* b,
             const int* index, const float* scale, bf16_t* out, int64_t os, int64_t M, int K, int N, int n, int r,
             void* workspace, hipStream_t stream) {
  if (K < 8 || K % 8 || N < 8 || N % 8 || r < 8 || r % 8 || r > kLoraMaxRank || n < 0 || M < 0 || xs % 8 || ys % 8 ||
      os % 8 || (M + 15) / 16 > 0x7fffffff || (N + 255) / 256 > 65535)
    return -1;
  if (M == 0) return 0;
  const int splits = k_splits(M, K);
  const int kpart = ((K + splits - 1) / splits + 31) & ~31;
  float* part = reinterpret_cast<float*>(workspace);
  const dim3 gd((unsigned)((M + 15) / 16), splits), gu((unsigned)((M + 15) / 16), (N + 255) / 256);
#define KOP_DOWN(RB)                                                                                           \
  case RB:                                                                                                     \
    lora_down_kernel<RB><<<gd, kT, 0, stream>>>(x, xs, a, index, part, M, K, n, r, kpart);                     \
    break;
  switch ((r + 15) / 16) {
    KOP_DOWN(1) KOP_DOWN(2) KOP_DOWN(3) KOP_DOWN(4) KOP_DOWN(5) KOP_DOWN(6) KOP_DOWN(7) KOP_DOWN(8)
  }
#undef KOP_DOWN
#define KOP_UP(RS)                                                                                             \
  case RS:                                                                                                     \
    lora_up_kernel<RS><<<gu, kT, 0, stream>>>(y, ys, b, index, scale, part, splits, out, os, M, N, n, r);      \
    break;
  switch ((r + 31) / 32) { KOP_UP(1) KOP_UP(2) KOP_UP(3) KOP_UP(4) }
#undef KOP_UP
  return hipGetLastError() == hipSuccess ? 0 : -9;
}

}  // namespace kop
