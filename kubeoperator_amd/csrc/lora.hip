// Low-rank adapters of many requests beside one shared projection (serving), for gfx950:
//
//   out[i] = y[i] + scale[j] * b[j] (a[j] x[i]),   j = index[i]        (j outside [0, n): out[i] = y[i])
//   x [M, K], y / out [M, N] bf16 rows; a [n, r, K], b [n, N, r] bf16; index [M] int32; scale [n] fp32
//
// Two launches: the rows' products with a (K split over workgroups, fp32 partials), then their products with b added to y.
// Both take up to 64 rows per workgroup as 16-column operands of v_mfma_f32_16x16x32_bf16, in one of two forms:
//   * by adapter (few rows: a decode step): a workgroup collects the rows of ONE adapter from the index list, so every
//     adapter that occurs is read once, however its rows are scattered; one more "adapter" collects the rows without any;
//   * by rows (many rows: a prefill): consecutive rows, the adapters that occur among them taken one after another
//     (lowest row first), each row keeping the result of its own only -- by selection, not by a zero factor, so a request's
//     NaN weights stay with its own rows.
// The low-rank values enter the second product as a bf16 pair (value and remainder: 2^-16 relative), so the only rounding
// that counts is the output's.
#include <algorithm>

#include "common.h"
#include "kernels.h"

namespace kop {

namespace {
constexpr int kT = 256;
// up to this many rows the index list is scanned by every workgroup
constexpr int kGroupRows = 1024;

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ bf16x8 zero8() { return bf16x8{0, 0, 0, 0, 0, 0, 0, 0}; }
__device__ __forceinline__ bf16x8 ld8(const bf16_t* p) { return *reinterpret_cast<const bf16x8*>(p); }

// 16-row groups per workgroup: fewer at high ranks, for the registers
constexpr int down_groups(int RB) { return RB <= 4 ? 4 : 2; }
constexpr int up_groups(int RS) { return RS <= 2 ? 4 : 2; }

// The rows of a workgroup. By adapter: number z * ROWS ... of the rows with index `aj` (aj = n: of the rows without an
// adapter), in order, in `list`; returns how many there are for this workgroup (0 .. ROWS), in every thread.
template <int ROWS>
__device__ __forceinline__ int collect(const int* __restrict__ index, int M, int n, int aj, int z, int* list, int* s_cnt) {
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
  int before = -z * ROWS;
  for (int i0 = 0; i0 < M; i0 += kT) {
    const int i = i0 + t, j = i < M ? index[i] : aj == n ? 0 : -1;
    const bool hit = i < M && (aj == n ? j < 0 || j >= n : j == aj);
    const uint64_t mask = __ballot(hit);
    if (lane == 0) s_cnt[wv] = __popcll(mask);
    __syncthreads();
    int at = before + __popcll(mask & ((1ull << lane) - 1));
#pragma unroll
    for (int w = 0; w < kT / 64; ++w) {
      at += w < wv ? s_cnt[w] : 0;
      before += s_cnt[w];
    }
    if (hit && at >= 0 && at < ROWS) list[at] = i;
    __syncthreads();
  }
  return min(max(before, 0), ROWS);
}
}  // namespace

// ---- part[split][row][r] = a[index[row]] . x[row] over the split's part of K. By adapter: grid (adapters, splits, lists);
// by rows: grid (tiles, splits). The 4 waves take a quarter of the part each and meet in LDS.
template <int RB, bool GROUP>  // RB: 16-row blocks of the rank
__global__ void __launch_bounds__(kT) lora_down_kernel(const bf16_t* __restrict__ x, int64_t xs,
                                                       const bf16_t* __restrict__ a, const int* __restrict__ index,
                                                       float* __restrict__ part, int64_t M, int K, int n, int r, int kpart) {
  constexpr int NG = down_groups(RB), ROWS = 16 * NG, U = RB == 1 ? 4 : RB == 2 ? 2 : 1;
  __shared__ f32x4 s_acc[RB * NG * 64];
  __shared__ int s_list[ROWS], s_cnt[kT / 64];
  const int t = threadIdx.x, lane = t & 63, col = lane & 15, g = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(t >> 6);
  int64_t row[NG];
  int j[NG], ng;
  if constexpr (GROUP) {
    const int cnt = collect<ROWS>(index, (int)M, n, blockIdx.x, blockIdx.z, s_list, s_cnt);
    if (cnt == 0) return;
    ng = (cnt + 15) / 16;
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      const bool in = 16 * q + col < cnt;
      row[q] = s_list[in ? 16 * q + col : 0];
      j[q] = in ? (int)blockIdx.x : -1;
    }
  } else {
    const int64_t row0 = (int64_t)blockIdx.x * ROWS;
    ng = (int)std::min<int64_t>(NG, (M - row0 + 15) / 16);
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      row[q] = row0 + 16 * q + col;
      const bool in = row[q] < M;
      row[q] = in ? row[q] : M - 1;
      j[q] = in ? index[row[q]] : -1;
      if (j[q] >= n) j[q] = -1;
    }
  }
  const bf16_t* xr[NG];
#pragma unroll
  for (int q = 0; q < NG; ++q) xr[q] = x + row[q] * xs + 8 * g;
  const int k0 = blockIdx.y * kpart, k1 = min(K, k0 + kpart);
  const int per = ((k1 - k0 + 127) / 128) * 32;  // a wave's part, a multiple of the product's 32
  const int w0 = k0 + wv * per, w1 = min(k1, w0 + per);
  f32x4 mine[NG][RB];
#pragma unroll
  for (int q = 0; q < NG; ++q)
#pragma unroll
    for (int i = 0; i < RB; ++i) mine[q][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  uint64_t todo[NG];
#pragma unroll
  for (int q = 0; q < NG; ++q) todo[q] = __ballot(j[q] >= 0) & 0xffffull;
  while (true) {
    int aj = -1;
#pragma unroll
    for (int q = NG - 1; q >= 0; --q)
      if (todo[q]) aj = __builtin_amdgcn_readlane(j[q], __builtin_ctzll(todo[q]));
    if (aj < 0) break;
    const bf16_t* ar = a + ((int64_t)aj * r + col) * K + 8 * g;
    f32x4 acc[NG][RB];
#pragma unroll
    for (int q = 0; q < NG; ++q)
#pragma unroll
      for (int i = 0; i < RB; ++i) acc[q][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    int k = w0;
    for (; k + 32 * U <= w1; k += 32 * U) {
      bf16x8 af[U][RB], xf[U][NG];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < RB; ++i) af[u][i] = 16 * i + col < r ? ld8(ar + (int64_t)16 * i * K + k + 32 * u) : zero8();
#pragma unroll
      for (int q = 0; q < NG; ++q)
        if (q < ng)
#pragma unroll
          for (int u = 0; u < U; ++u) xf[u][q] = ld8(xr[q] + k + 32 * u);
#pragma unroll
      for (int q = 0; q < NG; ++q)
        if (q < ng)
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < RB; ++i) acc[q][i] = mfma16(af[u][i], xf[u][q], acc[q][i]);
    }
    for (; k < w1; k += 32) {
      const bool kin = k + 8 * g < w1;  // K and the parts' ends are multiples of 8
      bf16x8 af[RB];
#pragma unroll
      for (int i = 0; i < RB; ++i) af[i] = kin && 16 * i + col < r ? ld8(ar + (int64_t)16 * i * K + k) : zero8();
#pragma unroll
      for (int q = 0; q < NG; ++q)
        if (q < ng) {
          const bf16x8 xf = kin ? ld8(xr[q] + k) : zero8();
#pragma unroll
          for (int i = 0; i < RB; ++i) acc[q][i] = mfma16(af[i], xf, acc[q][i]);
        }
    }
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      const bool match = j[q] == aj;
      todo[q] &= ~__ballot(match);
#pragma unroll
      for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) mine[q][i][e] = match ? acc[q][i][e] : mine[q][i][e];
    }
  }
  for (int w = 1; w < kT / 64; ++w) {
    __syncthreads();
    if (wv == w) {
#pragma unroll
      for (int q = 0; q < NG; ++q)
#pragma unroll
        for (int i = 0; i < RB; ++i) s_acc[(q * RB + i) * 64 + lane] = mine[q][i];
    }
    __syncthreads();
    if (wv == 0) {
#pragma unroll
      for (int q = 0; q < NG; ++q)
#pragma unroll
        for (int i = 0; i < RB; ++i) {
          const f32x4 o = s_acc[(q * RB + i) * 64 + lane];
#pragma unroll
          for (int e = 0; e < 4; ++e) mine[q][i][e] += o[e];
        }
    }
  }
  if (wv != 0) return;
#pragma unroll
  for (int q = 0; q < NG; ++q) {
    if (j[q] < 0) continue;
    float* p = part + ((int64_t)blockIdx.y * M + row[q]) * r + 4 * g;
#pragma unroll
    for (int i = 0; i < RB; ++i)
      if (16 * i + 4 * g < r) *reinterpret_cast<f32x4*>(p + 16 * i) = mine[q][i];
  }
}

// ---- out[row] = y[row] + scale b[index[row]] . (sum over splits of part). By adapter: grid (adapters + 1, column blocks,
// lists); by rows: grid (tiles, column blocks). A column block is `chunks` times 256 columns, 64 per wave. The 16 b rows
// of product c are columns n0 + 16 (i >> 2) + 4 c + (i & 3): over the 4 products a lane ends up with 16 consecutive
// columns of its row.
template <int RS, bool GROUP>  // RS: 32-steps of the rank
__global__ void __launch_bounds__(kT) lora_up_kernel(const bf16_t* y, int64_t ys, const bf16_t* __restrict__ b,
                                                     const int* __restrict__ index, const float* __restrict__ scale,
                                                     const float* __restrict__ part, int splits, bf16_t* out, int64_t os,
                                                     int64_t M, int N, int n, int r, int chunks) {
  constexpr int NG = up_groups(RS), ROWS = 16 * NG;
  __shared__ int s_list[ROWS], s_cnt[kT / 64];
  const int t = threadIdx.x, lane = t & 63, col = lane & 15, g = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(t >> 6);
  int64_t row[NG];
  int j[NG];
  bool in[NG];
  if constexpr (GROUP) {
    const int aj = blockIdx.x;
    if (aj == n && y == out) return;  // in place: the rows without an adapter are there already
    const int cnt = collect<ROWS>(index, (int)M, n, aj, blockIdx.z, s_list, s_cnt);
    if (cnt == 0) return;
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      in[q] = 16 * q + col < cnt;
      row[q] = s_list[in[q] ? 16 * q + col : 0];
      j[q] = in[q] && aj < n ? aj : -1;
    }
  } else {
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      row[q] = (int64_t)blockIdx.x * ROWS + 16 * q + col;
      in[q] = row[q] < M;
      row[q] = in[q] ? row[q] : M - 1;
      j[q] = in[q] ? index[row[q]] : -1;
      if (j[q] >= n) j[q] = -1;
    }
  }
  // the rows' low-rank values, scaled, as a bf16 value and its remainder: k = 32 s + 8 g .. +7
  bf16x8 hi[NG][RS], lo[NG][RS];
#pragma unroll
  for (int q = 0; q < NG; ++q)
#pragma unroll
    for (int s = 0; s < RS; ++s) {
      hi[q][s] = lo[q][s] = zero8();
      const int k = 32 * s + 8 * g;
      if (j[q] >= 0 && k < r) {
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int c = 0; c < splits; ++c) {
          const f32x4* p = reinterpret_cast<const f32x4*>(part + ((int64_t)c * M + row[q]) * r + k);
          const f32x4 p0 = p[0], p1 = p[1];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e] += p0[e];
            v[4 + e] += p1[e];
          }
        }
        const float sc = scale[j[q]];
        float h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= sc;
        const u32x4 hp = pack8(v);
        unpack8(hp, h);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = fabsf(h[e]) < INFINITY ? v[e] - h[e] : 0.f;
        hi[q][s] = __builtin_bit_cast(bf16x8, hp);
        lo[q][s] = __builtin_bit_cast(bf16x8, pack8(h));
      }
    }
  for (int ch = 0; ch < chunks; ++ch) {
    const int n0 = (blockIdx.y * chunks + ch) * 256 + wv * 64;
    if (n0 >= N) break;
    u32x4 yv[NG][2];
#pragma unroll
    for (int q = 0; q < NG; ++q)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (in[q] && n0 + 16 * g + 8 * h < N)
          yv[q][h] = *reinterpret_cast<const u32x4*>(y + row[q] * ys + n0 + 16 * g + 8 * h);
    f32x4 mine[NG][4];
#pragma unroll
    for (int q = 0; q < NG; ++q)
#pragma unroll
      for (int c = 0; c < 4; ++c) mine[q][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    uint64_t todo[NG];
#pragma unroll
    for (int q = 0; q < NG; ++q) todo[q] = __ballot(j[q] >= 0) & 0xffffull;
    while (true) {
      int aj = -1;
#pragma unroll
      for (int q = NG - 1; q >= 0; --q)
        if (todo[q]) aj = __builtin_amdgcn_readlane(j[q], __builtin_ctzll(todo[q]));
      if (aj < 0) break;
      bf16x8 bf[4][RS];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int nr = n0 + 16 * (col >> 2) + 4 * c + (col & 3);
        const bf16_t* br = b + ((int64_t)aj * N + nr) * r + 8 * g;
#pragma unroll
        for (int s = 0; s < RS; ++s) bf[c][s] = nr < N && 32 * s + 8 * g < r ? ld8(br + 32 * s) : zero8();
      }
#pragma unroll
      for (int q = 0; q < NG; ++q) {
        const bool match = j[q] == aj;
        const uint64_t some = __ballot(match);
        if (!some) continue;
        todo[q] &= ~some;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < RS; ++s) {
            acc = mfma16(bf[c][s], lo[q][s], acc);
            acc = mfma16(bf[c][s], hi[q][s], acc);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) mine[q][c][e] = match ? acc[e] : mine[q][c][e];
        }
      }
    }
#pragma unroll
    for (int q = 0; q < NG; ++q)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (!in[q] || n0 + 16 * g + 8 * h >= N) continue;
        u32x4 v = yv[q][h];
        if (j[q] >= 0) {
          float f[8];
          unpack8(v, f);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            f[e] += mine[q][2 * h][e];
            f[4 + e] += mine[q][2 * h + 1][e];
          }
          v = pack8(f);
        }
        *reinterpret_cast<u32x4*>(out + row[q] * os + n0 + 16 * g + 8 * h) = v;
      }
  }
}

namespace {
struct Plan {
  bool group;
  int splits, kpart;           // parts of K
  unsigned dgx, dgz, ugx, ugz;  // workgroups of each launch besides its splits / column blocks
  int chunks, blocks;          // 256-column chunks per column block, column blocks
};
Plan make_plan(int64_t M, int K, int N, int n, int r) {
  Plan p;
  p.group = M <= kGroupRows;
  const int drows = 16 * down_groups((r + 15) / 16), urows = 16 * up_groups((r + 31) / 32);
  const int64_t dt = (M + drows - 1) / drows, ut = (M + urows - 1) / urows;
  p.dgx = (unsigned)(p.group ? n : dt), p.dgz = (unsigned)(p.group ? dt : 1);
  p.ugx = (unsigned)(p.group ? n + 1 : ut), p.ugz = (unsigned)(p.group ? ut : 1);
  // workgroups that have rows: adapters cannot outnumber rows
  const int64_t dw = p.group ? std::min<int64_t>(M, n) : dt, uw = p.group ? std::min<int64_t>(M, n) : ut;
  p.splits = 1;
  while (p.splits < 16 && dw * p.splits < 256 && K / (2 * p.splits) >= 256) p.splits *= 2;
  p.kpart = ((K + p.splits - 1) / p.splits + 31) & ~31;
  const int nc = (N + 255) / 256;
  p.chunks = (int)std::max<int64_t>(1, std::min<int64_t>(8, uw * nc / 1024));
  p.blocks = (nc + p.chunks - 1) / p.chunks;
  return p;
}
}  // namespace

int64_t lora_workspace(int64_t M, int K, int N, int n, int r) { return (int64_t)make_plan(M, K, N, n, r).splits * M * r * 4; }

int lora_add(const bf16_t* y, int64_t ys, const bf16_t* x, int64_t xs, const bf16_t* a, const bf16_t* b,
             const int* index, const float* scale, bf16_t* out, int64_t os, int64_t M, int K, int N, int n, int r,
             void* workspace, hipStream_t stream) {
  if (K < 8 || K % 8 || N < 8 || N % 8 || r < 8 || r % 8 || r > kLoraMaxRank || n < 0 || M < 0 || xs % 8 || ys % 8 ||
      os % 8 || (M + 31) / 32 > 0x7fffffff || (N + 255) / 256 > 65535)
    return -1;
  if (M == 0) return 0;
  const Plan p = make_plan(M, K, N, n, r);
  float* part = reinterpret_cast<float*>(workspace);
  const dim3 gd(p.dgx, p.splits, p.dgz), gu(p.ugx, p.blocks, p.ugz);
#define KOP_DOWN(RB)                                                                                             \
  case RB:                                                                                                       \
    if (p.group) lora_down_kernel<RB, true><<<gd, kT, 0, stream>>>(x, xs, a, index, part, M, K, n, r, p.kpart);  \
    else lora_down_kernel<RB, false><<<gd, kT, 0, stream>>>(x, xs, a, index, part, M, K, n, r, p.kpart);         \
    break;
  if (n > 0) switch ((r + 15) / 16) {
      KOP_DOWN(1) KOP_DOWN(2) KOP_DOWN(3) KOP_DOWN(4) KOP_DOWN(5) KOP_DOWN(6) KOP_DOWN(7) KOP_DOWN(8)
    }
#undef KOP_DOWN
#define KOP_UP(RS)                                                                                                  \
  case RS:                                                                                                          \
    if (p.group)                                                                                                    \
      lora_up_kernel<RS, true><<<gu, kT, 0, stream>>>(y, ys, b, index, scale, part, p.splits, out, os, M, N, n, r,  \
                                                      p.chunks);                                                    \
    else                                                                                                            \
      lora_up_kernel<RS, false><<<gu, kT, 0, stream>>>(y, ys, b, index, scale, part, p.splits, out, os, M, N, n, r, \
                                                       p.chunks);                                                   \
    break;
  switch ((r + 31) / 32) { KOP_UP(1) KOP_UP(2) KOP_UP(3) KOP_UP(4) }
#undef KOP_UP
  return hipGetLastError() == hipSuccess ? 0 : -9;
}

}  // namespace kop
