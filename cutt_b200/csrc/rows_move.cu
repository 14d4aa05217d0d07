// Rows moved by the expert map: one token's row to its slots' rows (scatter: dispatch and the
// gradient of combine) and the sum of its slots' rows (gather: combine and the gradient of
// dispatch), with the gradient of the weights on the way.
//
// Both walk over tokens, so the token side is read or written once and the k-fold side once: the
// fewest bytes there are.  A team of threads (a warp, or a block where there are few tokens) owns a
// token, or a part of its row; every thread holds one access of the token's row and goes through
// the token's slots.  Sums are in 32 bits in the order of the slots, rounded once, so results do
// not depend on the launch shape.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "kernels.h"
#include "rows.h"

namespace cuttb {

namespace {

template <int VB> struct Raw;
template <> struct Raw<16> { typedef uint4 T; };
template <> struct Raw<8> { typedef uint2 T; };
template <> struct Raw<4> { typedef uint32_t T; };
template <> struct Raw<2> { typedef uint16_t T; };
template <> struct Raw<1> { typedef uint8_t T; };

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(uint8_t) { return 0.f; }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ uint8_t from_f<uint8_t>(float) { return 0; }

// VB bytes as elements.
template <typename T, int VB>
union Piece {
  static constexpr int N = VB / (int)sizeof(T);
  typename Raw<VB>::T raw;
  T e[N];
  __device__ Piece() {}
};

template <int TEAM>
__device__ __forceinline__ float team_sum(float v, float* s) {
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if (TEAM == 32) return v;
  const int w = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) s[w] = v;
  __syncthreads();
  float t = 0.f;
  for (int i = 0; i < TEAM / 32; i++) t += s[i];
  __syncthreads();
  return t;
}

constexpr int kThreads = 256;
constexpr int kPadBlocks = 4;    // blocks per expert that clear padding rows

// grid.x: blocks of padding (experts * kPadBlocks of them, or none), then blocks of teams;
// grid.y: parts of a row.
template <typename T, int VB, int KU, int TEAM, bool WEIGHT, bool DOT>
__global__ void __launch_bounds__(kThreads) scatter_kernel(const __grid_constant__ RowsMove m, int padBlocks) {
  typedef typename Raw<VB>::T R;
  __shared__ float scratch[kThreads / 32];
  const int vecs = m.width * (int)sizeof(T) / VB;
  const int part = (vecs + gridDim.y - 1) / gridDim.y;
  const int v0 = blockIdx.y * part, v1 = min(vecs, v0 + part);
  if ((int)blockIdx.x < padBlocks) {
    const int e = blockIdx.x / kPadBlocks;
    const int from = m.offset[e] + m.count[e], to = min(m.offset[e + 1], m.capacity);
    R zero = {};
    for (int r = max(0, from) + blockIdx.x % kPadBlocks; r < to; r += kPadBlocks) {
      R* y = (R*)(m.row + (long long)r * m.rowStride);
      for (int v = v0 + threadIdx.x; v < v1; v += kThreads) y[v] = zero;
    }
    return;
  }
  const int lane = threadIdx.x % TEAM;
  const int t = (blockIdx.x - padBlocks) * (kThreads / TEAM) + threadIdx.x / TEAM;
  if (t >= m.tokens) return;      // whole teams leave
  const R* x = (const R*)(m.token + (long long)t * m.tokenStride);
  const long long s0 = (long long)t * m.choices;
  for (int j0 = 0; j0 < m.choices; j0 += KU) {
    int row[KU];
    float w[KU], dot[KU];
#pragma unroll
    for (int j = 0; j < KU; j++) {
      row[j] = j0 + j < m.choices ? m.rowOf[s0 + j0 + j] : -1;
      if ((unsigned)row[j] >= (unsigned)m.capacity) row[j] = -1;
      w[j] = WEIGHT && row[j] >= 0 ? m.weight[s0 + j0 + j] : 1.f;
      dot[j] = 0.f;
    }
    for (int v = v0 + lane; v < v1; v += TEAM) {
      Piece<T, VB> a, o[DOT ? KU : 1];
      a.raw = x[v];
      if (DOT) {
#pragma unroll
        for (int j = 0; j < KU; j++)
          if (row[j] >= 0) o[j].raw = ((const R*)(m.other + (long long)row[j] * m.otherStride))[v];
      }
#pragma unroll
      for (int j = 0; j < KU; j++) {
        if (row[j] < 0) continue;
        Piece<T, VB> b;
        if (WEIGHT) {
#pragma unroll
          for (int i = 0; i < b.N; i++) b.e[i] = from_f<T>(to_f(a.e[i]) * w[j]);
        } else {
          b.raw = a.raw;
        }
        ((R*)(m.row + (long long)row[j] * m.rowStride))[v] = b.raw;
        if (DOT) {
#pragma unroll
          for (int i = 0; i < b.N; i++) dot[j] = fmaf(to_f(a.e[i]), to_f(o[DOT ? j : 0].e[i]), dot[j]);
        }
      }
    }
    if (DOT) {
#pragma unroll
      for (int j = 0; j < KU; j++) {
        const float d = team_sum<TEAM>(dot[j], scratch);
        if (lane == 0 && j0 + j < m.choices) m.dweight[s0 + j0 + j] = d;
      }
    }
  }
}

template <typename T, int VB, int KU, int TEAM, bool WEIGHT, bool DOT>
__global__ void __launch_bounds__(kThreads) gather_kernel(const __grid_constant__ RowsMove m) {
  typedef typename Raw<VB>::T R;
  __shared__ float scratch[kThreads / 32];
  const int vecs = m.width * (int)sizeof(T) / VB;
  const int part = (vecs + gridDim.y - 1) / gridDim.y;
  const int v0 = blockIdx.y * part, v1 = min(vecs, v0 + part);
  const int lane = threadIdx.x % TEAM;
  const int t = blockIdx.x * (kThreads / TEAM) + threadIdx.x / TEAM;
  if (t >= m.tokens) return;
  R* out = (R*)(m.token + (long long)t * m.tokenStride);
  const R* x = (const R*)(m.other + (long long)t * m.otherStride);
  const long long s0 = (long long)t * m.choices;
  // More choices than KU: the slots are gone through in groups, and a thread keeps the sum of its
  // access in registers over all groups (one access at a time); the weights' gradient is taken
  // group by group.
  const bool one = m.choices <= KU;
  for (int j0 = 0; j0 < m.choices; j0 += KU) {
    int row[KU];
    float w[KU], dot[KU];
#pragma unroll
    for (int j = 0; j < KU; j++) {
      row[j] = j0 + j < m.choices ? m.rowOf[s0 + j0 + j] : -1;
      if ((unsigned)row[j] >= (unsigned)m.capacity) row[j] = -1;
      w[j] = WEIGHT && row[j] >= 0 ? m.weight[s0 + j0 + j] : 1.f;
      dot[j] = 0.f;
    }
    if (one || DOT) {
      for (int v = v0 + lane; v < v1; v += TEAM) {
        Piece<T, VB> b[KU], a;
        float sum[Piece<T, VB>::N];
#pragma unroll
        for (int i = 0; i < a.N; i++) sum[i] = 0.f;
#pragma unroll
        for (int j = 0; j < KU; j++)
          if (row[j] >= 0) b[j].raw = ((const R*)(m.row + (long long)row[j] * m.rowStride))[v];
        if (DOT) a.raw = x[v];
#pragma unroll
        for (int j = 0; j < KU; j++) {
          if (row[j] < 0) continue;
#pragma unroll
          for (int i = 0; i < a.N; i++) {
            const float f = to_f(b[j].e[i]);
            sum[i] = WEIGHT ? fmaf(w[j], f, sum[i]) : sum[i] + f;
            if (DOT) dot[j] = fmaf(f, to_f(a.e[i]), dot[j]);
          }
        }
        if (one) {
          Piece<T, VB> r;
#pragma unroll
          for (int i = 0; i < r.N; i++) r.e[i] = from_f<T>(sum[i]);
          out[v] = r.raw;
        }
      }
    }
    if (DOT) {
#pragma unroll
      for (int j = 0; j < KU; j++) {
        const float d = team_sum<TEAM>(dot[j], scratch);
        if (lane == 0 && j0 + j < m.choices) m.dweight[s0 + j0 + j] = d;
      }
    }
  }
  if (one) return;
  for (int v = v0 + lane; v < v1; v += TEAM) {
    float sum[Piece<T, VB>::N];
#pragma unroll
    for (int i = 0; i < Piece<T, VB>::N; i++) sum[i] = 0.f;
    for (int j0 = 0; j0 < m.choices; j0 += KU) {
      Piece<T, VB> b[KU];
      int row[KU];
#pragma unroll
      for (int j = 0; j < KU; j++) {
        row[j] = j0 + j < m.choices ? m.rowOf[s0 + j0 + j] : -1;
        if ((unsigned)row[j] >= (unsigned)m.capacity) row[j] = -1;
        if (row[j] >= 0) b[j].raw = ((const R*)(m.row + (long long)row[j] * m.rowStride))[v];
      }
#pragma unroll
      for (int j = 0; j < KU; j++) {
        if (row[j] < 0) continue;
        const float w = WEIGHT ? m.weight[s0 + j0 + j] : 1.f;
#pragma unroll
        for (int i = 0; i < b[j].N; i++) {
          const float f = to_f(b[j].e[i]);
          sum[i] = WEIGHT ? fmaf(w, f, sum[i]) : sum[i] + f;
        }
      }
    }
    Piece<T, VB> r;
#pragma unroll
    for (int i = 0; i < r.N; i++) r.e[i] = from_f<T>(sum[i]);
    out[v] = r.raw;
  }
}

struct Shape {
  dim3 grid;
  int team;
};

// A warp per token where that fills the GPU; else a block per token, and (where no sum runs along
// the row) several blocks.
Shape shape_for(const RowsMove& m, int vecs, bool dot, int numSM) {
  Shape s;
  const long long warps = m.tokens;
  s.team = warps >= (long long)numSM * 32 ? 32 : kThreads;
  const int perBlock = kThreads / s.team;
  s.grid = dim3((unsigned)((m.tokens + perBlock - 1) / perBlock), 1, 1);
  if (!dot && s.team == kThreads) {
    int parts = (vecs + kThreads - 1) / kThreads;
    if (parts > 8) parts = 8;
    s.grid.y = parts;
  }
  return s;
}

template <typename T, int VB, int KU, int TEAM>
void scatter_flags(const RowsMove& m, dim3 grid, int pad, cudaStream_t stream) {
  const bool w = m.weight != nullptr, d = m.dweight != nullptr;
  if (sizeof(T) == 1) {
    scatter_kernel<T, VB, KU, TEAM, false, false><<<grid, kThreads, 0, stream>>>(m, pad);
    return;
  }
  if (w && d) scatter_kernel<T, VB, KU, TEAM, true, true><<<grid, kThreads, 0, stream>>>(m, pad);
  else if (w) scatter_kernel<T, VB, KU, TEAM, true, false><<<grid, kThreads, 0, stream>>>(m, pad);
  else if (d) scatter_kernel<T, VB, KU, TEAM, false, true><<<grid, kThreads, 0, stream>>>(m, pad);
  else scatter_kernel<T, VB, KU, TEAM, false, false><<<grid, kThreads, 0, stream>>>(m, pad);
}

template <typename T, int VB, int KU, int TEAM>
void gather_flags(const RowsMove& m, dim3 grid, cudaStream_t stream) {
  const bool w = m.weight != nullptr, d = m.dweight != nullptr;
  if (w && d) gather_kernel<T, VB, KU, TEAM, true, true><<<grid, kThreads, 0, stream>>>(m);
  else if (w) gather_kernel<T, VB, KU, TEAM, true, false><<<grid, kThreads, 0, stream>>>(m);
  else if (d) gather_kernel<T, VB, KU, TEAM, false, true><<<grid, kThreads, 0, stream>>>(m);
  else gather_kernel<T, VB, KU, TEAM, false, false><<<grid, kThreads, 0, stream>>>(m);
}

template <typename T, int VB>
cudaError_t move_vec(const RowsMove& m, bool scatter, int pad, int numSM, cudaStream_t stream) {
  const Shape s = shape_for(m, m.width * (int)sizeof(T) / VB, m.dweight != nullptr, numSM);
  dim3 g = s.grid;
  if (scatter) {
    g.x += pad;
    if (g.x == 0) return cudaSuccess;
    if (s.team == 32) {
      if (m.choices <= 4) scatter_flags<T, VB, 4, 32>(m, g, pad, stream);
      else scatter_flags<T, VB, 8, 32>(m, g, pad, stream);
    } else {
      if (m.choices <= 4) scatter_flags<T, VB, 4, kThreads>(m, g, pad, stream);
      else scatter_flags<T, VB, 8, kThreads>(m, g, pad, stream);
    }
  } else {
    if (g.x == 0) return cudaSuccess;
    if constexpr (sizeof(T) > 1) {
      if (s.team == 32) {
        if (m.choices <= 4) gather_flags<T, VB, 4, 32>(m, g, stream);
        else gather_flags<T, VB, 8, 32>(m, g, stream);
      } else {
        if (m.choices <= 4) gather_flags<T, VB, 4, kThreads>(m, g, stream);
        else gather_flags<T, VB, 8, kThreads>(m, g, stream);
      }
    }
  }
  count_launch();
  return cudaGetLastError();
}

template <typename T>
cudaError_t move_typed(const RowsMove& m, bool scatter, int pad, int numSM, cudaStream_t stream) {
  unsigned long long bits = (uintptr_t)m.token | (uintptr_t)m.row | (uintptr_t)m.other | (unsigned long long)m.tokenStride |
                            (unsigned long long)m.rowStride | (unsigned long long)(m.width * (long long)sizeof(T));
  if (m.other) bits |= (unsigned long long)m.otherStride;
  if (access_bytes(bits, sizeof(T)) == 16) return move_vec<T, 16>(m, scatter, pad, numSM, stream);
  return move_vec<T, sizeof(T)>(m, scatter, pad, numSM, stream);
}

cudaError_t move(const RowsMove& m, bool scatter, int pad, int numSM, cudaStream_t stream) {
  switch (m.type) {
    case 0: return move_typed<uint8_t>(m, scatter, pad, numSM, stream);
    case 1: return move_typed<__half>(m, scatter, pad, numSM, stream);
    case 2: return move_typed<__nv_bfloat16>(m, scatter, pad, numSM, stream);
    case 3: return move_typed<float>(m, scatter, pad, numSM, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_rows_scatter(const RowsMove& m, int align, int numSM, cudaStream_t stream) {
  return move(m, true, align > 1 ? m.experts * kPadBlocks : 0, numSM, stream);
}

cudaError_t launch_rows_gather(const RowsMove& m, int numSM, cudaStream_t stream) {
  return move(m, false, 0, numSM, stream);
}

}  // namespace cuttb
