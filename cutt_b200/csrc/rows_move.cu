// Rows moved by the expert map: one token's row to its slots' rows (scatter: dispatch and the
// gradient of combine) and the sum of its slots' rows (gather: combine and the gradient of
// dispatch), with the gradient of the weights on the way.
//
// Both walk over tokens, so the token side is read or written once and the k-fold side once: the
// fewest bytes there are.  (From memory: a token's row is read again for each four or eight of its slots,
// which finds it in the cache, and with more than 16 choices sums with the weights' gradient take a walk
// over the rows for the gradient and one for the sums.)  A block owns a token, or a part of its row; every
// thread holds one access of the token's row and goes through the token's slots.  Sums over slots are in
// 32 bits in the order of the slots, rounded once, so they do not depend on the launch shape.  The weights'
// gradients are sums along the row, made by a block's threads together: their order, and with it the last
// bits, depends on the number of threads, which is chosen from the tokens, the row's length and the SMs, and
// on the alignment of the rows.  The same call gives the same bits.
//
// What bounds them is memory: 16384 tokens to 8 rows of 8 KB (bf16) take 188 us, 6.4 TB/s, which is
// what a copy reaches.  Blocks of one token that end soon, many of them on an SM, do best: teams that
// stay and go over the tokens with the next one's slots prefetched took 238 us there, and a warp for a
// token 236.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "rows.h"

namespace cuttb {

namespace {

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(uint8_t) { return 0.f; }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ uint8_t from_f<uint8_t>(float) { return 0; }

// 16 bytes as elements.
template <typename T>
union Piece {
  static constexpr int N = 16 / (int)sizeof(T);
  uint4 raw;
  uint32_t w[4];
  T e[N];
  __device__ Piece() {}
};

// 16 bytes that start m bytes (0 .. 15) into the 32 of x and y.
__device__ __forceinline__ uint4 shift_bytes(const uint4& x, const uint4& y, int m) {
  uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
  if (m & 8) {
#pragma unroll
    for (int i = 0; i < 6; i++) w[i] = w[i + 2];
  }
  if (m & 4) {
#pragma unroll
    for (int i = 0; i < 5; i++) w[i] = w[i + 1];
  }
  const int sh = (m & 3) * 8;
  return make_uint4(__funnelshift_r(w[0], w[1], sh), __funnelshift_r(w[1], w[2], sh), __funnelshift_r(w[2], w[3], sh),
                    __funnelshift_r(w[3], w[4], sh));
}

// Rows are marked as not to be used again (ld.cs, st.cs): most moves are larger than the cache, and
// lines so marked make room for one another.  Gradients of 16384 tokens, 4 KB rows, half of 8 slots
// each dropped: 182 instead of 200 us; sums of 1024 x 8 rows 15.7 instead of 17.5.
__device__ __forceinline__ uint4 load_16(const unsigned char* a) { return __ldcs((const uint4*)a); }
__device__ __forceinline__ void store_16(unsigned char* a, const uint4& v) { __stcs((uint4*)a, v); }

// Rows at any address.  Bytes lo .. lo+15 of a row lie in two aligned 16-byte words.  Where lo grows
// by 16 from lane to lane, the second word is the first of the lane above: every lane loads one and
// gets the other by shuffle, and the last lane has no piece of its own.  (Both words loaded by every
// lane need twice the registers: sums over 8 rows of 2001 bf16 for 16384 tokens took 245 us that
// way, 163 this way.)
//
// The word in which byte lo lies: a single access if it lies in the tensor, which `near` (the row
// is within 16 bytes of the tensor's ends) tells; else, and beyond the row, what the row has of it.
__device__ __forceinline__ bool near_end(long long row, long long rows, long long stride) {
  return row * stride < 16 || (rows - 1 - row) * stride < 16;
}
template <typename T>
__device__ __forceinline__ uint4 load_word(const unsigned char* row, int lo, int bytes, bool near) {
  const int at = lo - (int)((uintptr_t)(row + lo) & 15);          // where the word begins, from the row's start
  Piece<T> p;
  p.raw = make_uint4(0, 0, 0, 0);
  if (at < bytes && at > -16) {
    if (!near || (at >= 0 && at + 16 <= bytes)) {
      p.raw = load_16(row + at);
    } else {
#pragma unroll
      for (int i = 0; i < p.N; i++) {
        const int e = at + i * (int)sizeof(T);
        if (e >= 0 && e < bytes) p.e[i] = *(const T*)(row + e);
      }
    }
  }
  return p.raw;
}
// The word of the lane above (d = 1) or below (d = -1).
__device__ __forceinline__ uint4 word_of(const uint4& w, int d) {
  uint4 r;
  if (d > 0) {
    r.x = __shfl_down_sync(0xffffffffu, w.x, 1);
    r.y = __shfl_down_sync(0xffffffffu, w.y, 1);
    r.z = __shfl_down_sync(0xffffffffu, w.z, 1);
    r.w = __shfl_down_sync(0xffffffffu, w.w, 1);
  } else {
    r.x = __shfl_up_sync(0xffffffffu, w.x, 1);
    r.y = __shfl_up_sync(0xffffffffu, w.y, 1);
    r.z = __shfl_up_sync(0xffffffffu, w.z, 1);
    r.w = __shfl_up_sync(0xffffffffu, w.w, 1);
  }
  return r;
}
// The piece from this lane's word and the next one's.
__device__ __forceinline__ uint4 join_words(const uint4& w, const unsigned char* row, int lo) {
  return shift_bytes(w, word_of(w, 1), (int)((uintptr_t)(row + lo) & 15));
}
// Elements that are not the row's own become zero (they count in sums along the row).
template <typename T>
__device__ __forceinline__ void clear_outside(Piece<T>& p, int lo, int bytes) {
  if (lo >= 0 && lo + 16 <= bytes) return;
#pragma unroll
  for (int i = 0; i < p.N; i++) {
    const int at = lo + i * (int)sizeof(T);
    if (at < 0 || at >= bytes) p.e[i] = from_f<T>(0.f);
  }
}

// Bytes by which a row starts behind a 16-byte boundary.
__device__ __forceinline__ int past_boundary(const unsigned char* base, int row, long long stride) {
  return (int)(((unsigned)(uintptr_t)base + (unsigned)row * (unsigned)stride) & 15u);
}

// Stores a piece that starts on a 16-byte boundary: all of it, or the elements that are the row's own.
template <typename T>
__device__ __forceinline__ void store_any(const Piece<T>& p, unsigned char* row, int lo, int bytes) {
  if (lo >= 0 && lo + 16 <= bytes) {
    store_16(row + lo, p.raw);
  } else {
#pragma unroll
    for (int i = 0; i < p.N; i++) {
      const int at = lo + i * (int)sizeof(T);
      if (at >= 0 && at < bytes) *(T*)(row + at) = p.e[i];
    }
  }
}

constexpr int kPadBlocks = 4;    // blocks per expert that clear padding rows

// Sums K values over the block and writes value j to dweight[j], j < n.  Within a warp every step
// halves the values a lane holds (K / 2 + K / 4 + .. shuffles, then one per step): lane l ends with
// value l * K / 32.
template <int K, int THREADS>
__device__ __forceinline__ void block_sums(float (&v)[K], float* dweight, int n, float (*part)[K]) {
  const int lane = threadIdx.x & 31;
  int d = 16;
#pragma unroll
  for (int h = K / 2; h >= 1; h >>= 1, d >>= 1) {
    const bool up = lane & d;
#pragma unroll
    for (int i = 0; i < h; i++) {
      const float keep = up ? v[i + h] : v[i], send = up ? v[i] : v[i + h];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, d);
    }
  }
  for (; d >= 1; d >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], d);
  if (lane % (32 / K) == 0) part[threadIdx.x >> 5][lane / (32 / K)] = v[0];
  __syncthreads();
  if ((int)threadIdx.x < K && (int)threadIdx.x < n) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < THREADS / 32; i++) t += part[i][threadIdx.x];
    dweight[threadIdx.x] = t;
  }
  __syncthreads();
}

// Rows (-1: dropped) and weights of the slots j0 .. j0+KU-1 of a token.  All loads are issued before the
// first is looked at; a dropped slot's weight is read with the others and not used.
template <int KU>
__device__ __forceinline__ void load_slots(const RowsMove& m, long long s0, int j0, int (&row)[KU], float (&w)[KU]) {
#pragma unroll
  for (int j = 0; j < KU; j++) row[j] = j0 + j < m.choices ? m.rowOf[s0 + j0 + j] : -1;
#pragma unroll
  for (int j = 0; j < KU; j++) w[j] = m.weight && j0 + j < m.choices ? m.weight[s0 + j0 + j] : 1.f;
#pragma unroll
  for (int j = 0; j < KU; j++)
    if ((unsigned)row[j] >= (unsigned)m.capacity) row[j] = -1;
}

template <int KU>
__device__ __forceinline__ bool near_rows(const RowsMove& m, const int (&row)[KU], long long stride) {
  bool near = false;
#pragma unroll
  for (int j = 0; j < KU; j++) near = near || (row[j] >= 0 && near_end(row[j], m.capacity, stride));
  return near;
}

// Warps that an SM is to hold at least, which limits a thread's registers.  A thread that keeps the
// pieces of many rows needs registers, the others do better with more warps.  Measured, us: rows out
// with the weights' gradient (16384 tokens, half of 8 slots dropped, 4 KB) 24 warps 110, 32 warps 124;
// 16384 tokens to 8 rows of 2001 bf16 with 32, 48, 64 warps 119, 126, 132; sums of 8 rows of 4 KB, half
// dropped, 24, 28, 32 warps 60, 57, 59; sums of 4 rows of 5 KB 32, 40, 48 warps 36.2, 35.2, 35.5; sums of 10
// rows of 4 KB with the weights' gradient 16, 20, 24 warps 171, 110, 139.  Sums of up to 4 rows with it, 32 and
// 40 warps: 3 rows of 1111 fp32 (1023 tokens) 8.4, 10.4; of 1112 fp32 6.0, 6.1; of 1024 bf16 4.6, 4.8; 4 rows of 4096
// bf16 (1024 tokens) 11.4, 11.8; of 2048 bf16 (16384 tokens) 64.9, 66.6; of 2048 fp32 (8192 tokens) 63.5, 64.0.
constexpr int scatter_warps(bool dot) { return dot ? 24 : 32; }
constexpr int gather_warps(int ku, bool dot) { return ku > 8 ? 20 : ku > 4 ? 28 : dot ? 32 : 40; }

// ANY: rows at any address; the pieces of a row are then cut at the 16-byte boundaries of the row
// that is written, so its first and last pieces may be partial.  The token's words are cut at its
// own boundaries; a piece lies in the lane's word and that of the lane below or above, so the first
// and the last lane have no pieces.
//
// grid.x: blocks of padding (experts * kPadBlocks of them, or none), then one for each token; grid.y:
// parts of a row.
template <typename T, bool ANY, int KU, int THREADS, bool WEIGHT, bool DOT>
__global__ void __launch_bounds__(THREADS, scatter_warps(DOT) * 32 / THREADS)
scatter_kernel(const __grid_constant__ RowsMove m, int padBlocks) {
  __shared__ float part[THREADS / 32][KU];
  begin_row_kernel();
  const int bytes = m.width * (int)sizeof(T);
  const int vecs = bytes / 16 + (ANY ? 2 : 0);
  const int share = (vecs + gridDim.y - 1) / gridDim.y;
  const int v0 = blockIdx.y * share, v1 = min(vecs, v0 + share);
  if ((int)blockIdx.x < padBlocks) {
    const int e = blockIdx.x / kPadBlocks;
    const int from = m.offset[e] + m.count[e], to = min(m.offset[e + 1], m.capacity);
    Piece<T> zero;
    zero.raw = make_uint4(0, 0, 0, 0);
    for (int r = max(0, from) + blockIdx.x % kPadBlocks; r < to; r += kPadBlocks) {
      unsigned char* y = const_cast<unsigned char*>(m.row) + (long long)r * m.rowStride;
      const int mis = ANY ? (int)((uintptr_t)y & 15) : 0;
      for (int v = v0 + threadIdx.x; v < v1; v += THREADS) {
        if (ANY) store_any(zero, y, v * 16 - mis, bytes);
        else store_16(y + v * 16, zero.raw);
      }
    }
    return;
  }
  constexpr int STEP = ANY ? THREADS / 32 * 30 : THREADS;
  const int lane = threadIdx.x;
  const int first = ANY ? lane / 32 * 30 + lane % 32 - 1 : lane;
  const bool lender = ANY && (lane % 32 == 0 || lane % 32 == 31);
  const int t = blockIdx.x - padBlocks;
  const unsigned char* x = m.token + (long long)t * m.tokenStride;
  const int misX = ANY ? (int)((uintptr_t)x & 15) : 0;
  const bool nearX = ANY && near_end(t, m.tokens, m.tokenStride);
  const long long s0 = (long long)t * m.choices;
  // the first piece is on its way while the slots are looked up
  bool ahead = true;
  uint4 early = make_uint4(0, 0, 0, 0);
  if (ANY) early = load_word<T>(x, (v0 + first) * 16 - misX, bytes, nearX);
  else if (v0 + first < v1) early = load_16(x + (v0 + first) * 16);
  for (int j0 = 0; j0 < m.choices; j0 += KU) {
    int row[KU];
    float w[KU], dot[KU];
    load_slots<KU>(m, s0, j0, row, w);
    const bool nearOther = ANY && DOT && near_rows<KU>(m, row, m.otherStride);
#pragma unroll
    for (int j = 0; j < KU; j++) dot[j] = 0.f;
    for (int v = v0 + first; ANY ? __any_sync(0xffffffffu, !lender && v < v1) : v < v1; v += STEP) {
      Piece<T> a, o[DOT ? KU : 1];
      uint4 below, here, above;
      if (ahead) here = early;
      else here = ANY ? load_word<T>(x, v * 16 - misX, bytes, nearX) : load_16(x + v * 16);
      ahead = false;
      if (!ANY) a.raw = here;
      if (DOT) {
#pragma unroll
        for (int j = 0; j < KU; j++) {
          if (row[j] < 0) continue;
          const unsigned char* z = m.other + (long long)row[j] * m.otherStride;
          if (ANY) {
            const int lo = v * 16 - past_boundary(m.row, row[j], m.rowStride);
            o[DOT ? j : 0].raw = load_word<T>(z, lo, bytes, nearOther);
          } else {
            o[DOT ? j : 0].raw = load_16(z + v * 16);
          }
        }
      }
      if (ANY) {
        below = word_of(here, -1);
        above = word_of(here, 1);
      }
#pragma unroll
      for (int j = 0; j < KU; j++) {
        if (row[j] < 0) continue;                                  // the same for all lanes
        unsigned char* y = const_cast<unsigned char*>(m.row) + (long long)row[j] * m.rowStride;
        const int misY = ANY ? past_boundary(m.row, row[j], m.rowStride) : 0;
        const int lo = v * 16 - misY;
        if (ANY) {
          if (DOT) o[DOT ? j : 0].raw = join_words(o[DOT ? j : 0].raw, m.other + (long long)row[j] * m.otherStride, lo);
          a.raw = misX >= misY ? shift_bytes(here, above, misX - misY) : shift_bytes(below, here, 16 + misX - misY);
          if (lender || v >= v1 || lo >= bytes) continue;
          if (DOT) {
            clear_outside(a, lo, bytes);
            clear_outside(o[DOT ? j : 0], lo, bytes);
          }
        }
        Piece<T> b;
        if (WEIGHT) {
#pragma unroll
          for (int i = 0; i < b.N; i++) b.e[i] = from_f<T>(to_f(a.e[i]) * w[j]);
        } else {
          b.raw = a.raw;
        }
        if (ANY) store_any(b, y, lo, bytes);
        else store_16(y + lo, b.raw);
        if (DOT) {
#pragma unroll
          for (int i = 0; i < b.N; i++) dot[j] = fmaf(to_f(a.e[i]), to_f(o[DOT ? j : 0].e[i]), dot[j]);
        }
      }
    }
    if (DOT) block_sums<KU, THREADS>(dot, m.dweight + s0 + j0, m.choices - j0, part);
  }
}

template <typename T, bool ANY, int KU, int THREADS, bool DOT>
__global__ void __launch_bounds__(THREADS, gather_warps(KU, DOT) * 32 / THREADS)
gather_kernel(const __grid_constant__ RowsMove m) {
  __shared__ float part[THREADS / 32][KU];
  begin_row_kernel();
  constexpr int N = Piece<T>::N;
  constexpr int H = KU < 8 ? KU : 8;       // rows whose pieces are loaded at once
  // pieces that the block takes at once: with ANY the last lane of every warp only lends its bytes
  constexpr int STEP = ANY ? THREADS / 32 * 31 : THREADS;
  const int bytes = m.width * (int)sizeof(T);
  const int vecs = bytes / 16 + (ANY ? 2 : 0);
  const int share = (vecs + gridDim.y - 1) / gridDim.y;
  const int v0 = blockIdx.y * share, v1 = min(vecs, v0 + share);
  const int lane = threadIdx.x;
  const int first = ANY ? lane - lane / 32 : lane;
  const bool lender = ANY && lane % 32 == 31;
  const int t = blockIdx.x;
  unsigned char* out = const_cast<unsigned char*>(m.token) + (long long)t * m.tokenStride;
  const unsigned char* x = m.other + (long long)t * m.otherStride;
  const int mis = ANY ? (int)((uintptr_t)out & 15) : 0;
  const bool nearX = ANY && DOT && near_end(t, m.tokens, m.otherStride);
  const long long s0 = (long long)t * m.choices;
  // Up to KU choices: one walk over the row does everything.  More: the weights' gradient takes a
  // walk for each group of KU slots, then one walk sums over all groups in registers.
  const bool one = m.choices <= KU;
  // KU of 16: the rows of the eight that are at work only, read again for every piece (they stay in L1), so
  // that registers are left for enough warps.
  constexpr bool AGAIN = KU > H;
  int row[H];
  float w[H];
  bool near = false;
  if (one || DOT) {
    for (int j0 = 0; j0 < m.choices; j0 += KU) {
      float dot[KU];
      if (!AGAIN) {
        load_slots<H>(m, s0, j0, row, w);
        if (ANY) near = near_rows<H>(m, row, m.rowStride);
      }
#pragma unroll
      for (int j = 0; j < KU; j++) dot[j] = 0.f;
      for (int v = v0 + first; ANY ? __any_sync(0xffffffffu, v < v1) : v < v1; v += STEP) {
        const int lo = v * 16 - mis;
        const bool idle = v >= v1 || (ANY && (lender || lo >= bytes));      // (without ANY: never)
        Piece<T> b[H], a;
        float sum[N];
#pragma unroll
        for (int i = 0; i < N; i++) sum[i] = 0.f;
        if (DOT) a.raw = ANY ? load_word<T>(x, lo, bytes, nearX) : load_16(x + lo);
#pragma unroll
        for (int h = 0; h < KU; h += H) {
          if (AGAIN) {
            load_slots<H>(m, s0, j0 + h, row, w);
            if (ANY) near = near_rows<H>(m, row, m.rowStride);
          }
#pragma unroll
          for (int j = 0; j < H; j++) {
            if (row[j] < 0) continue;
            const unsigned char* y = m.row + (long long)row[j] * m.rowStride;
            b[j].raw = ANY ? load_word<T>(y, lo, bytes, near) : load_16(y + lo);
          }
          if (ANY) {
#pragma unroll
            for (int j = 0; j < H; j++)
              if (row[j] >= 0) b[j].raw = join_words(b[j].raw, m.row + (long long)row[j] * m.rowStride, lo);
            if (DOT && h == 0) {
              a.raw = join_words(a.raw, x, lo);
              clear_outside(a, lo, bytes);
            }
            if (idle) continue;
          }
#pragma unroll
          for (int j = 0; j < H; j++) {
            if (row[j] < 0) continue;
            if (ANY && DOT) clear_outside(b[j], lo, bytes);
#pragma unroll
            for (int i = 0; i < N; i++) {
              const float f = to_f(b[j].e[i]);
              sum[i] = fmaf(w[j], f, sum[i]);
              if (DOT) dot[h + j] = fmaf(f, to_f(a.e[i]), dot[h + j]);
            }
          }
        }
        if (one && !idle) {
          Piece<T> r;
#pragma unroll
          for (int i = 0; i < N; i++) r.e[i] = from_f<T>(sum[i]);
          if (ANY) store_any(r, out, lo, bytes);
          else store_16(out + lo, r.raw);
        }
      }
      if (DOT) block_sums<KU, THREADS>(dot, m.dweight + s0 + j0, m.choices - j0, part);
    }
  }
  if (one) return;
  for (int v = v0 + first; ANY ? __any_sync(0xffffffffu, v < v1) : v < v1; v += STEP) {
    const int lo = v * 16 - mis;
    float sum[N];
#pragma unroll
    for (int i = 0; i < N; i++) sum[i] = 0.f;
    for (int j0 = 0; j0 < m.choices; j0 += H) {
      Piece<T> b[H];
      load_slots<H>(m, s0, j0, row, w);
      if (ANY) near = near_rows<H>(m, row, m.rowStride);
#pragma unroll
      for (int j = 0; j < H; j++) {
        if (row[j] < 0) continue;
        const unsigned char* y = m.row + (long long)row[j] * m.rowStride;
        b[j].raw = ANY ? load_word<T>(y, lo, bytes, near) : load_16(y + lo);
      }
#pragma unroll
      for (int j = 0; j < H; j++) {
        if (row[j] < 0) continue;
        if (ANY) b[j].raw = join_words(b[j].raw, m.row + (long long)row[j] * m.rowStride, lo);
#pragma unroll
        for (int i = 0; i < N; i++) sum[i] = fmaf(w[j], to_f(b[j].e[i]), sum[i]);
      }
    }
    if (ANY && (lender || v >= v1 || lo >= bytes)) continue;
    Piece<T> r;
#pragma unroll
    for (int i = 0; i < N; i++) r.e[i] = from_f<T>(sum[i]);
    if (ANY) store_any(r, out, lo, bytes);
    else store_16(out + lo, r.raw);
  }
}

// Threads of a token's block.  Measured with 16384 tokens in bf16, us with 64, 128, 256 and 512 threads:
//   to 8 rows of 8 KB      204, 199, 195, 192      to 2 rows of 8 KB      73, 74, 79, 93
//   to 4 rows of 8 KB      118, 116, 114, 125      to 8 rows of 2 KB      55, 54, 54, 69
// so a thread is to have at least 8 stores.  With weights it needs registers, and 512 threads took 201
// where 256 took 193.
int scatter_threads(long long pieces, bool weight) {
  if (pieces >= 8 * 512 && !weight) return 512;
  return pieces >= 8 * 256 ? 256 : pieces >= 8 * 128 ? 128 : 64;
}
// With the weights' gradient, us with 64, 128 and 256 threads (bf16, 8 slots to a token):
//                                        rows out (combine_grad)     sums (dispatch_grad)
//   16384 tokens, rows of 8 KB             361, 354, 352               214, 209, 226
//     half of the slots dropped            206, 207, 226               147, 145, 173
//   16384 tokens, rows of 4 KB             193, 191, 195               116, 115, 135
//     half of the slots dropped            106, 116, 135               77, 81, 109
//   16384 tokens, rows of 2 KB             98, 100, 133                60, 65, 107
//   1024 tokens, rows of 8 KB              28.3, 30.4, 27.3            21.0, 19.4, 20.1
//   256 tokens, rows of 8 KB               14.8, 11.1, 9.8             13.7, 9.2, 7.4
// Few tokens (less than 8 for an SM): without a sum along the row several blocks of 128 threads share
// one.  With a sum one block has to make it, and more threads are better unless blocks are many and
// rows too short for them (1023 tokens, 3 rows of 1111 fp32, sums with 128 threads 8.4, with 256 10.8).
constexpr int kFewTokens = 8;            // for an SM
constexpr int kMostParts = 8;

int sum_threads(const RowsMove& m, int vecs, int numSM) {
  const bool few = m.tokens < numSM * kFewTokens;
  return few && (vecs >= 512 || m.tokens < 2 * numSM) ? 256 : vecs > 256 ? 128 : 64;
}

dim3 token_grid(const RowsMove& m, int vecs, int threads, bool few) {
  dim3 g(m.tokens, 1, 1);
  if (few && !m.dweight) {
    const int parts = (vecs + threads - 1) / threads;
    g.y = parts < kMostParts ? parts : kMostParts;
  }
  return g;
}

template <typename T, bool ANY, int KU, int THREADS>
cudaError_t run_scatter_dot(const RowsMove& m, dim3 grid, int pad, cudaStream_t stream) {
  if (m.weight) return launch_row_kernel(scatter_kernel<T, ANY, KU, THREADS, true, true>, grid, THREADS, 0, 0, stream, m, pad);
  return launch_row_kernel(scatter_kernel<T, ANY, KU, THREADS, false, true>, grid, THREADS, 0, 0, stream, m, pad);
}

template <typename T, bool ANY, int KU, int THREADS>
cudaError_t run_scatter(const RowsMove& m, dim3 grid, int pad, cudaStream_t stream) {
  if constexpr (sizeof(T) > 1 && THREADS <= 256) {
    if (m.weight) return launch_row_kernel(scatter_kernel<T, ANY, KU, THREADS, true, false>, grid, THREADS, 0, 0, stream, m, pad);
  }
  return launch_row_kernel(scatter_kernel<T, ANY, KU, THREADS, false, false>, grid, THREADS, 0, 0, stream, m, pad);
}

template <typename T, bool ANY, int KU>
cudaError_t scatter(const RowsMove& m, int pad, int numSM, cudaStream_t stream) {
  const int vecs = m.width * (int)sizeof(T) / 16 + (ANY ? 2 : 0);
  const bool few = m.tokens < numSM * kFewTokens;
  // (rows at any address: four at a time, see move_rows)
  if constexpr (sizeof(T) > 1 && !(ANY && KU > 4)) {
    if (m.dweight) {
      const int threads = sum_threads(m, vecs, numSM);
      dim3 g = token_grid(m, vecs, threads, few);
      g.x += pad;
      if (threads == 256) return run_scatter_dot<T, ANY, KU, 256>(m, g, pad, stream);
      if (threads == 128) return run_scatter_dot<T, ANY, KU, 128>(m, g, pad, stream);
      return run_scatter_dot<T, ANY, KU, 64>(m, g, pad, stream);
    }
  }
  const int threads = few ? 128 : scatter_threads((long long)m.choices * vecs, m.weight != nullptr);
  dim3 g = token_grid(m, vecs, threads, few);
  g.x += pad;
  if (threads == 512) return run_scatter<T, ANY, KU, 512>(m, g, pad, stream);
  if (threads == 256) return run_scatter<T, ANY, KU, 256>(m, g, pad, stream);
  if (threads == 128) return run_scatter<T, ANY, KU, 128>(m, g, pad, stream);
  return run_scatter<T, ANY, KU, 64>(m, g, pad, stream);
}

template <typename T, bool ANY, int KU>
cudaError_t gather(const RowsMove& m, int numSM, cudaStream_t stream) {
  const int vecs = m.width * (int)sizeof(T) / 16 + (ANY ? 2 : 0);
  const bool few = m.tokens < numSM * kFewTokens;
  if (m.dweight) {
    const int threads = few ? sum_threads(m, vecs, numSM) : vecs >= 512 ? 128 : 64;
    const dim3 g = token_grid(m, vecs, threads, few);
    if (threads == 256) return launch_row_kernel(gather_kernel<T, ANY, KU, 256, true>, g, 256, 0, 0, stream, m);
    if (threads == 128) return launch_row_kernel(gather_kernel<T, ANY, KU, 128, true>, g, 128, 0, 0, stream, m);
    return launch_row_kernel(gather_kernel<T, ANY, KU, 64, true>, g, 64, 0, 0, stream, m);
  }
  if constexpr (KU <= 8) {
    const int threads = few || vecs >= 512 ? 128 : 64;
    const dim3 g = token_grid(m, vecs, threads, few);
    if (threads == 128) return launch_row_kernel(gather_kernel<T, ANY, KU, 128, false>, g, 128, 0, 0, stream, m);
    return launch_row_kernel(gather_kernel<T, ANY, KU, 64, false>, g, 64, 0, 0, stream, m);
  }
  return cudaErrorInvalidValue;          // sixteen at a time only with the weights' gradient: move_rows
}

template <typename T, bool ANY>
cudaError_t move_rows(const RowsMove& m, bool rowsOut, int pad, int numSM, cudaStream_t stream) {
  if (rowsOut) {
    // Four or eight of a token's rows at a time.  At any address and with the weights' gradient eight leave
    // too few registers for enough warps: 16384 tokens, 8 rows of 2001 bf16, 471 us, with four 361.
    if (m.choices <= 4 || (ANY && m.dweight)) return scatter<T, ANY, 4>(m, pad, numSM, stream);
    return scatter<T, ANY, 8>(m, pad, numSM, stream);
  }
  if constexpr (sizeof(T) > 1) {
    if (m.choices <= 4) return gather<T, ANY, 4>(m, numSM, stream);
    // Up to 16 rows in one walk with the weights' gradient: sums of 10 rows of 4 KB for 8192 tokens took 135 us
    // in a walk for the gradient and one for the sums, 110 in one.
    if (m.choices > 8 && m.dweight) return gather<T, ANY, 16>(m, numSM, stream);
    return gather<T, ANY, 8>(m, numSM, stream);
  }
  return cudaErrorInvalidValue;          // bytes are not summed: check_rows_move
}

template <typename T>
cudaError_t move_typed(const RowsMove& m, bool rowsOut, int pad, int numSM, cudaStream_t stream) {
  if (m.tokens == 0 && pad == 0) return cudaSuccess;
  unsigned long long bits = (uintptr_t)m.token | (uintptr_t)m.row | (uintptr_t)m.other | (unsigned long long)m.tokenStride |
                            (unsigned long long)m.rowStride | (unsigned long long)(m.width * (long long)sizeof(T));
  if (m.other) bits |= (unsigned long long)m.otherStride;
  return bits % 16 ? move_rows<T, true>(m, rowsOut, pad, numSM, stream) : move_rows<T, false>(m, rowsOut, pad, numSM, stream);
}

cudaError_t move(const RowsMove& m, bool rowsOut, int pad, int numSM, cudaStream_t stream) {
  switch (m.type) {
    case 0: return move_typed<uint8_t>(m, rowsOut, pad, numSM, stream);
    case 1: return move_typed<__half>(m, rowsOut, pad, numSM, stream);
    case 2: return move_typed<__nv_bfloat16>(m, rowsOut, pad, numSM, stream);
    case 3: return move_typed<float>(m, rowsOut, pad, numSM, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_rows_scatter(const RowsMove& m, int align, int numSM, cudaStream_t stream) {
  return move(m, true, align > 1 ? m.experts * kPadBlocks : 0, numSM, stream);
}

cudaError_t launch_rows_gather(const RowsMove& m, int numSM, cudaStream_t stream) {
  return m.tokens ? move(m, false, 0, numSM, stream) : cudaSuccess;
}

}  // namespace cuttb
