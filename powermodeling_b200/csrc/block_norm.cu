// The norms around a block, fused with its gate and residual scale:
//   p = b rsqrt(mean b^2 + eps) w_post,  h = r + scale gate p,
//   y = h rsqrt(mean h^2 + eps) w_pre,
// and the gradients of r, b, both weights and the gate.
//
// Both directions are bound by the rows' bytes (forward: two arrays read, two
// written; backward: four read, two written), so each row is read once and
// kept on chip between its reductions.
//  * Persistent CTAs take runs of consecutive rows, each thread the same
//    columns of every row: the parameters stay in registers, and the next rows
//    arrive meanwhile in a ring of thread-private 16-byte asynchronous copies
//    (each thread reads what it copied: no barrier but the reductions').  512
//    threads an SM hold rows of up to 1024 pieces; wider ones are shared by a
//    cluster, and rows of up to 64 pieces go by warps.
//  * Backward: h is recomputed from r, b and the two saved statistics, which
//    costs no bytes (b is needed anyway) and no rounding.  With gp = scale
//    gate w_post and bu = b r1 the sums over rows that the parameters need are
//    only P = sum dy u and, per gate row, A = sum dh bu: dw_pre = P, dgate =
//    scale w_post A, dw_post = sum scale gate A; they too stay in registers,
//    and a second kernel adds the CTAs' in order.
//  * Rows that 16-byte pieces do not fit (odd widths, strides, addresses): the
//    same with single elements, neighbours in neighbouring lanes, the next
//    row's loaded ahead into registers.  What is wider than that, and the
//    gradients of rows by warps with more gate rows than CTAs, reads its rows
//    again in each pass (the loop kernels).
//  * Sums and statistics are 32-bit, h enters the second norm unrounded; only
//    the outputs are rounded to their type.
// Measured, bf16 with both weights, inputs out of the L2 (a copy runs at 6.55
// TB/s): forward 8192 rows x 8192 93.8 us = 5.7 TB/s, x 4096 51.8 us = 5.2
// TB/s; backward 157.9 us = 5.1 and 81.8 us = 4.9 TB/s.  One row of 4096: 3.0
// us, and 8.6 us for the backward's two launches.  Beside HBM the issue slots
// are short (half and two thirds of them busy at 8192 wide): the conversions
// and the reductions' barriers, not the copies, keep it from the copy's rate.
#include <cooperative_groups.h>

#include <algorithm>

#include "blocks.cuh"

namespace cg = cooperative_groups;

namespace pm {
namespace blk {
namespace {

// A parameter row of type T or float.
template <class T>
struct Param {
  const void* p;
  int f32;
  __device__ __forceinline__ float at(int64_t i) const {
    return f32 ? static_cast<const float*>(p)[i] : to_float(static_cast<const T*>(p)[i]);
  }
};

template <class T>
struct NormArgs {
  int64_t rows, gate_rows, rows_per_gate, residual_stride, block_stride;
  int width;
  float scale, eps;
  const T* residual;
  const T* block;
  Param<T> pre, post, gate;              // post.p NULL: no post norm
  T* hidden;
  T* normed;
  float* stats;
};

template <class T>
struct GradArgs {
  NormArgs<T> f;
  int64_t grad_hidden_stride, grad_normed_stride;
  const T* grad_hidden;
  const T* grad_normed;
  T* grad_residual;
  T* grad_block;
  // Partial sums, [parts, width] each: P; A of each piece of a gate segment
  // (pieces), or, with more segments than CTAs, sum scale gate A (post) with
  // the gate's gradient written where a segment ends (gate_out, gate_tmp).
  float* part_pre;
  float* part_a;
  float* part_post;
  float* gate_tmp;
  void* gate_out;
  int gate_out32;
  int64_t segments;                      // gate rows, or 1
  int chunks;                            // pieces that each segment's rows are cut into
  int slice;                             // 16-byte pieces of a row that one CTA of the cluster takes
};

constexpr int kSingles = 8;              // single elements of a thread, where pieces do not fit

// N neighbouring elements: 16 bytes of them, or one.
template <class T, int N> struct Raw {
  uint4 q;
  __device__ __forceinline__ void unpack(float (&v)[N]) const {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, bf16>::value) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  }
};
template <class T> struct Raw<T, 1> {
  T q;
  __device__ __forceinline__ void unpack(float (&v)[1]) const { v[0] = to_float(q); }
};
template <class T> constexpr int kWide = 16 / sizeof(T);
template <class T, int N>
__device__ __forceinline__ Raw<T, N> load_raw(const T* p) {
  if constexpr (N == 1) return {__ldcs(p)};
  else return {__ldcs(reinterpret_cast<const uint4*>(p))};
}
template <class T, int N>
__device__ __forceinline__ void store(T* p, const float (&v)[N]) {
  if constexpr (N == 1) {
    __stcs(p, from_float<T>(v[0]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        w[i] = __float_as_uint(v[i]);
      } else if constexpr (std::is_same<T, bf16>::value) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
  }
}
template <int N>
__device__ __forceinline__ void store32(float* p, const float (&v)[N]) {
  if constexpr (N == 1) p[0] = v[0];
  else
#pragma unroll
    for (int i = 0; i < N / 4; ++i) reinterpret_cast<float4*>(p)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
}
template <class T, int N>
__device__ __forceinline__ void param_piece(const Param<T>& w, int64_t at, float (&v)[N]) {
  if constexpr (N == 1) {
    v[0] = w.at(at);
  } else if (w.f32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(w.p) + at);
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const float4 q = __ldg(p + i);
      v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w;
    }
  } else {
    Raw<T, N>{__ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(w.p) + at))}.unpack(v);
  }
}
// scale gate w_post of N columns; parts that are not there count as one.
template <class T, int N>
__device__ __forceinline__ void factor_piece(const NormArgs<T>& f, int64_t segment, int col, float (&v)[N]) {
  float g[N];
  if (f.post.p) param_piece<T, N>(f.post, col, v);
  if (f.gate_rows) param_piece<T, N>(f.gate, segment * f.width + col, g);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = (f.post.p ? v[i] : 1.0f) * (f.gate_rows ? g[i] * f.scale : f.scale);
}

// ---------------------------------------------------------------- forward, a row at a time
// Rows that 16-byte pieces do not fit, wider than a thread's registers hold
// beside the next row's: a CTA each, kSingles elements of a thread.  Bound by
// the latency of a row's loads and its two sums with two rows to an SM (4000
// rows of 5001 bf16: 1.8 TB/s, 2500 of 8191 1.5); the parameters come from the L1 each time.
template <class T>
__global__ void __launch_bounds__(1024) norm_row_kernel(const __grid_constant__ NormArgs<T> a) {
  __shared__ float red[2][32];
  constexpr int C = kSingles;
  const int64_t row = blockIdx.x;
  const T* r = a.residual + row * a.residual_stride;
  const T* b = a.block + row * a.block_stride;
  const int64_t segment = a.gate_rows ? row / a.rows_per_gate : 0;
  float h[C], x[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int p = threadIdx.x + c * blockDim.x;
    x[c] = p < a.width ? to_float(__ldcs(b + p)) : 0.0f;
    h[c] = p < a.width ? to_float(__ldcs(r + p)) : 0.0f;
  }
  float r1 = 1.0f;
  if (a.post.p) {
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) s += x[c] * x[c];
    r1 = rsqrtf(cta_sum(s, red[0]) / float(a.width) + a.eps);
  }
  float s = 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int p = threadIdx.x + c * blockDim.x;
    if (p < a.width) {
      float w[1];
      factor_piece<T, 1>(a, segment, p, w);
      h[c] += w[0] * (x[c] * r1);
      s += h[c] * h[c];
      __stcs(a.hidden + row * a.width + p, from_float<T>(h[c]));
    }
  }
  const float r2 = rsqrtf(cta_sum(s, red[1]) / float(a.width) + a.eps);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int p = threadIdx.x + c * blockDim.x;
    if (p < a.width) __stcs(a.normed + row * a.width + p, from_float<T>(h[c] * (r2 * a.pre.at(p))));
  }
  if (a.stats && threadIdx.x == 0) {
    a.stats[2 * row] = r1;
    a.stats[2 * row + 1] = r2;
  }
}

// Sum over the threads of a row: a warp, a CTA or a cluster's CTAs, the same
// on each of them.  One barrier a call; buffers alternate, so a slow thread
// still reads the last sum's while a fast one writes this one's.
template <bool Warps, bool Cluster>
struct RowSum {
  float (*red)[32];
  float (*shared_sum)[8];
  int ranks, rank, parity;
  __device__ __forceinline__ float operator()(float v) {
    v = warp_sum(v);
    if constexpr (Warps) return v;
    if ((threadIdx.x & 31) == 0) red[parity][threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.0f;
    const int warps = (blockDim.x + 127) >> 7;           // in fours; those that are not there are zero
    for (int w = 0; w < warps; ++w) {
      const float4 q = reinterpret_cast<const float4*>(red[parity])[w];
      s += (q.x + q.y) + (q.z + q.w);
    }
    if constexpr (Cluster) {
      if (threadIdx.x < ranks) cg::this_cluster().map_shared_rank(&shared_sum[parity][0], threadIdx.x)[rank] = s;
      cg::this_cluster().sync();
      s = 0.0f;
      for (int k = 0; k < ranks; ++k) s += shared_sum[parity][k];
    }
    parity ^= 1;
    return s;
  }
};
// The buffers' first use; in a cluster also the point from which the others' shared memory may be written.
template <bool Warps, bool Cluster>
__device__ __forceinline__ RowSum<Warps, Cluster> row_sum(float (&red)[2][32], float (&shared_sum)[2][8]) {
  RowSum<Warps, Cluster> r{red, shared_sum, 1, 0, 0};
  if constexpr (!Warps) {
    if (threadIdx.x < 32) red[0][threadIdx.x] = red[1][threadIdx.x] = 0.0f;
    if constexpr (Cluster) {
      r.ranks = int(cg::this_cluster().num_blocks());
      r.rank = int(cg::this_cluster().block_rank());
      cg::this_cluster().sync();
    } else {
      __syncthreads();
    }
  }
  return r;
}

// ---------------------------------------------------------------- forward, rows of single elements
// Rows that 16-byte pieces do not fit, up to 512 * kSingles wide: a CTA per run
// of consecutive rows, the parameters in registers, the next row's elements
// loaded ahead.  Bound by the LSU's instructions, four an element.
template <class T>
__global__ void __launch_bounds__(512) norm_singles_kernel(const __grid_constant__ NormArgs<T> a) {
  constexpr int C = kSingles;
  __shared__ __align__(16) float red[2][32];
  __shared__ float shared_sum[2][8];
  auto total = row_sum<false, false>(red, shared_sum);
  const float inv = 1.0f / float(a.width);
  const int64_t from = a.rows * blockIdx.x / gridDim.x, to = a.rows * (blockIdx.x + 1) / gridDim.x;
  float pre[C], gp[C][1];
  T next_x[C], next_h[C];                                // beyond the row zeros, which add nothing
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int p = threadIdx.x + c * blockDim.x;
    pre[c] = p < a.width ? a.pre.at(p) : 0.0f;
    gp[c][0] = 0.0f;
    next_x[c] = next_h[c] = from_float<T>(0.0f);
  }
  auto fetch = [&](int64_t row) {
    const T* b = a.block + row * a.block_stride + threadIdx.x;
    const T* r = a.residual + row * a.residual_stride + threadIdx.x;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (int(threadIdx.x + c * blockDim.x) < a.width) {
        next_x[c] = __ldcs(b + c * blockDim.x);
        next_h[c] = __ldcs(r + c * blockDim.x);
      }
  };
  if (from < to) fetch(from);
  int64_t segment = -1, segment_end = from;
  for (int64_t row = from; row < to; ++row) {
    if (row == segment_end) {
      segment = a.gate_rows ? row / a.rows_per_gate : 0;
      segment_end = a.gate_rows ? (segment + 1) * a.rows_per_gate : to;
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (int(threadIdx.x + c * blockDim.x) < a.width) factor_piece<T, 1>(a, segment, threadIdx.x + c * blockDim.x, gp[c]);
    }
    float x[C], h[C];
#pragma unroll
    for (int c = 0; c < C; ++c) x[c] = to_float(next_x[c]), h[c] = to_float(next_h[c]);
    if (row + 1 < to) fetch(row + 1);
    float r1 = 1.0f;
    if (a.post.p) {
      float s = 0.0f;
#pragma unroll
      for (int c = 0; c < C; ++c) s += x[c] * x[c];
      r1 = rsqrtf(total(s) * inv + a.eps);
    }
    float s = 0.0f;
    T* hidden = a.hidden + row * a.width + threadIdx.x;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      h[c] += gp[c][0] * (x[c] * r1);
      s += h[c] * h[c];
      if (int(threadIdx.x + c * blockDim.x) < a.width) __stcs(hidden + c * blockDim.x, from_float<T>(h[c]));
    }
    const float r2 = rsqrtf(total(s) * inv + a.eps);
    T* normed = a.normed + row * a.width + threadIdx.x;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (int(threadIdx.x + c * blockDim.x) < a.width) __stcs(normed + c * blockDim.x, from_float<T>(h[c] * (r2 * pre[c])));
    if (a.stats && threadIdx.x == 0) {
      a.stats[2 * row] = r1;
      a.stats[2 * row + 1] = r2;
    }
  }
}

// ---------------------------------------------------------------- forward, rows streamed
// C 16-byte pieces of each array per thread.  Warps: rows by warps, a CTA's
// warps in turn; else a CTA, or a cluster's CTAs, per run of consecutive rows.
// EachRow: the gate changes with every row, and streams with them when it is
// of type T.
constexpr int kNormStages = 4;
template <class T, int C, bool Warps, bool EachRow, bool Cluster, int kTwo = 0>
__global__ void __launch_bounds__(Warps ? 256 : kTwo ? 384 : C == 1 ? 1024 : 512, Warps ? (C == 1 ? 4 : 2) : kTwo ? 2 : 1) norm_stream_kernel(const __grid_constant__ NormArgs<T> a, int slice_pieces) {
  constexpr int N = kWide<T>, kArrays = EachRow ? 3 : 2;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ __align__(16) float red[2][32];
  __shared__ float shared_sum[2][8];
  auto total = row_sum<Warps, Cluster>(red, shared_sum);
  const int pieces = a.width / N, threads = Warps ? 32 : blockDim.x, me = Warps ? threadIdx.x & 31 : threadIdx.x;
  const int part = blockIdx.x / total.ranks, parts = gridDim.x / total.ranks, warp = threadIdx.x >> 5;
  const int piece0 = total.rank * slice_pieces, slice = min(slice_pieces, pieces - piece0);
  const int row_step = Warps ? blockDim.x >> 5 : 1;
  const int64_t from = a.rows * part / parts + (Warps ? warp : 0), to = a.rows * (part + 1) / parts;
  const float inv = 1.0f / float(a.width);
  int col[C];
  bool own[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int p = me + c * threads;
    own[c] = p < slice;
    col[c] = (piece0 + (own[c] ? p : 0)) * N;
  }
  const int row_bytes = kArrays * C * threads * 16;      // a thread's copies: [stage][array][c], threads side by side
  uint8_t* ring = smem + (Warps ? warp * kNormStages * row_bytes : 0) + me * 16;
  const uint32_t ring_addr = smem_addr(ring);
  const bool gate_streams = EachRow && !a.gate.f32;
  auto slot = [&](int stage, int array, int c) { return stage * row_bytes + (array * C + c) * threads * 16; };
  // a piece beyond the row stays zero and adds nothing: only copies, parameters and stores ask whose it is
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (!own[c])
      for (int i = 0; i < kNormStages * kArrays; ++i) *reinterpret_cast<uint4*>(ring + slot(0, i, c)) = make_uint4(0, 0, 0, 0);
  int left = to > from ? int((to - from + row_step - 1) / row_step) : 0, to_fetch = left, place = 0;
  const T* next_r = a.residual + from * a.residual_stride;
  const T* next_b = a.block + from * a.block_stride;
  const T* next_g = static_cast<const T*>(a.gate.p) + from * a.width;
  auto fetch = [&]() {
    if (to_fetch > 0) {
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (own[c]) {
          copy16(ring_addr + slot(place, 0, c), next_r + col[c], 16);
          copy16(ring_addr + slot(place, 1, c), next_b + col[c], 16);
          if (gate_streams) copy16(ring_addr + slot(place, 2, c), next_g + col[c], 16);
        }
      next_r += row_step * a.residual_stride;
      next_b += row_step * a.block_stride;
      if (EachRow) next_g += int64_t(row_step) * a.width;
      --to_fetch;
    }
    place = place + 1 == kNormStages ? 0 : place + 1;
    commit();
  };
  auto piece = [&](int stage, int array, int c, float (&v)[N]) {
    Raw<T, N>{*reinterpret_cast<const uint4*>(ring + slot(stage, array, c))}.unpack(v);
  };
#pragma unroll
  for (int i = 0; i < kNormStages - 1; ++i) fetch();
  float pre[C][N] = {}, gp[C][N] = {};                   // gp: scale gate w_post (EachRow: w_post)
  int64_t row = from, segment = EachRow || !a.gate_rows ? 0 : from / a.rows_per_gate;
  int64_t segment_end = EachRow || !a.gate_rows ? to : (segment + 1) * a.rows_per_gate;
  auto load_factor = [&]() {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (own[c]) {
        if constexpr (EachRow) {
          if (a.post.p) param_piece<T, N>(a.post, col[c], gp[c]);
          else
#pragma unroll
            for (int i = 0; i < N; ++i) gp[c][i] = 1.0f;
        } else {
          factor_piece<T, N>(a, segment, col[c], gp[c]);
        }
      }
  };
  if (left) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (own[c]) param_piece<T, N>(a.pre, col[c], pre[c]);
    load_factor();
  }
  T* hidden = a.hidden + from * a.width;
  T* normed = a.normed + from * a.width;
  int stage = 0;
  for (; left > 0; --left) {
    if constexpr (!EachRow) {
      if (row >= segment_end) {
        segment = row / a.rows_per_gate;
        segment_end = (segment + 1) * a.rows_per_gate;
        load_factor();
      }
    }
    fetch();                                             // to the place of the row before, which this thread is done with
    wait_groups<kNormStages - 1>();
    float r1 = 1.0f, h[C][N], s[4] = {};
    if (a.post.p) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float x[N];
        piece(stage, 1, c, x);
#pragma unroll
        for (int i = 0; i < N; ++i) s[i & 3] += x[i] * x[i];
      }
      r1 = rsqrtf(total((s[0] + s[1]) + (s[2] + s[3])) * inv + a.eps);
      s[0] = s[1] = s[2] = s[3] = 0.0f;
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float x[N], g[N];
      piece(stage, 0, c, h[c]);
      piece(stage, 1, c, x);
      if constexpr (EachRow) {
        if (gate_streams) piece(stage, 2, c, g);
        else param_piece<T, N>(a.gate, row * a.width + col[c], g);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        h[c][i] += (EachRow ? g[i] * a.scale * gp[c][i] : gp[c][i]) * (x[i] * r1);
        s[i & 3] += h[c][i] * h[c][i];
      }
      if (own[c]) store<T, N>(hidden + col[c], h[c]);
    }
    const float r2 = rsqrtf(total((s[0] + s[1]) + (s[2] + s[3])) * inv + a.eps);
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < N; ++i) h[c][i] *= r2 * pre[c][i];
      if (own[c]) store<T, N>(normed + col[c], h[c]);
    }
    if (a.stats && me == 0 && total.rank == 0) *reinterpret_cast<float2*>(a.stats + 2 * row) = make_float2(r1, r2);
    hidden += int64_t(row_step) * a.width;
    normed += int64_t(row_step) * a.width;
    row += row_step;
    stage = stage + 1 == kNormStages ? 0 : stage + 1;
  }
  if constexpr (Cluster) cg::this_cluster().sync();      // no CTA leaves while another may still write its sums here
}

// ---------------------------------------------------------------- backward, rows streamed
// The rows of a CTA: pieces [from, to) of the segments, consecutive rows.
struct Run {
  int64_t from, to, segment_rows;
  int chunks;
  __device__ __forceinline__ int64_t row_of(int64_t item) const {
    return item / chunks * segment_rows + segment_rows * (item % chunks) / chunks;
  }
};
__device__ __forceinline__ Run run_of(int64_t rows, int64_t segments, int chunks, int part, int parts) {
  const int64_t items = segments * chunks;
  return {items * part / parts, items * (part + 1) / parts, rows / segments, chunks};
}

// Whether w_pre lives in shared memory: where a warp with two pieces runs out of registers.
constexpr __host__ __device__ bool pre_shared(int n, int c, bool warps) { return n == 8 && warps && c == 2; }
// Rows in a ring: 512 threads of an SM then hold 192 (EachRow: 160) KB of them.
constexpr __host__ __device__ int stages_of(bool each_row) { return each_row ? 2 : 3; }

// N: elements of a piece, 16 bytes of them in the ring, or one in registers,
// where two rows of four arrays with kSingles of each pass 128 registers (fp32
// spills 164 bytes, in a cluster 328).
// Threads of a row (Warps == false: the CTA, or the cluster's CTAs; true: a
// warp, the CTA's warps then taking rows in turn).  EachRow: a gate per row,
// which streams with the rows; its gradient is complete with the row.
template <class T, int N, int C, bool Warps, bool EachRow, bool Cluster>
__global__ void __launch_bounds__(Warps ? 256 : 512, Warps ? 2 : 1) grad_row_kernel(const __grid_constant__ GradArgs<T> a) {
  constexpr bool kRing = N > 1;
  constexpr int kArrays = EachRow ? 5 : 4, kStages = stages_of(EachRow);
  constexpr bool kPreShared = pre_shared(N, C, Warps);
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ __align__(16) float red[2][32];
  __shared__ float shared_sum[2][8];
  const NormArgs<T>& f = a.f;
  auto total = row_sum<Warps, Cluster>(red, shared_sum);
  const int ranks = total.ranks, rank = total.rank;
  const int part = blockIdx.x / ranks, parts = gridDim.x / ranks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int width_threads = Warps ? 32 : blockDim.x, me = Warps ? lane : threadIdx.x;
  const int row_step = Warps ? blockDim.x >> 5 : 1;
  const int pieces = f.width / N, piece0 = rank * a.slice, slice = min(a.slice, pieces - piece0);
  const Run run = run_of(f.rows, a.segments, a.chunks, part, parts);
  const int64_t row_end = run.row_of(run.to);
  const float inv = 1.0f / float(f.width);
  const bool has_post = f.post.p != nullptr, has_gh = a.grad_hidden != nullptr, has_gy = a.grad_normed != nullptr;

  int col[C];
  bool own[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int p = me + c * width_threads;
    own[c] = p < slice;
    col[c] = (piece0 + (own[c] ? p : 0)) * N;
  }
  // a thread's copies: [stage][array][c], 16 bytes each, threads side by side.  A piece beyond the row, and a gradient
  // that does not come in, stay zero and add nothing: only copies, parameters and stores ask whose a piece is.
  const int row_bytes = kArrays * C * width_threads * 16;
  const int ring_bytes = kStages * kArrays * C * blockDim.x * 16;
  uint8_t* ring = smem + (Warps ? warp * kStages * row_bytes : 0) + me * 16;
  const uint32_t ring_addr = smem_addr(ring);
  Raw<T, N> now[kRing ? 1 : 4][C], next[kRing ? 1 : 4][C];
  auto slot = [&](int stage, int array, int c) { return stage * row_bytes + (array * C + c) * width_threads * 16; };
  if constexpr (kRing) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      for (int i = 0; i < kStages; ++i)
        for (int k = 0; k < kArrays; ++k)
          if (!own[c] || (k == 2 && !has_gh) || (k == 3 && !has_gy)) *reinterpret_cast<uint4*>(ring + slot(i, k, c)) = make_uint4(0, 0, 0, 0);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int c = 0; c < C; ++c) next[k][c].q = from_float<T>(0.0f);
  }
  int64_t item = run.from, row = run.row_of(item) + (Warps ? warp : 0), item_end = run.row_of(item + 1);
  int left = row_end > row ? int((row_end - row + row_step - 1) / row_step) : 0, to_fetch = left, place = 0;
  const T* next_r = f.residual + row * f.residual_stride;
  const T* next_b = f.block + row * f.block_stride;
  const T* next_h = a.grad_hidden + row * a.grad_hidden_stride;
  const T* next_y = a.grad_normed + row * a.grad_normed_stride;
  const T* next_g = static_cast<const T*>(f.gate.p) + row * f.width;
  auto fetch = [&]() {
    if (to_fetch > 0) {
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (own[c]) {
          if constexpr (kRing) {
            copy16(ring_addr + slot(place, 0, c), next_r + col[c], 16);
            copy16(ring_addr + slot(place, 1, c), next_b + col[c], 16);
            if (has_gh) copy16(ring_addr + slot(place, 2, c), next_h + col[c], 16);
            if (has_gy) copy16(ring_addr + slot(place, 3, c), next_y + col[c], 16);
            if constexpr (EachRow) {
              if (!f.gate.f32) copy16(ring_addr + slot(place, 4, c), next_g + col[c], 16);
            }
          } else {
            next[0][c] = load_raw<T, N>(next_r + col[c]);
            next[1][c] = load_raw<T, N>(next_b + col[c]);
            if (has_gh) next[2][c] = load_raw<T, N>(next_h + col[c]);
            if (has_gy) next[3][c] = load_raw<T, N>(next_y + col[c]);
          }
        }
      next_r += row_step * f.residual_stride;
      next_b += row_step * f.block_stride;
      next_h += row_step * a.grad_hidden_stride;
      next_y += row_step * a.grad_normed_stride;
      if (EachRow) next_g += int64_t(row_step) * f.width;
      --to_fetch;
    }
    if constexpr (kRing) {
      place = place + 1 == kStages ? 0 : place + 1;
      commit();
    }
  };
  float pre_held[kPreShared ? 1 : C][N] = {};
  // w_pre of a piece: in registers, or, where those are short, in this thread's own shared memory behind the ring
  auto pre_place = [&](int c) { return reinterpret_cast<float*>(smem + ring_bytes + ((Warps ? warp * C : 0) + c) * width_threads * N * 4) + me * 4; };
  auto pre_of = [&](int c, float (&w)[N]) {
    if constexpr (kPreShared) {
#pragma unroll
      for (int i = 0; i < N / 4; ++i) {
        const float4 q = *reinterpret_cast<const float4*>(pre_place(c) + i * width_threads * 4);
        w[4 * i] = q.x; w[4 * i + 1] = q.y; w[4 * i + 2] = q.z; w[4 * i + 3] = q.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = pre_held[c][i];
    }
  };
  auto piece = [&](int stage, int array, int c, float (&v)[N]) {
    if constexpr (kRing) Raw<T, N>{*reinterpret_cast<const uint4*>(ring + slot(stage, array, c))}.unpack(v);
    else now[array][c].unpack(v);
  };

  // gp = scale gate w_post of the segment (EachRow: w_post)
  float gp[C][N] = {}, sum_p[C][N] = {}, sum_a[C][N] = {};   // EachRow: sum_a is sum scale gate dh bu
  auto load_gp = [&](int64_t segment) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (own[c]) {
        if constexpr (EachRow) {
          if (has_post) param_piece<T, N>(f.post, col[c], gp[c]);
          else
#pragma unroll
            for (int i = 0; i < N; ++i) gp[c][i] = 1.0f;
        } else {
          factor_piece<T, N>(f, segment, col[c], gp[c]);
        }
      }
  };

  // A of a finished piece of a segment, or the gate's gradient itself and the post weight's sum so far
  auto flush = [&](int64_t item) {
    const int64_t segment = item / a.chunks;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (own[c]) {
        if (a.part_a) {
          store32<N>(a.part_a + item * f.width + col[c], sum_a[c]);
        } else {
          float g[N], w[N];
          param_piece<T, N>(f.gate, segment * f.width + col[c], g);
          if (has_post) param_piece<T, N>(f.post, col[c], w);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const int64_t at = segment * f.width + col[c] + i;
            const float v = f.scale * (has_post ? w[i] : 1.0f) * sum_a[c][i];
            if (a.gate_out && a.gate_out32) static_cast<float*>(a.gate_out)[at] = v;
            else if (a.gate_out) static_cast<T*>(a.gate_out)[at] = from_float<T>(v);
            if (a.part_post) {
              float* post = a.part_post + int64_t(part) * f.width + col[c] + i;
              *post = (item == run.from ? 0.0f : *post) + f.scale * g[i] * sum_a[c][i];
            }
          }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) sum_a[c][i] = 0.0f;
      }
  };

#pragma unroll
  for (int i = 0; i < (kRing ? kStages - 1 : 1); ++i) fetch();
#pragma unroll
  for (int c = 0; c < C; ++c)
    if constexpr (kPreShared) {
      float w[N] = {};                                   // zeros for a piece beyond the row
      if (own[c]) param_piece<T, N>(f.pre, col[c], w);
#pragma unroll
      for (int i = 0; i < N / 4; ++i)
        *reinterpret_cast<float4*>(pre_place(c) + i * width_threads * 4) = make_float4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    } else {
      if (own[c]) param_piece<T, N>(f.pre, col[c], pre_held[c]);
    }
  load_gp(EachRow ? 0 : item / a.chunks);
  const float2* st = reinterpret_cast<const float2*>(f.stats) + row;
  float2 st_next = left ? *st : make_float2(0.0f, 0.0f);
  T* grad_residual = a.grad_residual + row * f.width;
  T* grad_block = a.grad_block + row * f.width;
  int stage = 0;
  for (; left > 0; --left) {
    if constexpr (!EachRow && !Warps) {
      if (row >= item_end) {
        flush(item);
        ++item;
        item_end = run.row_of(item + 1);
        load_gp(item / a.chunks);
      }
    }
    const float r1 = st_next.x, r2 = st_next.y;
    st += row_step;
    if (left > 1) st_next = *st;
    if constexpr (kRing) {
      fetch();                                           // to the place of the row before, which this thread is done with
      wait_groups<kStages - 1>();
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int c = 0; c < C; ++c) now[k][c] = next[k][c];
      fetch();
    }
    float u[C][N], gate[EachRow ? C : 1][N], s[4] = {};
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float x[N], gy[N], pre[N];
      piece(stage, 0, c, u[c]);
      piece(stage, 1, c, x);
      piece(stage, 3, c, gy);
      pre_of(c, pre);
      if constexpr (EachRow) {
        if (kRing && !f.gate.f32) {
          if constexpr (kRing) piece(stage, 4, c, gate[c]);
        } else {
          param_piece<T, N>(f.gate, row * f.width + col[c], gate[c]);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) gate[c][i] *= f.scale;
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        u[c][i] = (u[c][i] + (EachRow ? gate[c][i] * gp[c][i] : gp[c][i]) * (x[i] * r1)) * r2;
        s[(N == 1 ? c : i) & 3] += gy[i] * pre[i] * u[c][i];
      }
    }
    const float m2 = has_gy ? total((s[0] + s[1]) + (s[2] + s[3])) * inv * r2 : 0.0f;
    s[0] = s[1] = s[2] = s[3] = 0.0f;
    asm volatile("" ::: "memory");                       // the next part's loads stay there: their registers are needed here
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float x[N], gy[N], dr[N];
      piece(stage, 1, c, x);
      piece(stage, 2, c, dr);
      if (has_gy) {
        float pre[N];
        pre_of(c, pre);
        piece(stage, 3, c, gy);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          dr[i] += pre[i] * (r2 * gy[i]) - u[c][i] * m2;
          sum_p[c][i] += gy[i] * u[c][i];
        }
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float bu = x[i] * r1;
        if constexpr (EachRow) {
          // gate holds scale gate; what the gate's gradient needs is kept in its place
          const float dgb = gate[c][i] * dr[i];
          sum_a[c][i] += dgb * bu;
          u[c][i] = dgb * gp[c][i];
          gate[c][i] = f.scale * dr[i] * gp[c][i] * bu;
        } else {
          sum_a[c][i] += dr[i] * bu;
          u[c][i] = dr[i] * gp[c][i];
        }
        s[(N == 1 ? c : i) & 3] += u[c][i] * bu;
      }
      if (own[c]) {
        store<T, N>(grad_residual + col[c], dr);
        if constexpr (EachRow) {
          if (a.gate_out && a.gate_out32) store32<N>(static_cast<float*>(a.gate_out) + row * f.width + col[c], gate[c]);
          else if (a.gate_out) store<T, N>(static_cast<T*>(a.gate_out) + row * f.width + col[c], gate[c]);
        }
      }
    }
    if (has_post) {
      const float m1 = total((s[0] + s[1]) + (s[2] + s[3])) * inv * r1 * r1;
      asm volatile("" ::: "memory");
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float x[N];
        piece(stage, 1, c, x);
#pragma unroll
        for (int i = 0; i < N; ++i) u[c][i] = r1 * u[c][i] - x[i] * m1;
      }
    }
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (own[c]) store<T, N>(grad_block + col[c], u[c]);
    grad_residual += int64_t(row_step) * f.width;
    grad_block += int64_t(row_step) * f.width;
    row += row_step;
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  if constexpr (kRing) wait_groups<0>();

  if constexpr (Warps) {
    // the warps' sums, in their order, through shared memory
    __syncthreads();
    float* sums = reinterpret_cast<float*>(smem);        // [2][warps][width]
    const int warps = blockDim.x >> 5;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (own[c]) {
        store32<N>(sums + warp * f.width + col[c], sum_p[c]);
        store32<N>(sums + (warps + warp) * f.width + col[c], sum_a[c]);
      }
    __syncthreads();
    float* second = EachRow ? a.part_post : a.part_a;
    const int64_t second_row = EachRow ? part : item;
    for (int x = threadIdx.x; x < f.width; x += blockDim.x) {
      float p = 0.0f, q = 0.0f;
      for (int w = 0; w < warps; ++w) {
        p += sums[w * f.width + x];
        q += sums[(warps + w) * f.width + x];
      }
      if (a.part_pre) a.part_pre[int64_t(part) * f.width + x] = p;
      if (second) second[second_row * f.width + x] = q;
    }
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (own[c]) {
        if (EachRow && a.part_post) store32<N>(a.part_post + int64_t(part) * f.width + col[c], sum_a[c]);
        if (a.part_pre) store32<N>(a.part_pre + int64_t(part) * f.width + col[c], sum_p[c]);
      }
    if constexpr (!EachRow) flush(item);
    if constexpr (Cluster) cg::this_cluster().sync();    // no CTA leaves while another may still write its sums here
  }
}

// ---------------------------------------------------------------- any width
// One CTA per row, the row read again in each pass.
template <class T>
__global__ void __launch_bounds__(256) norm_loop_kernel(NormArgs<T> a) {
  __shared__ float red[2][32];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* r = a.residual + row * a.residual_stride;
    const T* b = a.block + row * a.block_stride;
    const int64_t g = a.gate_rows ? row / a.rows_per_gate * a.width : 0;
    float r1 = 1.0f;
    if (a.post.p) {
      float s = 0.0f;
      for (int c = threadIdx.x; c < a.width; c += blockDim.x) {
        const float v = to_float(b[c]);
        s += v * v;
      }
      r1 = rsqrtf(cta_sum(s, red[0]) / float(a.width) + a.eps);
    }
    auto hidden = [&](int c) {
      float p = to_float(b[c]) * r1;
      if (a.post.p) p *= a.post.at(c);
      const float gate = a.gate_rows ? a.gate.at(g + c) * a.scale : a.scale;
      return to_float(r[c]) + gate * p;
    };
    float s = 0.0f;
    for (int c = threadIdx.x; c < a.width; c += blockDim.x) {
      const float h = hidden(c);
      s += h * h;
    }
    const float r2 = rsqrtf(cta_sum(s, red[1]) / float(a.width) + a.eps);
    for (int c = threadIdx.x; c < a.width; c += blockDim.x) {
      const float h = hidden(c);
      a.hidden[row * a.width + c] = from_float<T>(h);
      a.normed[row * a.width + c] = from_float<T>(h * r2 * a.pre.at(c));
    }
    if (a.stats && threadIdx.x == 0) {
      a.stats[2 * row] = r1;
      a.stats[2 * row + 1] = r2;
    }
    __syncthreads();
  }
}

// The gradients of any width: a CTA per run of consecutive rows, the sums over
// rows in its rows of scratch, each column with one thread.
template <class T>
__global__ void __launch_bounds__(256) grad_loop_kernel(const __grid_constant__ GradArgs<T> a) {
  __shared__ float red[2][32];
  const NormArgs<T>& f = a.f;
  const int width = f.width;
  float* pre = a.part_pre ? a.part_pre + int64_t(blockIdx.x) * width : nullptr;
  float* post = a.part_post ? a.part_post + int64_t(blockIdx.x) * width : nullptr;
  for (int c = threadIdx.x; c < width; c += blockDim.x) {
    if (pre) pre[c] = 0.0f;
    if (post) post[c] = 0.0f;
  }
  const Run run = run_of(f.rows, a.segments, a.chunks, blockIdx.x, gridDim.x);
  const float inv = 1.0f / float(width);
  for (int64_t item = run.from; item < run.to; ++item) {
    const int64_t seg = item / a.chunks, g = seg * width;
    float* sum_a = a.part_a ? a.part_a + item * width : a.gate_tmp + int64_t(blockIdx.x) * width;
    for (int c = threadIdx.x; c < width; c += blockDim.x) sum_a[c] = 0.0f;
    const int64_t last = run.row_of(item + 1);
    auto gate_at = [&](int c) { return f.gate_rows ? f.gate.at(g + c) * f.scale : f.scale; };
    auto post_at = [&](int c) { return f.post.p ? f.post.at(c) : 1.0f; };
    for (int64_t row = run.row_of(item); row < last; ++row) {
      const T* r = f.residual + row * f.residual_stride;
      const T* b = f.block + row * f.block_stride;
      const T* gh = a.grad_hidden ? a.grad_hidden + row * a.grad_hidden_stride : nullptr;
      const T* gy = a.grad_normed ? a.grad_normed + row * a.grad_normed_stride : nullptr;
      const float r1 = f.stats[2 * row], r2 = f.stats[2 * row + 1];
      auto unit_p = [&](int c) { return to_float(b[c]) * r1; };
      auto unit_h = [&](int c) { return (to_float(r[c]) + gate_at(c) * post_at(c) * unit_p(c)) * r2; };
      float s = 0.0f;
      if (gy)
        for (int c = threadIdx.x; c < width; c += blockDim.x) s += to_float(gy[c]) * f.pre.at(c) * unit_h(c);
      const float m2 = cta_sum(s, red[0]) * inv;
      auto grad_h = [&](int c, float u) {
        float d = gh ? to_float(gh[c]) : 0.0f;
        if (gy) d += r2 * (to_float(gy[c]) * f.pre.at(c) - u * m2);
        return d;
      };
      float s1 = 0.0f;
      for (int c = threadIdx.x; c < width; c += blockDim.x) {
        const float u = unit_h(c), d = grad_h(c, u), bu = unit_p(c);
        a.grad_residual[row * width + c] = from_float<T>(d);
        if (pre && gy) pre[c] += to_float(gy[c]) * u;
        sum_a[c] += d * bu;
        s1 += d * gate_at(c) * post_at(c) * bu;
      }
      const float m1 = f.post.p ? cta_sum(s1, red[1]) * inv : 0.0f;
      for (int c = threadIdx.x; c < width; c += blockDim.x) {
        const float d = grad_h(c, unit_h(c));
        const float v = gate_at(c) * d * post_at(c);
        a.grad_block[row * width + c] = from_float<T>(f.post.p ? r1 * (v - unit_p(c) * m1) : v);
      }
      __syncthreads();
    }
    if (!a.part_a)
      for (int c = threadIdx.x; c < width; c += blockDim.x) {
        const float v = f.scale * post_at(c) * sum_a[c];
        if (a.gate_out && a.gate_out32) static_cast<float*>(a.gate_out)[g + c] = v;
        else if (a.gate_out) static_cast<T*>(a.gate_out)[g + c] = from_float<T>(v);
        if (post) post[c] += gate_at(c) * sum_a[c];
      }
  }
}

// Adds the partial sums in order: 32 columns of one output row per CTA, 16
// threads a column, or 16 columns and 32 threads where CTAs would be fewer than
// SMs (forward and backward, 512 rows x 1024: 16.9 us with 32 columns, 16.0
// with 16; 16384 x 8192: 464 and 468).  Output rows: grad_pre, grad_post, then the gate's; with
// one segment the gate's and grad_post come from the same sum.
constexpr int kJoinThreads = 512;
template <class T>
struct JoinArgs {
  const float* part_pre;
  const float* part_a;
  const float* part_post;
  void* grad_pre;
  void* grad_post;
  void* grad_gate;                       // from part_a only
  Param<T> post, gate;
  int64_t gate_rows;
  int parts, chunks, width, pre32, post32, gate32, items;
  int64_t jobs;                          // output rows
  float scale;
};

template <class T, int Columns>
__global__ void __launch_bounds__(kJoinThreads) grad_join_kernel(const __grid_constant__ JoinArgs<T> a) {
  constexpr int kLanes = kJoinThreads / Columns;
  __shared__ float sums[kLanes][Columns + 1];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int x = threadIdx.x % Columns, y = threadIdx.x / Columns, c = blockIdx.x * Columns + x;
  const bool single = a.part_a && a.items == a.chunks;   // one segment, with or without a gate
  for (int64_t job = blockIdx.y; job < a.jobs; job += gridDim.y) {
    const float* part = job == 0 ? a.part_pre : job == 1 ? (a.part_post ? a.part_post : a.part_a) : a.part_a;
    if (!part || !(job == 0 ? a.grad_pre : job == 1 ? (single && a.grad_gate ? a.grad_gate : a.grad_post) : a.grad_gate)) continue;
    const bool gated = job == 1 && part == a.part_a && !single;                // dw_post from every segment's A
    const int count = job == 0 ? a.parts : job == 1 ? (part == a.part_a ? a.items : a.parts) : a.chunks;
    const float* from = part + (job >= 2 ? (job - 2) * a.chunks * int64_t(a.width) : 0);
    float sum = 0.0f;
    if (c < a.width) {
#pragma unroll 10
      for (int k = y; k < count; k += kLanes) {
        float v = __ldcg(from + int64_t(k) * a.width + c);
        if (gated) v *= a.gate_rows ? a.gate.at(int64_t(k / a.chunks) * a.width + c) * a.scale : a.scale;
        sum += v;
      }
    }
    sums[y][x] = sum;
    __syncthreads();
    if (y == 0 && c < a.width) {
      float v = 0.0f;
#pragma unroll
      for (int k = 0; k < kLanes; ++k) v += sums[k][x];
      auto put = [&](void* out, int f32, int64_t at, float value) {
        if (f32) static_cast<float*>(out)[at] = value;
        else static_cast<T*>(out)[at] = from_float<T>(value);
      };
      const float to_gate = a.scale * (a.post.p ? a.post.at(c) : 1.0f);
      if (job == 0) {
        put(a.grad_pre, a.pre32, c, v);
      } else if (job >= 2) {
        put(a.grad_gate, a.gate32, (job - 2) * a.width + c, to_gate * v);
      } else {
        if (a.grad_post) put(a.grad_post, a.post32, c, single ? v * (a.gate_rows ? a.gate.at(c) * a.scale : a.scale) : v);
        if (single && a.grad_gate) put(a.grad_gate, a.gate32, c, to_gate * v);
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- how the rows are shared out
constexpr int kMaxParts = 148 * 4;       // CTAs (clusters) of the backward pass at most: sizes the scratch

struct Split {
  int64_t segments;
  int chunks, parts;                     // parts: CTAs or clusters
  bool joined;                           // A is kept per piece of a segment and joined; else the segment's CTA finishes it
};

Split split_rows(int64_t rows, int64_t gate_rows, int want) {
  Split s;
  s.segments = gate_rows > 0 ? gate_rows : 1;
  const int64_t per = rows / s.segments;
  int64_t chunks = s.segments < want ? want / s.segments : 1;
  if (chunks > per) chunks = per;
  s.chunks = int(chunks);
  const int64_t items = s.segments * chunks;
  s.parts = int(items < want ? items : want);
  s.joined = items <= want;
  return s;
}

template <class T>
NormArgs<T> forward_args(const pm_block_norm* j) {
  NormArgs<T> a;
  a.rows = j->rows;
  a.gate_rows = j->gate_rows;
  a.rows_per_gate = j->gate_rows ? j->rows / j->gate_rows : 1;
  a.residual_stride = j->residual_stride;
  a.block_stride = j->block_stride;
  a.width = j->width;
  a.scale = j->scale;
  a.eps = j->eps;
  a.residual = static_cast<const T*>(j->residual);
  a.block = static_cast<const T*>(j->block);
  a.pre = {j->pre_weight, j->pre_dtype == PM_DT_F32};
  a.post = {j->post_weight, j->post_dtype == PM_DT_F32};
  a.gate = {j->gate, j->gate_dtype == PM_DT_F32};
  a.hidden = static_cast<T*>(j->hidden);
  a.normed = static_cast<T*>(j->normed);
  a.stats = j->stats;
  return a;
}

// Whether 16-byte accesses serve every array of the call.
template <class T>
bool wide(const NormArgs<T>& a, bool outputs) {
  bool ok = a.width % kWide<T> == 0 && a.residual_stride % kWide<T> == 0 && a.block_stride % kWide<T> == 0 &&
            aligned(a.residual, 16) && aligned(a.block, 16) && aligned(a.pre.p, 16) && aligned(a.post.p, 16) && aligned(a.gate.p, 16);
  if (outputs) ok = ok && aligned(a.hidden, 16) && aligned(a.normed, 16);
  return ok;
}
int threads_for(int pieces, int per) { return ((pieces + per - 1) / per + 31) / 32 * 32; }
// CTAs of so many threads that an SM holds, of `room` threads at most.
int share_of_sm(int threads, int room) { return room / threads > 8 ? 8 : room / threads; }
// CTAs of the cluster that shares a row, as few as hold it: 16384 bf16 wide, 2 take 199 us for 4096 rows and 4 take 298 us
// (two rows an SM under way do not make up for the wider cluster's barriers).
int ranks_for(int pieces, int most) { return pieces <= most ? 1 : pieces <= 2 * most ? 2 : pieces <= 4 * most ? 4 : 8; }

template <class... Args>
cudaError_t launch_rows(void (*kernel)(Args...), int ctas, int ranks, int threads, size_t bytes, std::atomic<int>* limits, cudaStream_t s, Args... args) {
  if (bytes) ensure_dynamic_smem(kernel, 1024, bytes, limits);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(ctas * ranks));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ranks > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <class T, int C, bool Warps, bool EachRow, bool Cluster, int kTwo = 0>
cudaError_t launch_norm_stream(const NormArgs<T>& a, int ctas, int ranks, int threads, int slice, cudaStream_t s) {
  static std::atomic<int> limits[kMaxDevices];           // of this kernel
  return launch_rows(norm_stream_kernel<T, C, Warps, EachRow, Cluster, kTwo>, ctas, ranks, threads,
                     size_t(kNormStages) * (EachRow ? 3 : 2) * C * threads * 16, limits, s, a, slice);
}
template <class T, bool EachRow>
cudaError_t launch_norm_streams(const NormArgs<T>& a, int pieces, int sms, cudaStream_t s) {
  auto of_rows = [&](int64_t per, int most) { return int((a.rows + per - 1) / per < most ? (a.rows + per - 1) / per : most); };
  // by warps and by CTAs, 65536 rows: 256 bf16 wide 26 and 38 us, 512 wide 50 and 49 (both at HBM's rate)
  if (pieces <= 32) return launch_norm_stream<T, 1, true, EachRow, false>(a, of_rows(8, sms * 4), 1, 256, pieces, s);
  if (pieces <= 64) return launch_norm_stream<T, 2, true, EachRow, false>(a, of_rows(8, sms * 2), 1, 256, pieces, s);
  // one piece a thread (64 registers, 1024 threads an SM); of more than 768, two (512 threads of 128): 4.5 against 3.6
  // of 6.5 TB/s at 1024 pieces, where 32 warps wait for one another in every sum
  if (pieces > 512 && pieces <= 768) return launch_norm_stream<T, 2, false, EachRow, false, 1>(a, of_rows(1, sms * 2), 1, threads_for(pieces, 2), pieces, s);
  const int ranks = ranks_for(pieces, 1024), slice = (pieces + ranks - 1) / ranks, per = slice > 768 ? 2 : 1, threads = threads_for(slice, per);
  if (ranks > 1) {
    const int pairs = threads_for(slice, 2), most = sms * share_of_sm(pairs, 512) / ranks;
    return launch_norm_stream<T, 2, false, EachRow, true>(a, of_rows(1, most > 1 ? most : 1), ranks, pairs, slice, s);
  }
  return per == 2 ? launch_norm_stream<T, 2, false, EachRow, false>(a, of_rows(1, sms), 1, threads, slice, s)
                  : launch_norm_stream<T, 1, false, EachRow, false>(a, of_rows(1, sms * share_of_sm(threads, 1024)), 1, threads, slice, s);
}

template <class T>
cudaError_t launch_forward(const pm_block_norm* j, int sms, cudaStream_t s) {
  const NormArgs<T> a = forward_args<T>(j);
  const bool fits = a.rows <= 0x7fffffff, each_row = a.gate_rows == a.rows && a.rows > 1;
  const int pieces = a.width / kWide<T>;
  if (wide(a, true) && fits && pieces <= 8192 && aligned(a.stats, 8))
    return each_row ? launch_norm_streams<T, true>(a, pieces, sms, s) : launch_norm_streams<T, false>(a, pieces, sms, s);
  // 20000 rows of 1023 bf16: 60 us, with a CTA for each row 89
  if (fits && a.width <= 512 * kSingles) {
    const int threads = threads_for(a.width, kSingles);
    const int64_t most = int64_t(sms) * std::min(512 / threads, 16);
    norm_singles_kernel<T><<<unsigned(a.rows < most ? a.rows : most), threads, 0, s>>>(a);
    return cudaGetLastError();
  }
  // a row in registers of 1024 threads; 20000 rows of 1023 so took 89 us and by the loops 162
  if (fits && a.width <= 1024 * kSingles) {
    norm_row_kernel<T><<<unsigned(a.rows), threads_for(a.width, kSingles), 0, s>>>(a);
    return cudaGetLastError();
  }
  const int64_t most = int64_t(sms) * 8;
  norm_loop_kernel<T><<<int(a.rows < most ? a.rows : most), 256, 0, s>>>(a);
  return cudaGetLastError();
}

template <class T, int N, int C, bool Warps, bool EachRow, bool Cluster>
cudaError_t launch_grad_rows(const GradArgs<T>& a, int parts, int ranks, int threads, cudaStream_t s) {
  size_t bytes = 0;
  if (N > 1) {
    bytes = size_t(stages_of(EachRow)) * (EachRow ? 5 : 4) * C * threads * 16 + (pre_shared(N, C, Warps) ? size_t(C) * threads * N * 4 : 0);
    if constexpr (Warps) bytes = std::max(bytes, size_t(2) * (threads / 32) * a.f.width * 4);
  }
  static std::atomic<int> limits[kMaxDevices];           // of this kernel
  return launch_rows(grad_row_kernel<T, N, C, Warps, EachRow, Cluster>, parts, ranks, threads, bytes, limits, s, a);
}
template <class T, bool EachRow>
cudaError_t launch_grad_streams(const GradArgs<T>& a, bool rows16, bool by_warps, int per, int parts, int ranks, int threads, cudaStream_t s) {
  constexpr int N = kWide<T>;
  if (!rows16)
    return ranks > 1 ? launch_grad_rows<T, 1, kSingles, false, EachRow, true>(a, parts, ranks, threads, s)
                     : launch_grad_rows<T, 1, kSingles, false, EachRow, false>(a, parts, 1, threads, s);
  if (by_warps)
    return per == 1 ? launch_grad_rows<T, N, 1, true, EachRow, false>(a, parts, 1, 256, s)
                    : launch_grad_rows<T, N, 2, true, EachRow, false>(a, parts, 1, 256, s);
  if (ranks > 1) return launch_grad_rows<T, N, 2, false, EachRow, true>(a, parts, ranks, threads, s);
  return launch_grad_rows<T, N, 2, false, EachRow, false>(a, parts, 1, threads, s);
}

template <class T>
cudaError_t launch_backward(const pm_block_norm* j, const pm_block_norm_grads* d, float* scratch, int sms, cudaStream_t s) {
  constexpr int N = kWide<T>;
  GradArgs<T> a{};
  a.f = forward_args<T>(j);
  a.grad_hidden = static_cast<const T*>(d->grad_hidden);
  a.grad_normed = static_cast<const T*>(d->grad_normed);
  a.grad_hidden_stride = d->grad_hidden_stride;
  a.grad_normed_stride = d->grad_normed_stride;
  a.grad_residual = static_cast<T*>(d->grad_residual);
  a.grad_block = static_cast<T*>(d->grad_block);
  const int64_t w = j->width;
  const bool each_row = j->gate_rows == j->rows && j->rows > 1;
  const bool rows16 = wide(a.f, false) && aligned(a.grad_residual, 16) && aligned(a.grad_block, 16) && aligned(d->grad_gate, 16) &&
                      (!a.grad_hidden || (aligned(a.grad_hidden, 16) && a.grad_hidden_stride % N == 0)) &&
                      (!a.grad_normed || (aligned(a.grad_normed, 16) && a.grad_normed_stride % N == 0));
  // pieces of 16 bytes, or single elements; 512 threads of a CTA at most, with two pieces or kSingles elements each (one
  // piece and up to 640 threads took 386 us instead of 348 for forward and backward of 16384 rows x 5120 bf16)
  const int pieces = rows16 ? j->width / N : j->width;
  const int ranks = ranks_for(pieces, rows16 ? 1024 : 512 * kSingles);
  bool streamed = j->rows <= 0x7fffffff && aligned(a.f.stats, 8) && pieces <= 8 * (rows16 ? 1024 : 512 * kSingles);
  a.slice = (pieces + ranks - 1) / ranks;
  // Rows of up to 64 pieces go by warps, 8 of them a CTA, where a CTA stays in one segment or every row has its gate
  // (forward and backward of 65536 rows, by warps and by CTAs: 256 bf16 wide 69 and 184 us, 512 wide 137 and 207).
  const bool by_warps = streamed && rows16 && pieces <= 64;
  int per = rows16 ? 2 : kSingles, row_threads = 256, want = 2 * sms;
  if (by_warps) {
    per = pieces <= 32 ? 1 : 2;
    want = 2 * sms;
  } else if (streamed) {
    row_threads = threads_for(a.slice, per);
    want = sms * share_of_sm(row_threads, 512) / ranks;
  }
  if (want > kMaxParts) want = kMaxParts;
  if (want < 1) want = 1;
  const Split sp = split_rows(j->rows, j->gate_rows, want);
  if (by_warps && !each_row && !sp.joined) streamed = false;
  a.segments = sp.segments;
  a.chunks = sp.chunks;
  const bool wants_gate = d->grad_gate && j->gate_rows;
  const bool wants_post = d->grad_post && j->post_weight;
  if (d->grad_pre) a.part_pre = scratch;
  scratch += sp.parts * w;
  const bool by_a = sp.joined && !(streamed && each_row);
  if (by_a) {
    a.part_a = scratch;
  } else {
    if (wants_post) a.part_post = scratch;
    a.gate_tmp = scratch + sp.parts * w;
    a.gate_out = wants_gate ? d->grad_gate : nullptr;
    a.gate_out32 = j->gate_dtype == PM_DT_F32;
  }
  cudaError_t e;
  if (!streamed) {
    grad_loop_kernel<T><<<sp.parts, 256, 0, s>>>(a);
    e = cudaGetLastError();
  } else {
    e = each_row ? launch_grad_streams<T, true>(a, rows16, by_warps, per, sp.parts, ranks, row_threads, s)
                 : launch_grad_streams<T, false>(a, rows16, by_warps, per, sp.parts, ranks, row_threads, s);
  }
  if (e != cudaSuccess) return e;
  const bool gate_joined = wants_gate && by_a;
  if (!d->grad_pre && !wants_post && !gate_joined) return cudaSuccess;
  const int64_t jobs = by_a && sp.segments == 1 ? 2 : 2 + (gate_joined ? j->gate_rows : 0);
  JoinArgs<T> q{a.part_pre, a.part_a, a.part_post, d->grad_pre, wants_post ? d->grad_post : nullptr,
                gate_joined ? d->grad_gate : nullptr, a.f.post, a.f.gate, j->gate_rows, sp.parts, sp.chunks, j->width,
                j->pre_dtype == PM_DT_F32, j->post_dtype == PM_DT_F32, j->gate_dtype == PM_DT_F32,
                int(by_a ? sp.segments * sp.chunks : 0), jobs, j->scale};
  cudaLaunchConfig_t cfg{};
  const bool few = (w + 31) / 32 * jobs < sms;
  cfg.gridDim = dim3(unsigned(few ? (w + 15) / 16 : (w + 31) / 32), unsigned(jobs < 65535 ? jobs : 65535));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = s;
  cudaLaunchAttribute early[1];
  early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = early;
  cfg.numAttrs = 1;
  return few ? cudaLaunchKernelEx(&cfg, grad_join_kernel<T, 16>, q) : cudaLaunchKernelEx(&cfg, grad_join_kernel<T, 32>, q);
}

int check_forward(const char* who, const pm_block_norm* j, bool backward) {
  if (!j) return fail(PM_E_INVALID, "%s: NULL job", who);
  if (j->rows < 0 || j->width < 1 || j->width > (1 << 20)) return fail(PM_E_INVALID, "%s: rows must be >= 0 and width in 1..2^20", who);
  if (!known_type(j->dtype)) return fail(PM_E_INVALID, "%s: unknown element type %d", who, j->dtype);
  auto param_type = [&](int t) { return t == j->dtype || t == PM_DT_F32; };
  if (!param_type(j->pre_dtype) || (j->post_weight && !param_type(j->post_dtype)) || (j->gate_rows && !param_type(j->gate_dtype)))
    return fail(PM_E_INVALID, "%s: weights and gate are of the activations' type or 32-bit floats", who);
  if (j->gate_rows < 0 || (j->rows && j->gate_rows && j->rows % j->gate_rows))
    return fail(PM_E_INVALID, "%s: gate_rows must divide rows", who);
  if ((j->gate != nullptr) != (j->gate_rows > 0)) return fail(PM_E_INVALID, "%s: gate and gate_rows come together", who);
  if (!(j->eps >= 0.0f) || !(j->scale - j->scale == 0.0f)) return fail(PM_E_INVALID, "%s: eps must be >= 0 and scale finite", who);
  if (j->rows > (int64_t(1) << 40) / j->width) return fail(PM_E_LIMIT, "%s: rows x width must be at most 2^40", who);
  if (!j->rows) return PM_OK;
  if (j->residual_stride < j->width || j->block_stride < j->width) return fail(PM_E_INVALID, "%s: row strides must be at least the width", who);
  if (!j->residual || !j->block || !j->pre_weight || (!backward && (!j->hidden || !j->normed)) || (backward && !j->stats))
    return fail(PM_E_INVALID, "%s: NULL buffer", who);
  const size_t e = type_bytes(j->dtype);
  if (!aligned(j->residual, e) || !aligned(j->block, e) || !aligned(j->pre_weight, type_bytes(j->pre_dtype)) ||
      (j->post_weight && !aligned(j->post_weight, type_bytes(j->post_dtype))) ||
      (j->gate && !aligned(j->gate, type_bytes(j->gate_dtype))) || !aligned(j->stats, 4) ||
      (!backward && (!aligned(j->hidden, e) || !aligned(j->normed, e))))
    return fail(PM_E_INVALID, "%s: a buffer is not aligned to its elements", who);
  return PM_OK;
}

}  // namespace

int sm_count(int* sms) {
  static std::atomic<int> known[kMaxDevices];
  int device = 0;
  int rc = PM_OK;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= kMaxDevices || !known[device].load(std::memory_order_relaxed)) {
    rc = current_device(&device);
    if (rc != PM_OK) return rc;
    int n = 0;
    const cudaError_t e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device);
    if (e != cudaSuccess) return cuda_fail(e, "cudaDeviceGetAttribute");
    known[device].store(n, std::memory_order_relaxed);
  }
  *sms = known[device].load(std::memory_order_relaxed);
  return PM_OK;
}

}  // namespace blk
}  // namespace pm

using namespace pm;
using namespace pm::blk;

extern "C" int pm_block_norm_device(const pm_block_norm* job, void* stream) {
  int rc = check_forward("pm_block_norm_device", job, false);
  if (rc != PM_OK || !job->rows) return rc;
  int sms = 0;
  if ((rc = sm_count(&sms)) != PM_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = job->dtype == PM_DT_F32 ? launch_forward<float>(job, sms, s)
                        : job->dtype == PM_DT_BF16 ? launch_forward<bf16>(job, sms, s) : launch_forward<fp16>(job, sms, s);
  return e == cudaSuccess ? PM_OK : cuda_fail(e, "pm_block_norm_device launch");
}

extern "C" size_t pm_block_norm_backward_scratch_bytes(int64_t rows, int64_t gate_rows, int32_t width) {
  if (rows < 1 || width < 1 || gate_rows < 0 || (gate_rows && rows % gate_rows)) return 0;
  // three rows of partial sums for every CTA, whatever the SM count
  return size_t(3) * size_t(kMaxParts < rows ? kMaxParts : rows) * size_t(width) * 4;
}

extern "C" int pm_block_norm_backward_device(const pm_block_norm* forward, const pm_block_norm_grads* grads, void* scratch,
                                             size_t scratch_bytes, void* stream) {
  const char* who = "pm_block_norm_backward_device";
  int rc = check_forward(who, forward, true);
  if (rc != PM_OK) return rc;
  if (!grads) return fail(PM_E_INVALID, "%s: NULL grads", who);
  if (!forward->rows) {
    // no row contributes: the sums are zero
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    const size_t w = size_t(forward->width);
    if (grads->grad_pre) e = cudaMemsetAsync(grads->grad_pre, 0, w * type_bytes(forward->pre_dtype), s);
    if (e == cudaSuccess && grads->grad_post && forward->post_weight) e = cudaMemsetAsync(grads->grad_post, 0, w * type_bytes(forward->post_dtype), s);
    if (e == cudaSuccess && grads->grad_gate && forward->gate_rows)
      e = cudaMemsetAsync(grads->grad_gate, 0, size_t(forward->gate_rows) * w * type_bytes(forward->gate_dtype), s);
    return e == cudaSuccess ? PM_OK : cuda_fail(e, who);
  }
  if (!grads->grad_residual || !grads->grad_block) return fail(PM_E_INVALID, "%s: NULL buffer", who);
  if ((grads->grad_hidden && grads->grad_hidden_stride < forward->width) || (grads->grad_normed && grads->grad_normed_stride < forward->width))
    return fail(PM_E_INVALID, "%s: row strides must be at least the width", who);
  const size_t e = type_bytes(forward->dtype);
  if (!aligned(grads->grad_hidden, e) || !aligned(grads->grad_normed, e) || !aligned(grads->grad_residual, e) || !aligned(grads->grad_block, e) ||
      !aligned(grads->grad_pre, type_bytes(forward->pre_dtype)) || !aligned(grads->grad_post, type_bytes(forward->post_dtype)) ||
      !aligned(grads->grad_gate, type_bytes(forward->gate_dtype)))
    return fail(PM_E_INVALID, "%s: a buffer is not aligned to its elements", who);
  const size_t need = pm_block_norm_backward_scratch_bytes(forward->rows, forward->gate_rows, forward->width);
  if (!scratch || !aligned(scratch, 256) || scratch_bytes < need)
    return fail(PM_E_INVALID, "%s: needs %zu bytes of scratch, 256-byte aligned", who, need);
  int sms = 0;
  if ((rc = sm_count(&sms)) != PM_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  float* f = static_cast<float*>(scratch);
  const cudaError_t err = forward->dtype == PM_DT_F32 ? launch_backward<float>(forward, grads, f, sms, s)
                          : forward->dtype == PM_DT_BF16 ? launch_backward<bf16>(forward, grads, f, sms, s)
                                                         : launch_backward<fp16>(forward, grads, f, sms, s);
  return err == cudaSuccess ? PM_OK : cuda_fail(err, "pm_block_norm_backward_device launch");
}
