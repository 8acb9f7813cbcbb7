// The norms around a block, fused with its gate and residual scale:
//   p = b rsqrt(mean b^2 + eps) w_post,  h = r + scale gate p,
//   y = h rsqrt(mean h^2 + eps) w_pre,
// and the gradients of r, b, both weights and the gate.
//
// Both directions are bound by the rows' bytes (forward: two arrays read, two
// written; backward: four read, two written), so each row is read once and
// kept on chip between its reductions.
//  * Forward: a warp (rows of up to 64 16-byte pieces) or a CTA per row, two
//    pieces of each array per thread in registers (four for 32-bit rows of
//    more than 2048 pieces).
//  * Backward: h is recomputed from r, b and the two saved statistics, which
//    costs no bytes (b is needed anyway) and no rounding.  With gp = scale
//    gate w_post and bu = b r1 the sums over rows that the parameters need are
//    only P = sum dy u and, per gate row, A = sum dh bu: dw_pre = P, dgate =
//    scale w_post A, dw_post = sum scale gate A.  Persistent CTAs take runs of
//    consecutive rows, each thread the same columns of every row, P and A in
//    registers; the next rows arrive meanwhile in a ring of thread-private
//    asynchronous copies (each thread reads what it copied: no barrier but
//    the reductions').  Rows beyond 1024 pieces are shared by a cluster.
//    A second kernel adds the CTAs' partial sums in order.
//  * Any other width, stride or alignment: the loop kernels, which read a row
//    again in each pass.
#include <cooperative_groups.h>

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

// 16 bytes of T.
template <class T> struct Vec {
  static constexpr int n = 16 / sizeof(T);
  uint4 q;
  __device__ __forceinline__ float at(int i) const { return to_float(reinterpret_cast<const T*>(&q)[i]); }
};
template <class T>
__device__ __forceinline__ uint4 pack(const float (&v)[Vec<T>::n]) {
  uint4 q;
  T* t = reinterpret_cast<T*>(&q);
#pragma unroll
  for (int i = 0; i < Vec<T>::n; ++i) t[i] = from_float<T>(v[i]);
  return q;
}
template <class T>
__device__ __forceinline__ Vec<T> load_stream(const T* p) {
  return {__ldcs(reinterpret_cast<const uint4*>(p))};
}
template <class T>
__device__ __forceinline__ void param_piece(const Param<T>& w, int64_t at, float (&v)[Vec<T>::n]) {
  constexpr int n = Vec<T>::n;
  if (w.f32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(w.p) + at);
#pragma unroll
    for (int i = 0; i < n / 4; ++i) {
      const float4 q = __ldg(p + i);
      v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w;
    }
  } else {
    const Vec<T> q{__ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(w.p) + at))};
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] = q.at(i);
  }
}

// ---------------------------------------------------------------- forward, rows in registers
// C 16-byte pieces per thread; WarpRow: one warp per row, else one CTA.
template <class T, int C, bool WarpRow>
__global__ void __launch_bounds__(1024) norm_row_kernel(const __grid_constant__ NormArgs<T> a) {
  constexpr int n = Vec<T>::n;
  __shared__ float red[2][32];
  const int64_t row = WarpRow ? int64_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= a.rows) return;                             // whole warps of the last CTA, which has no barrier
  const int first = WarpRow ? threadIdx.x & 31 : threadIdx.x, step = WarpRow ? 32 : blockDim.x;
  const int pieces = a.width / n;
  const T* r = a.residual + row * a.residual_stride;
  const T* b = a.block + row * a.block_stride;
  const int64_t g = a.gate_rows ? row / a.rows_per_gate * a.width : 0;
  Vec<T> rv[C], bv[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int p = first + c * step;
    if (p < pieces) {
      bv[c] = load_stream(b + p * n);
      rv[c] = load_stream(r + p * n);
    } else {
      bv[c].q = rv[c].q = make_uint4(0, 0, 0, 0);
    }
  }
  auto total = [&](float v, float* where) { return WarpRow ? warp_sum(v) : cta_sum(v, where); };
  float r1 = 1.0f;
  if (a.post.p) {
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < n; ++i) s += bv[c].at(i) * bv[c].at(i);
    r1 = rsqrtf(total(s, red[0]) / float(a.width) + a.eps);
  }
  float h[C][n], s = 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int p = first + c * step;
    if (p < pieces) {
      float w[n], v[n];
      if (a.post.p) param_piece(a.post, p * n, w);
      if (a.gate_rows) param_piece(a.gate, g + p * n, v);
#pragma unroll
      for (int i = 0; i < n; ++i) {
        float x = bv[c].at(i) * r1;
        if (a.post.p) x *= w[i];
        h[c][i] = rv[c].at(i) + (a.gate_rows ? v[i] * a.scale : a.scale) * x;
        s += h[c][i] * h[c][i];
      }
      __stcs(reinterpret_cast<uint4*>(a.hidden + row * a.width + p * n), pack<T>(h[c]));
    }
  }
  const float r2 = rsqrtf(total(s, red[1]) / float(a.width) + a.eps);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int p = first + c * step;
    if (p < pieces) {
      float w[n];
      param_piece(a.pre, p * n, w);
#pragma unroll
      for (int i = 0; i < n; ++i) h[c][i] *= r2 * w[i];
      __stcs(reinterpret_cast<uint4*>(a.normed + row * a.width + p * n), pack<T>(h[c]));
    }
  }
  if (a.stats && first == 0) {
    a.stats[2 * row] = r1;
    a.stats[2 * row + 1] = r2;
  }
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

// Rows in a ring: 512 threads of an SM then hold 192 (EachRow: 160) KB of them.
constexpr __host__ __device__ int stages_of(bool each_row) { return each_row ? 2 : 3; }

// Threads of a row (Warps == false: the CTA, or the cluster's CTAs; true: a
// warp, the CTA's warps then taking rows in turn).  EachRow: a gate per row,
// which streams with the rows; its gradient is complete with the row.
template <class T, bool Warps, bool EachRow, bool Cluster>
__global__ void __launch_bounds__(512) grad_row_kernel(const __grid_constant__ GradArgs<T> a) {
  constexpr int n = Vec<T>::n, C = 2, kArrays = EachRow ? 5 : 4, kStages = stages_of(EachRow);
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ __align__(16) float red[2][32];
  __shared__ float shared_sum[2][8];
  const NormArgs<T>& f = a.f;
  const int ranks = Cluster ? int(cg::this_cluster().num_blocks()) : 1, rank = Cluster ? int(cg::this_cluster().block_rank()) : 0;
  if constexpr (Cluster) cg::this_cluster().sync();      // the others' shared memory is written only once they run
  const int part = blockIdx.x / ranks, parts = gridDim.x / ranks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int width_threads = Warps ? 32 : blockDim.x, me = Warps ? lane : threadIdx.x;
  const int row_step = Warps ? blockDim.x >> 5 : 1;
  const int pieces = f.width / n, piece0 = rank * a.slice, slice = min(a.slice, pieces - piece0);
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
    col[c] = (piece0 + (own[c] ? p : 0)) * n;
  }
  // a thread's copies: [stage][array][c], 16 bytes each, threads side by side
  const int row_bytes = kArrays * C * width_threads * 16;
  uint8_t* ring = smem + (Warps ? warp * kStages * row_bytes : 0) + me * 16;
  const uint32_t ring_addr = smem_addr(ring);
  auto slot = [&](int stage, int array, int c) { return stage * row_bytes + (array * C + c) * width_threads * 16; };
  auto fetch = [&](int64_t row, int stage) {
    if (row < row_end) {
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (own[c]) {
          copy16(ring_addr + slot(stage, 0, c), f.residual + row * f.residual_stride + col[c], 16);
          copy16(ring_addr + slot(stage, 1, c), f.block + row * f.block_stride + col[c], 16);
          if (has_gh) copy16(ring_addr + slot(stage, 2, c), a.grad_hidden + row * a.grad_hidden_stride + col[c], 16);
          if (has_gy) copy16(ring_addr + slot(stage, 3, c), a.grad_normed + row * a.grad_normed_stride + col[c], 16);
          if constexpr (EachRow) {
            if (!f.gate.f32) copy16(ring_addr + slot(stage, 4, c), static_cast<const T*>(f.gate.p) + row * f.width + col[c], 16);
          }
        }
    }
    commit();
  };
  auto piece = [&](int stage, int array, int c) { return Vec<T>{*reinterpret_cast<const uint4*>(ring + slot(stage, array, c))}; };

  int parity = 0;
  auto total = [&](float v) {
    if constexpr (Warps) return warp_sum(v);
    v = warp_sum(v);
    if (lane == 0) red[parity][warp] = v;
    __syncthreads();
    const int warps = blockDim.x >> 5;
    float s = 0.0f;
    for (int w = 0; w < warps; ++w) s += red[parity][w];
    if constexpr (Cluster) {
      if (threadIdx.x < ranks) cg::this_cluster().map_shared_rank(&shared_sum[parity][0], threadIdx.x)[rank] = s;
      cg::this_cluster().sync();
      s = 0.0f;
      for (int k = 0; k < ranks; ++k) s += shared_sum[parity][k];
    }
    parity ^= 1;
    return s;
  };

  // pre, and gp = scale gate w_post of the segment (EachRow: w_post)
  float pre[C][n], gp[C][n], sum_p[C][n] = {}, sum_a[C][n] = {};   // EachRow: sum_a is sum scale gate dh bu
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (own[c]) param_piece(f.pre, col[c], pre[c]);
  auto load_gp = [&](int64_t segment) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (own[c]) {
        if (has_post) param_piece(f.post, col[c], gp[c]);
        else
#pragma unroll
          for (int i = 0; i < n; ++i) gp[c][i] = 1.0f;
        if constexpr (!EachRow) {
          float g[n];
          if (f.gate_rows) param_piece(f.gate, segment * f.width + col[c], g);
#pragma unroll
          for (int i = 0; i < n; ++i) gp[c][i] *= f.gate_rows ? g[i] * f.scale : f.scale;
        }
      }
  };
  if constexpr (EachRow) load_gp(0);

  // A of a finished piece of a segment (each warp its own where rows go by warps; joined below)
  auto flush = [&](int64_t item) {
    if (a.part_a) {
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (own[c]) {
          float4* at = reinterpret_cast<float4*>(a.part_a + item * f.width + col[c]);
#pragma unroll
          for (int i = 0; i < n / 4; ++i) at[i] = make_float4(sum_a[c][4 * i], sum_a[c][4 * i + 1], sum_a[c][4 * i + 2], sum_a[c][4 * i + 3]);
        }
    } else {
      const int64_t segment = item / a.chunks;
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (own[c]) {
          float g[n], w[n];
          param_piece(f.gate, segment * f.width + col[c], g);
          if (has_post) param_piece(f.post, col[c], w);
          if (a.gate_out) {
#pragma unroll
            for (int i = 0; i < n; ++i) {
              const float v = f.scale * (has_post ? w[i] : 1.0f) * sum_a[c][i];
              const int64_t at = segment * f.width + col[c] + i;
              if (a.gate_out32) static_cast<float*>(a.gate_out)[at] = v;
              else static_cast<T*>(a.gate_out)[at] = from_float<T>(v);
            }
          }
          if (a.part_post) {
            float* at = a.part_post + int64_t(part) * f.width + col[c];
            const bool fresh = item == run.from;
#pragma unroll
            for (int i = 0; i < n; ++i) at[i] = (fresh ? 0.0f : at[i]) + f.scale * g[i] * sum_a[c][i];
          }
        }
    }
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < n; ++i) sum_a[c][i] = 0.0f;
  };

  int64_t item = run.from;
  int64_t row = run.row_of(item) + (Warps ? warp : 0), item_end = run.row_of(item + 1);
  if constexpr (!EachRow) load_gp(item / a.chunks);
  int64_t ahead = row;
  for (int i = 0; i < kStages - 1; ++i, ahead += row_step) fetch(ahead, i);
  float2 st_next = row < row_end ? *reinterpret_cast<const float2*>(f.stats + 2 * row) : make_float2(0.0f, 0.0f);
  int stage = 0;
  for (; row < row_end; row += row_step) {
    if constexpr (!EachRow && !Warps) {
      if (row >= item_end) {
        flush(item);
        ++item;
        item_end = run.row_of(item + 1);
        load_gp(item / a.chunks);
      }
    }
    const float r1 = st_next.x, r2 = st_next.y;
    if (row + row_step < row_end) st_next = *reinterpret_cast<const float2*>(f.stats + 2 * (row + row_step));
    fetch(ahead, stage == 0 ? kStages - 1 : stage - 1);  // the place of the row before, which this thread is done with
    ahead += row_step;
    if constexpr (EachRow) wait_groups<1>();
    else wait_groups<2>();
    float u[C][n], gate[EachRow ? C : 1][n], s = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (own[c]) {
        const Vec<T> rv = piece(stage, 0, c), bv = piece(stage, 1, c);
        Vec<T> gy{};
        if (has_gy) gy = piece(stage, 3, c);
        if constexpr (EachRow) {
          if (f.gate.f32) {
            param_piece(f.gate, row * f.width + col[c], gate[c]);
          } else {
            const Vec<T> gv = piece(stage, 4, c);
#pragma unroll
            for (int i = 0; i < n; ++i) gate[c][i] = gv.at(i);
          }
#pragma unroll
          for (int i = 0; i < n; ++i) gate[c][i] *= f.scale;
        }
#pragma unroll
        for (int i = 0; i < n; ++i) {
          const float w = EachRow ? gate[c][i] * gp[c][i] : gp[c][i];
          u[c][i] = (rv.at(i) + w * (bv.at(i) * r1)) * r2;
          if (has_gy) s += gy.at(i) * pre[c][i] * u[c][i];
        }
      }
    const float m2 = has_gy ? total(s) * inv : 0.0f;
    float s1 = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (own[c]) {
        const Vec<T> bv = piece(stage, 1, c);
        Vec<T> gh{}, gy{};
        if (has_gh) gh = piece(stage, 2, c);
        if (has_gy) gy = piece(stage, 3, c);
        float dr[n];
#pragma unroll
        for (int i = 0; i < n; ++i) {
          float d = has_gh ? gh.at(i) : 0.0f;
          if (has_gy) {
            d += r2 * (gy.at(i) * pre[c][i] - u[c][i] * m2);
            sum_p[c][i] += gy.at(i) * u[c][i];
          }
          dr[i] = d;
          const float bu = bv.at(i) * r1;
          if constexpr (EachRow) {
            // gate holds scale gate; what the gate's gradient needs is kept in its place
            const float dgb = gate[c][i] * d;
            sum_a[c][i] += dgb * bu;
            u[c][i] = dgb * gp[c][i];
            gate[c][i] = f.scale * d * gp[c][i] * bu;
          } else {
            sum_a[c][i] += d * bu;
            u[c][i] = d * gp[c][i];
          }
          s1 += u[c][i] * bu;
        }
        __stcs(reinterpret_cast<uint4*>(a.grad_residual + row * f.width + col[c]), pack<T>(dr));
        if constexpr (EachRow) {
          if (a.gate_out) {
            const int64_t at = row * f.width + col[c];
            if (a.gate_out32) {
              float4* o = reinterpret_cast<float4*>(static_cast<float*>(a.gate_out) + at);
#pragma unroll
              for (int i = 0; i < n / 4; ++i) o[i] = make_float4(gate[c][4 * i], gate[c][4 * i + 1], gate[c][4 * i + 2], gate[c][4 * i + 3]);
            } else {
              __stcs(reinterpret_cast<uint4*>(static_cast<T*>(a.gate_out) + at), pack<T>(gate[c]));
            }
          }
        }
      }
    const float m1 = has_post ? total(s1) * inv : 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (own[c]) {
        const Vec<T> bv = piece(stage, 1, c);
        float db[n];
#pragma unroll
        for (int i = 0; i < n; ++i) db[i] = has_post ? r1 * (u[c][i] - bv.at(i) * r1 * m1) : u[c][i];
        __stcs(reinterpret_cast<uint4*>(a.grad_block + row * f.width + col[c]), pack<T>(db));
      }
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  wait_groups<0>();

  if constexpr (Warps) {
    // the warps' sums, in their order, through shared memory
    __syncthreads();
    float* sums = reinterpret_cast<float*>(smem);        // [2][warps][width]
    const int warps = blockDim.x >> 5;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (own[c])
#pragma unroll
        for (int i = 0; i < n; ++i) {
          sums[warp * f.width + col[c] + i] = sum_p[c][i];
          sums[(warps + warp) * f.width + col[c] + i] = sum_a[c][i];
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
    if constexpr (EachRow) {
      if (a.part_post) {
#pragma unroll
        for (int c = 0; c < C; ++c)
          if (own[c])
#pragma unroll
            for (int i = 0; i < n; ++i) a.part_post[int64_t(part) * f.width + col[c] + i] = sum_a[c][i];
      }
    } else {
      flush(item);
    }
    if (a.part_pre) {
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (own[c])
#pragma unroll
          for (int i = 0; i < n; ++i) a.part_pre[int64_t(part) * f.width + col[c] + i] = sum_p[c][i];
    }
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
// threads a column.  Output rows: grad_pre, grad_post, then the gate's.
constexpr int kLanes = 16;
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
  float scale;
};

template <class T>
__global__ void __launch_bounds__(32 * kLanes) grad_join_kernel(const __grid_constant__ JoinArgs<T> a) {
  __shared__ float sums[kLanes][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, c = blockIdx.x * 32 + x;
  for (int64_t job = blockIdx.y; job < 2 + a.gate_rows; job += gridDim.y) {
    const float* part = job == 0 ? a.part_pre : job == 1 ? (a.part_post ? a.part_post : a.part_a) : a.part_a;
    void* out = job == 0 ? a.grad_pre : job == 1 ? a.grad_post : a.grad_gate;
    if (!out || !part) continue;
    const bool gated = job == 1 && part == a.part_a;     // dw_post from A
    const int count = job == 0 ? a.parts : job == 1 ? (gated ? a.items : a.parts) : a.chunks;
    const float* from = part + (job >= 2 ? (job - 2) * a.chunks * int64_t(a.width) : 0);
    float sum = 0.0f;
    if (c < a.width)
#pragma unroll 4
      for (int k = y; k < count; k += kLanes) {
        float v = __ldcg(from + int64_t(k) * a.width + c);
        if (gated) v *= a.gate_rows ? a.gate.at(int64_t(k / a.chunks) * a.width + c) * a.scale : a.scale;
        sum += v;
      }
    sums[y][x] = sum;
    __syncthreads();
    if (y == 0 && c < a.width) {
      float v = 0.0f;
#pragma unroll
      for (int k = 0; k < kLanes; ++k) v += sums[k][x];
      if (job >= 2) v *= a.scale * (a.post.p ? a.post.at(c) : 1.0f);
      const int64_t at = (job >= 2 ? (job - 2) * a.width : 0) + c;
      if (job == 0 ? a.pre32 : job == 1 ? a.post32 : a.gate32) static_cast<float*>(out)[at] = v;
      else static_cast<T*>(out)[at] = from_float<T>(v);
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
  bool ok = a.width % Vec<T>::n == 0 && a.residual_stride % Vec<T>::n == 0 && a.block_stride % Vec<T>::n == 0 &&
            aligned(a.residual, 16) && aligned(a.block, 16) && aligned(a.pre.p, 16) && aligned(a.post.p, 16) && aligned(a.gate.p, 16);
  if (outputs) ok = ok && aligned(a.hidden, 16) && aligned(a.normed, 16);
  return ok;
}

template <class T>
cudaError_t launch_forward(const pm_block_norm* j, int sms, cudaStream_t s) {
  const NormArgs<T> a = forward_args<T>(j);
  const int pieces = a.width / Vec<T>::n;
  auto threads_for = [&](int per) { return ((pieces + per - 1) / per + 31) / 32 * 32; };
  if (wide(a, true) && a.rows <= 0x7fffffff) {
    if (pieces <= 64) {
      const unsigned grid = unsigned((a.rows + 7) / 8);
      if (pieces <= 32) norm_row_kernel<T, 1, true><<<grid, 256, 0, s>>>(a);
      else norm_row_kernel<T, 2, true><<<grid, 256, 0, s>>>(a);
      return cudaGetLastError();
    }
    if (pieces <= 2048) {
      norm_row_kernel<T, 2, false><<<unsigned(a.rows), threads_for(2), 0, s>>>(a);
      return cudaGetLastError();
    }
    if (pieces <= 4096 && sizeof(T) == 4) {              // 16-bit rows this wide would not fit the registers
      norm_row_kernel<T, sizeof(T) == 4 ? 4 : 2, false><<<unsigned(a.rows), threads_for(4), 0, s>>>(a);
      return cudaGetLastError();
    }
  }
  const int64_t most = int64_t(sms) * 8;
  norm_loop_kernel<T><<<int(a.rows < most ? a.rows : most), 256, 0, s>>>(a);
  return cudaGetLastError();
}

std::atomic<int> g_grad_smem[3][3][2][kMaxDevices];      // by type, threads of a row, gate per row

template <class T, bool Warps, bool EachRow, bool Cluster>
cudaError_t launch_grad_rows(const GradArgs<T>& a, int parts, int ranks, int threads, cudaStream_t s) {
  constexpr int type = sizeof(T) == 4 ? 0 : std::is_same<T, bf16>::value ? 1 : 2;
  const auto kernel = grad_row_kernel<T, Warps, EachRow, Cluster>;
  size_t bytes = size_t(stages_of(EachRow)) * (EachRow ? 5 : 4) * 2 * threads * 16;
  if (Warps) {
    const size_t sums = size_t(2) * (threads / 32) * a.f.width * 4;
    if (sums > bytes) bytes = sums;
  }
  ensure_dynamic_smem(kernel, 1024, bytes, g_grad_smem[type][Warps ? 0 : Cluster ? 1 : 2][EachRow]);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(parts * ranks));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = Cluster ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <class T>
cudaError_t launch_backward(const pm_block_norm* j, const pm_block_norm_grads* d, float* scratch, int sms, cudaStream_t s) {
  GradArgs<T> a{};
  a.f = forward_args<T>(j);
  a.grad_hidden = static_cast<const T*>(d->grad_hidden);
  a.grad_normed = static_cast<const T*>(d->grad_normed);
  a.grad_hidden_stride = d->grad_hidden_stride;
  a.grad_normed_stride = d->grad_normed_stride;
  a.grad_residual = static_cast<T*>(d->grad_residual);
  a.grad_block = static_cast<T*>(d->grad_block);
  const int64_t w = j->width;
  const int pieces = j->width / Vec<T>::n;
  const bool each_row = j->gate_rows == j->rows && j->rows > 1;
  const bool rows16 = wide(a.f, false) && aligned(a.grad_residual, 16) && aligned(a.grad_block, 16) && aligned(d->grad_gate, 16) &&
                      aligned(a.f.stats, 8) && (!a.grad_hidden || (aligned(a.grad_hidden, 16) && a.grad_hidden_stride % Vec<T>::n == 0)) &&
                      (!a.grad_normed || (aligned(a.grad_normed, 16) && a.grad_normed_stride % Vec<T>::n == 0));
  const int ranks = pieces <= 1024 ? 1 : pieces <= 2048 ? 2 : pieces <= 4096 ? 4 : 8;
  bool streamed = rows16 && pieces <= 8192;
  a.slice = (pieces + ranks - 1) / ranks;
  const int row_threads = streamed ? ((a.slice + 1) / 2 + 31) / 32 * 32 : 256;
  // rows of up to 64 pieces go by warps, 8 of them a CTA, where a warp stays in one segment or gates every row
  const bool by_warps = streamed && pieces <= 64;
  // CTAs that fit an SM at 128 registers a thread, and rings of at most 200 KB together
  int per_sm = by_warps ? 2 : ranks > 1 ? 1 : 512 / row_threads;
  if (per_sm > 4) per_sm = 4;
  int want = streamed ? sms * per_sm / ranks : 2 * sms;
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
  } else if (by_warps) {
    e = each_row ? launch_grad_rows<T, true, true, false>(a, sp.parts, 1, 256, s)
                 : launch_grad_rows<T, true, false, false>(a, sp.parts, 1, 256, s);
  } else {
    if (ranks > 1)
      e = each_row ? launch_grad_rows<T, false, true, true>(a, sp.parts, ranks, row_threads, s)
                   : launch_grad_rows<T, false, false, true>(a, sp.parts, ranks, row_threads, s);
    else
      e = each_row ? launch_grad_rows<T, false, true, false>(a, sp.parts, 1, row_threads, s)
                   : launch_grad_rows<T, false, false, false>(a, sp.parts, 1, row_threads, s);
  }
  if (e != cudaSuccess) return e;
  const bool gate_joined = wants_gate && by_a;
  if (!d->grad_pre && !wants_post && !gate_joined) return cudaSuccess;
  JoinArgs<T> q{a.part_pre, a.part_a, a.part_post, d->grad_pre, wants_post ? d->grad_post : nullptr,
                gate_joined ? d->grad_gate : nullptr, a.f.post, a.f.gate, j->gate_rows, sp.parts, sp.chunks, j->width,
                j->pre_dtype == PM_DT_F32, j->post_dtype == PM_DT_F32, j->gate_dtype == PM_DT_F32,
                int(by_a ? sp.segments * sp.chunks : 0), j->scale};
  const int64_t jobs = 2 + (gate_joined ? j->gate_rows : 0);
  if (!gate_joined) q.grad_gate = nullptr;
  grad_join_kernel<T><<<dim3(unsigned((j->width + 31) / 32), unsigned(jobs < 65535 ? jobs : 65535)), 32 * kLanes, 0, s>>>(q);
  return cudaGetLastError();
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
