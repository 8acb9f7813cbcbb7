// The norms around a block, fused with its gate and residual scale:
//   p = b rsqrt(mean b^2 + eps) w_post,  h = r + scale gate p,
//   y = h rsqrt(mean h^2 + eps) w_pre,
// and the gradients of r, b, both weights and the gate.
#include "blocks.cuh"

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
  float* part_pre;                       // [parts, width] partial sums, one row per CTA
  float* part_post;
  float* part_gate;                      // [segments * chunks, width]
  T* grad_gate_direct;                   // chunks == 1: the gate's gradient itself, of type T ...
  float* grad_gate_direct32;             // ... or float
  int64_t segments;                      // gate rows, or 1
  int chunks;                            // pieces that each segment's rows are cut into
};

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

// One CTA per piece of consecutive rows of one gate segment; each thread owns
// the same columns of every row, so the sums over rows stay with one thread.
template <class T>
__global__ void __launch_bounds__(256) grad_loop_kernel(GradArgs<T> a) {
  __shared__ float red[2][32];
  const NormArgs<T>& f = a.f;
  const int width = f.width;
  float* pre = a.part_pre ? a.part_pre + int64_t(blockIdx.x) * width : nullptr;
  float* post = a.part_post ? a.part_post + int64_t(blockIdx.x) * width : nullptr;
  for (int c = threadIdx.x; c < width; c += blockDim.x) {
    if (pre) pre[c] = 0.0f;
    if (post) post[c] = 0.0f;
  }
  const int64_t items = a.segments * a.chunks;
  const int64_t segment_rows = f.rows / a.segments;
  const int64_t from = items * blockIdx.x / gridDim.x, to = items * (blockIdx.x + 1) / gridDim.x;
  const float inv = 1.0f / float(width);
  for (int64_t item = from; item < to; ++item) {
    const int64_t seg = item / a.chunks, chunk = item % a.chunks;
    const int64_t first = seg * segment_rows + segment_rows * chunk / a.chunks;
    const int64_t last = seg * segment_rows + segment_rows * (chunk + 1) / a.chunks;
    const int64_t g = seg * width;
    float* gate_part = a.part_gate ? a.part_gate + item * width : nullptr;
    if (gate_part)
      for (int c = threadIdx.x; c < width; c += blockDim.x) gate_part[c] = 0.0f;
    for (int64_t row = first; row < last; ++row) {
      const T* r = f.residual + row * f.residual_stride;
      const T* b = f.block + row * f.block_stride;
      const T* gh = a.grad_hidden ? a.grad_hidden + row * a.grad_hidden_stride : nullptr;
      const T* gy = a.grad_normed ? a.grad_normed + row * a.grad_normed_stride : nullptr;
      const float r1 = f.stats[2 * row], r2 = f.stats[2 * row + 1];
      auto unit_p = [&](int c) { return to_float(b[c]) * r1; };
      auto gate_at = [&](int c) { return f.gate_rows ? f.gate.at(g + c) * f.scale : f.scale; };
      auto post_at = [&](int c) { return f.post.p ? f.post.at(c) : 1.0f; };
      auto unit_h = [&](int c) { return (to_float(r[c]) + gate_at(c) * (unit_p(c) * post_at(c))) * r2; };
      float s = 0.0f;
      if (gy)
        for (int c = threadIdx.x; c < width; c += blockDim.x) s += to_float(gy[c]) * f.pre.at(c) * unit_h(c);
      const float m2 = cta_sum(s, red[0]) * inv;
      float s1 = 0.0f;
      auto grad_h = [&](int c, float u) {
        float d = gh ? to_float(gh[c]) : 0.0f;
        if (gy) d += r2 * (to_float(gy[c]) * f.pre.at(c) - u * m2);
        return d;
      };
      for (int c = threadIdx.x; c < width; c += blockDim.x) {
        const float u = unit_h(c), d = grad_h(c, u), bu = unit_p(c);
        a.grad_residual[row * width + c] = from_float<T>(d);
        if (pre && gy) pre[c] += to_float(gy[c]) * u;
        const float p = bu * post_at(c);
        if (gate_part) gate_part[c] += f.scale * d * p;
        if (a.grad_gate_direct || a.grad_gate_direct32) {
          // a segment of one row: its gradient is complete
          if (a.grad_gate_direct32) a.grad_gate_direct32[g + c] = f.scale * d * p;
          else a.grad_gate_direct[g + c] = from_float<T>(f.scale * d * p);
        }
        const float dp = gate_at(c) * d;
        if (post) post[c] += dp * bu;
        s1 += dp * post_at(c) * bu;
      }
      if (f.post.p) {
        const float m1 = cta_sum(s1, red[1]) * inv;
        for (int c = threadIdx.x; c < width; c += blockDim.x) {
          const float d = grad_h(c, unit_h(c));
          a.grad_block[row * width + c] = from_float<T>(r1 * (gate_at(c) * d * post_at(c) - unit_p(c) * m1));
        }
      } else {
        for (int c = threadIdx.x; c < width; c += blockDim.x)
          a.grad_block[row * width + c] = from_float<T>(gate_at(c) * grad_h(c, unit_h(c)));
      }
      __syncthreads();
    }
  }
}

// Sums the partial rows in order: out[s, c] = sum_i part[s * count + i, c].
template <class T>
__global__ void __launch_bounds__(256) grad_reduce_kernel(const float* part, int count, int64_t total, int width, T* out) {
  for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += int64_t(gridDim.x) * blockDim.x) {
    const int64_t s = i / width;
    const int c = int(i - s * width);
    const float* p = part + s * count * width + c;
    float sum = 0.0f;
    for (int k = 0; k < count; ++k) sum += p[int64_t(k) * width];
    out[i] = from_float<T>(sum);
  }
}

// ---------------------------------------------------------------- how the rows are shared out
constexpr int kMaxParts = 512;           // CTAs of the backward pass at most

struct Split {
  int64_t segments;
  int chunks, parts;                     // parts: CTAs
  bool gate_partials;                    // the gate's gradient is joined from partial rows
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
  s.gate_partials = gate_rows > 0 && per > 1;
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

template <class T>
cudaError_t launch_forward(const pm_block_norm* j, int sms, cudaStream_t s) {
  const NormArgs<T> a = forward_args<T>(j);
  const int64_t most = int64_t(sms) * 8;
  norm_loop_kernel<T><<<int(a.rows < most ? a.rows : most), 256, 0, s>>>(a);
  return cudaGetLastError();
}

template <class T>
cudaError_t reduce(const float* part, int count, int64_t segments, int width, void* out, bool f32, int sms, cudaStream_t s) {
  const int64_t total = segments * width, want = (total + 255) / 256, most = int64_t(sms) * 8;
  const int grid = int(want < most ? want : most);
  if (f32) grad_reduce_kernel<float><<<grid, 256, 0, s>>>(part, count, total, width, static_cast<float*>(out));
  else grad_reduce_kernel<T><<<grid, 256, 0, s>>>(part, count, total, width, static_cast<T*>(out));
  return cudaGetLastError();
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
  const int want = 2 * sms < kMaxParts ? 2 * sms : kMaxParts;
  const Split sp = split_rows(j->rows, j->gate_rows, want);
  a.segments = sp.segments;
  a.chunks = sp.chunks;
  const int64_t w = j->width;
  if (d->grad_pre) { a.part_pre = scratch; scratch += sp.parts * w; }
  if (d->grad_post && j->post_weight) { a.part_post = scratch; scratch += sp.parts * w; }
  const bool gate32 = j->gate_dtype == PM_DT_F32;
  if (d->grad_gate && j->gate_rows) {
    if (sp.gate_partials) a.part_gate = scratch;
    else if (gate32) a.grad_gate_direct32 = static_cast<float*>(d->grad_gate);
    else a.grad_gate_direct = static_cast<T*>(d->grad_gate);
  }
  grad_loop_kernel<T><<<sp.parts, 256, 0, s>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess && a.part_pre) e = reduce<T>(a.part_pre, sp.parts, 1, j->width, d->grad_pre, j->pre_dtype == PM_DT_F32, sms, s);
  if (e == cudaSuccess && a.part_post) e = reduce<T>(a.part_post, sp.parts, 1, j->width, d->grad_post, j->post_dtype == PM_DT_F32, sms, s);
  if (e == cudaSuccess && a.part_gate) e = reduce<T>(a.part_gate, sp.chunks, sp.segments, j->width, d->grad_gate, gate32, sms, s);
  return e;
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
  // an upper bound over every SM count: parts <= kMaxParts, joined gate pieces <= kMaxParts or one per segment
  const Split s = split_rows(rows, gate_rows, kMaxParts);
  const int64_t pieces = s.gate_partials ? (s.segments > kMaxParts ? s.segments : kMaxParts) : 0;
  return size_t(2 * int64_t(kMaxParts < rows ? kMaxParts : rows) + (pieces < rows ? pieces : rows)) * size_t(width) * 4;
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
