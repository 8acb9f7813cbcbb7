// The product of a few tokens with a matrix of 4-bit weights with a scale
// (and a zero point) per group:
//   y[m, n] = sum_g s[n, g] sum_{k in g} x[m, k] (q[n, k] - z[n, g]).
#include "blocks.cuh"

namespace pm {
namespace blk {
namespace {

struct W4Args {
  int tokens, n, k, group, groups, scales32;
  int64_t x_stride, weight_stride;
  const void* x;
  const uint8_t* weight;
  const void* scales;
  const uint8_t* zeros;
  void* y;
};

// One warp per row of weights and token.
template <class T>
__global__ void __launch_bounds__(256) w4_warp_kernel(W4Args a) {
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int n = int(unit % a.n), m = int(unit / a.n);
  if (m >= a.tokens) return;
  const T* x = static_cast<const T*>(a.x) + m * a.x_stride;
  const uint8_t* w = a.weight + n * a.weight_stride;
  float sum = 0.0f;
  for (int g = 0; g < a.groups; ++g) {
    const int64_t at = int64_t(n) * a.groups + g;
    const float s = a.scales32 ? static_cast<const float*>(a.scales)[at] : to_float(static_cast<const T*>(a.scales)[at]);
    const float z = a.zeros ? float(a.zeros[at]) : 8.0f;
    const int end = min(a.k, (g + 1) * a.group);
    float part = 0.0f;
    for (int k = g * a.group + lane; k < end; k += 32) {
      const int q = (w[k >> 1] >> (4 * (k & 1))) & 15;
      part += to_float(x[k]) * (float(q) - z);
    }
    sum += s * part;
  }
  sum = warp_sum(sum);
  if (lane == 0) static_cast<T*>(a.y)[int64_t(m) * a.n + n] = from_float<T>(sum);
}

template <class T>
cudaError_t launch(const W4Args& a, cudaStream_t s) {
  const int64_t units = int64_t(a.n) * a.tokens;
  w4_warp_kernel<T><<<unsigned((units + 7) / 8), 256, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace
}  // namespace blk
}  // namespace pm

using namespace pm;
using namespace pm::blk;

extern "C" int pm_matvec_w4_device(const pm_matvec_w4* j, void* stream) {
  const char* who = "pm_matvec_w4_device";
  if (!j) return fail(PM_E_INVALID, "%s: NULL job", who);
  if (j->tokens < 0 || j->n < 1 || j->k < 1) return fail(PM_E_INVALID, "%s: tokens must be >= 0, n and k >= 1", who);
  if (j->tokens > (1 << 16) || j->n > (1 << 24) || j->k > (1 << 24))
    return fail(PM_E_LIMIT, "%s: at most 2^16 tokens, n and k at most 2^24", who);
  if (j->group < 32 || j->group % 32) return fail(PM_E_INVALID, "%s: group must be a multiple of 32", who);
  if (j->dtype != PM_DT_BF16 && j->dtype != PM_DT_F16) return fail(PM_E_INVALID, "%s: x and y are 16-bit floats", who);
  if (j->scales_dtype != j->dtype && j->scales_dtype != PM_DT_F32)
    return fail(PM_E_INVALID, "%s: scales are of the activations' type or 32-bit floats", who);
  if (!j->tokens) return PM_OK;
  if (j->x_stride < j->k || j->weight_stride < (int64_t(j->k) + 1) / 2)
    return fail(PM_E_INVALID, "%s: strides must be at least a row", who);
  if (!j->x || !j->weight || !j->scales || !j->y) return fail(PM_E_INVALID, "%s: NULL buffer", who);
  if (!aligned(j->x, 2) || !aligned(j->y, 2) || !aligned(j->scales, type_bytes(j->scales_dtype)))
    return fail(PM_E_INVALID, "%s: a buffer is not aligned to its elements", who);
  int sms = 0;
  const int rc = sm_count(&sms);
  if (rc != PM_OK) return rc;
  W4Args a{j->tokens, j->n, j->k, j->group, int((int64_t(j->k) + j->group - 1) / j->group), j->scales_dtype == PM_DT_F32,
           j->x_stride, j->weight_stride, j->x, j->weight, j->scales, j->zeros, j->y};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = j->dtype == PM_DT_BF16 ? launch<bf16>(a, s) : launch<fp16>(a, s);
  return e == cudaSuccess ? PM_OK : cuda_fail(e, "pm_matvec_w4_device launch");
}
