// Attention of one query token per sequence over a paged key-value cache:
//   out = softmax(scale q K^T) V over the live positions.
#include <climits>
#include <cmath>

#include "blocks.cuh"

namespace pm {
namespace blk {
namespace {

// Writes the new token's key and value to its entry of the cache.
template <class T>
__global__ void __launch_bounds__(128) append_kernel(pm_paged_attention j) {
  const int b = blockIdx.x / j.kv_heads, g = blockIdx.x % j.kv_heads;
  const int pos = j.lengths[b] - 1;
  if (pos < 0 || pos / j.page_size >= j.table_columns) return;
  const int page = j.table[b * j.table_stride + pos / j.page_size];
  if (page < 0 || page >= j.n_pages) return;
  const int off = pos % j.page_size;
  T* k = static_cast<T*>(j.k_cache) + page * j.k_page_stride + off * j.k_token_stride + g * j.k_head_stride;
  T* v = static_cast<T*>(j.v_cache) + page * j.v_page_stride + off * j.v_token_stride + g * j.v_head_stride;
  const T* nk = static_cast<const T*>(j.new_k) + b * j.new_k_stride + g * j.new_k_head_stride;
  const T* nv = static_cast<const T*>(j.new_v) + b * j.new_v_stride + g * j.new_v_head_stride;
  for (int c = threadIdx.x; c < j.head_dim; c += blockDim.x) {
    k[c] = nk[c];
    v[c] = nv[c];
  }
}

// One CTA per sequence and query head; each warp takes every fourth position,
// with its own running maximum and sum.
template <class T>
__global__ void __launch_bounds__(128) attention_kernel(pm_paged_attention j) {
  __shared__ float tops[4], sums[4], acc[4][256];
  const int b = blockIdx.x / j.q_heads, h = blockIdx.x % j.q_heads, g = h / (j.q_heads / j.kv_heads);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T* q = static_cast<const T*>(j.q) + b * j.q_stride + h * j.q_head_stride;
  float qf[8], o[8];
  for (int i = 0; i < 8; ++i) {
    qf[i] = lane + 32 * i < j.head_dim ? to_float(q[lane + 32 * i]) : 0.0f;
    o[i] = 0.0f;
  }
  const int64_t room = int64_t(j.table_columns) * j.page_size;
  const int64_t length = j.lengths[b] < 0 ? 0 : j.lengths[b];
  const int64_t from = j.window && length > j.window ? length - j.window : 0;
  const int64_t to = length < room ? length : room;
  float top = -INFINITY, sum = 0.0f;
  for (int64_t pos = from + warp; pos < to; pos += 4) {
    const int page = j.table[b * j.table_stride + pos / j.page_size];
    if (page < 0 || page >= j.n_pages) continue;
    const int off = int(pos % j.page_size);
    const T* k = static_cast<const T*>(j.k_cache) + page * j.k_page_stride + off * j.k_token_stride + g * j.k_head_stride;
    const T* v = static_cast<const T*>(j.v_cache) + page * j.v_page_stride + off * j.v_token_stride + g * j.v_head_stride;
    float s = 0.0f;
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < j.head_dim) s += qf[i] * to_float(k[lane + 32 * i]);
    s = warp_sum(s) * j.scale;
    const float next = fmaxf(top, s), base = next == -INFINITY ? 0.0f : next;
    const float keep = expf(top - base), w = expf(s - base);
    sum = sum * keep + w;
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < j.head_dim) o[i] = o[i] * keep + w * to_float(v[lane + 32 * i]);
    top = next;
  }
  if (lane == 0) { tops[warp] = top; sums[warp] = sum; }
  for (int i = 0; i < 8; ++i) acc[warp][lane + 32 * i] = o[i];
  __syncthreads();
  float best = -INFINITY, total = 0.0f;
  for (int w = 0; w < 4; ++w) best = fmaxf(best, tops[w]);
  const float base = best == -INFINITY ? 0.0f : best;
  for (int w = 0; w < 4; ++w) total += sums[w] * expf(tops[w] - base);
  T* out = static_cast<T*>(j.out) + (int64_t(b) * j.q_heads + h) * j.head_dim;
  for (int c = threadIdx.x; c < j.head_dim; c += 128) {
    float v = 0.0f;
    for (int w = 0; w < 4; ++w) v += acc[w][c] * expf(tops[w] - base);
    out[c] = from_float<T>(total == 0.0f ? 0.0f : v / total);
  }
  if (j.lse && threadIdx.x == 0) j.lse[int64_t(b) * j.q_heads + h] = base + logf(total);
}

template <class T>
cudaError_t launch(const pm_paged_attention& j, cudaStream_t s) {
  if (j.new_k) append_kernel<T><<<j.batch * j.kv_heads, 128, 0, s>>>(j);
  attention_kernel<T><<<j.batch * j.q_heads, 128, 0, s>>>(j);
  return cudaGetLastError();
}

}  // namespace
}  // namespace blk
}  // namespace pm

using namespace pm;
using namespace pm::blk;

extern "C" size_t pm_paged_attention_scratch_bytes(int32_t batch, int32_t q_heads, int32_t kv_heads, int32_t head_dim) {
  if (batch < 1 || q_heads < 1 || kv_heads < 1 || head_dim < 1) return 0;
  return 256;
}

extern "C" int pm_paged_attention_device(const pm_paged_attention* j, void* scratch, size_t scratch_bytes, void* stream) {
  const char* who = "pm_paged_attention_device";
  if (!j) return fail(PM_E_INVALID, "%s: NULL job", who);
  if (j->batch < 0 || j->q_heads < 1 || j->kv_heads < 1 || j->q_heads % j->kv_heads)
    return fail(PM_E_INVALID, "%s: batch must be >= 0 and kv_heads divide q_heads", who);
  if (j->head_dim < 8 || j->head_dim > 256 || j->head_dim % 8)
    return fail(PM_E_INVALID, "%s: head_dim must be a multiple of 8 in 8..256", who);
  if (j->page_size < 1 || j->page_size > 65536 || j->n_pages < 0 || j->table_columns < 0 || j->window < 0)
    return fail(PM_E_INVALID, "%s: page_size must be in 1..65536, n_pages, table_columns and window >= 0", who);
  if (int64_t(j->batch) * j->q_heads > (1 << 24)) return fail(PM_E_LIMIT, "%s: at most 2^24 query rows", who);
  if (j->dtype != PM_DT_BF16 && j->dtype != PM_DT_F16) return fail(PM_E_INVALID, "%s: q and the caches are 16-bit floats", who);
  if (!(j->scale - j->scale == 0.0f)) return fail(PM_E_INVALID, "%s: scale must be finite", who);
  if ((j->new_k != nullptr) != (j->new_v != nullptr)) return fail(PM_E_INVALID, "%s: new_k and new_v come together", who);
  if (!j->batch) return PM_OK;
  const bool cached = j->n_pages > 0 && j->table_columns > 0;
  if (!j->q || !j->lengths || !j->out || (cached && (!j->k_cache || !j->v_cache || !j->table)))
    return fail(PM_E_INVALID, "%s: NULL buffer", who);
  if (!aligned(j->q, 16) || !aligned(j->k_cache, 16) || !aligned(j->v_cache, 16) || !aligned(j->new_k, 16) || !aligned(j->new_v, 16) ||
      !aligned(j->out, 16) || !aligned(j->table, 4) || !aligned(j->lengths, 4) || !aligned(j->lse, 4))
    return fail(PM_E_INVALID, "%s: q, the caches, new_k, new_v and out must be 16-byte aligned", who);
  const int64_t strides[] = {j->q_stride, j->q_head_stride, j->k_page_stride, j->k_token_stride, j->k_head_stride,
                             j->v_page_stride, j->v_token_stride, j->v_head_stride,
                             j->new_k ? j->new_k_stride : 0, j->new_k ? j->new_k_head_stride : 0,
                             j->new_k ? j->new_v_stride : 0, j->new_k ? j->new_v_head_stride : 0};
  for (const int64_t s : strides)
    if (s < 0 || s % 8) return fail(PM_E_INVALID, "%s: strides must be multiples of 8 elements", who);
  if (j->table_stride < 0) return fail(PM_E_INVALID, "%s: table_stride must be >= 0", who);
  const size_t need = pm_paged_attention_scratch_bytes(j->batch, j->q_heads, j->kv_heads, j->head_dim);
  if (!scratch || !aligned(scratch, 256) || scratch_bytes < need)
    return fail(PM_E_INVALID, "%s: needs %zu bytes of scratch, 256-byte aligned", who, need);
  int sms = 0;
  const int rc = sm_count(&sms);
  if (rc != PM_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = j->dtype == PM_DT_BF16 ? launch<bf16>(*j, s) : launch<fp16>(*j, s);
  return e == cudaSuccess ? PM_OK : cuda_fail(e, "pm_paged_attention_device launch");
}
