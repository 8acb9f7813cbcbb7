// The product of a few tokens with a matrix of 4-bit weights with a scale
// (and a zero point) per group:
//   y[m, n] = sum_g s[n, g] sum_{k in g} x[m, k] (q[n, k] - z[n, g]).
//
// The weights are read once and bound it.
//  * A warp owns 16 rows of weights and 256 values of k at a time, 2 KB that
//    it copies into shared memory asynchronously, four stages deep.  The 8
//    warps of a CTA stand side by side along n or along k, so a stage is 16 KB
//    whatever the matrix's shape: enough bytes in flight with two CTAs an SM.
//    The tokens' values for a stage are copied beside it, for all warps.
//  * q - z is an integer that 16-bit floats hold exactly: four nibbles are
//    masked into the mantissas of 128 (bf16) or 1024 (fp16) and the same
//    number plus z is subtracted.  The matrix instruction multiplies 16 rows
//    by 8 tokens with exact products and 32-bit sums; the scale enters once a
//    group, in 32 bits.  So nothing is rounded before the output.
//  * k is summed in an order that suits the nibbles: a lane's word holds k =
//    0..7 of its eight, and the pairs (0,4), (1,5), (2,6), (3,7) are the
//    instruction's neighbours, for the weights and for the tokens alike.
//  * 8 tokens (16 in two halves) are the instruction's columns: mma.sync, as
//    tcgen05's tiles begin at 128 x 8 with both operands in shared memory,
//    and the unpacked weights come from registers.
//  * Few rows: the CTAs of a cluster share k and add their sums through
//    distributed shared memory, in rank order, so results do not vary.
#include <cooperative_groups.h>

#include "blocks.cuh"

namespace cg = cooperative_groups;

namespace pm {
namespace blk {
namespace {

constexpr int kWarps = 8, kThreads = 256, kStages = 4;
constexpr int kWarpK = 256;                              // k of a warp's tile
constexpr int kTileBytes = 16 * kWarpK / 2;              // 16 rows
constexpr int kWeightBytes = kWarps * kTileBytes;        // a stage
constexpr int kXPad = 64;                                // bytes after a token's values: neighbours in other banks

struct W4Args {
  int tokens, n, k, group, groups, scales32;
  int64_t x_stride, weight_stride;
  const void* x;
  const uint8_t* weight;
  const void* scales;
  const uint8_t* zeros;
  void* y;
  int warps_n;                                           // warps along n; the others along k
  int slice;                                             // k of one CTA of the cluster, a multiple of the stage's
};

template <class T> struct Magic;
template <> struct Magic<bf16> { static constexpr uint32_t value = 0x43004300u; };   // 128
template <> struct Magic<fp16> { static constexpr uint32_t value = 0x64006400u; };   // 1024

__device__ __forceinline__ uint32_t sub2(bf16*, uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t sub2(fp16*, uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// The pairs (0,4), (1,5), (2,6), (3,7) of a word's nibbles, less the zero point.
template <class T>
__device__ __forceinline__ void unpack(uint32_t w, uint32_t zero, uint32_t (&p)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    p[i] = sub2(static_cast<T*>(nullptr), ((w >> (4 * i)) & 0x000f000fu) | Magic<T>::value, zero);
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" :: "r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// 16 bytes from any address, of which `bytes` are read: aligned words that
// hold at least one of them, shifted into place.
__device__ __forceinline__ uint4 load_any(const uint8_t* p, int bytes) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  const uint32_t* w = reinterpret_cast<const uint32_t*>(a & ~uintptr_t(3));
  const int skew = int(a & 3), words = bytes > 0 ? (skew + bytes + 3) >> 2 : 0;
  uint32_t v[5];
#pragma unroll
  for (int i = 0; i < 5; ++i) v[i] = i < words ? __ldg(w + i) : 0u;
  uint4 r;
  r.x = __funnelshift_r(v[0], v[1], 8 * skew);
  r.y = __funnelshift_r(v[1], v[2], 8 * skew);
  r.z = __funnelshift_r(v[2], v[3], 8 * skew);
  r.w = __funnelshift_r(v[3], v[4], 8 * skew);
  return r;
}

// The first `count` of eight 16-bit values, zeros after them.
__device__ __forceinline__ uint4 keep(uint4 v, int count) {
  auto word = [&](uint32_t w, int i) { return count >= 2 * i + 2 ? w : count == 2 * i + 1 ? w & 0xffffu : 0u; };
  return make_uint4(word(v.x, 0), word(v.y, 1), word(v.z, 2), word(v.w, 3));
}

// GB: blocks of 32 k per scale within a warp's 256 (1, 2, 4, 8); 1 also serves
// the group sizes that 256 is no multiple of, or no divisor.
// Aligned: rows of weights and tokens start on 16-byte boundaries.
template <class T, int NT, int GB, bool Aligned>
__global__ void __launch_bounds__(kThreads, 2) w4_kernel(const __grid_constant__ W4Args a) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int kGroups = 8 / GB;                        // scales of a row in a warp's tile
  constexpr int kRegs = GB == 1 ? 2 : 1;                 // ... of which each of four lanes holds this many
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int warps_k = kWarps / a.warps_n, wn = warp % a.warps_n, wk = warp / a.warps_n;
  const int stage_k = warps_k * kWarpK;
  const int m0 = blockIdx.z * 8 * NT, tokens = min(a.tokens - m0, 8 * NT);
  const int x_row = stage_k * 2 + kXPad;
  const int stage_bytes = kWeightBytes + min(a.tokens, 8 * NT) * x_row;
  const int k_first = blockIdx.x * a.slice, k_last = min(a.k, k_first + a.slice);
  const int n_stages = k_last > k_first ? (k_last - k_first + stage_k - 1) / stage_k : 0;
  const int n0 = (blockIdx.y * a.warps_n + wn) * 16;
  const uint32_t ring = smem_addr(smem);
  const T* xs = static_cast<const T*>(a.x) + int64_t(m0) * a.x_stride;

  auto fetch = [&](int i) {
    if (i < n_stages) {
      const uint32_t stage = ring + (i % kStages) * stage_bytes;
      // this warp's tile: 16 rows of 128 bytes, the row's 16-byte pieces in an order of its own (piece ^ row)
      const int k0 = k_first + i * stage_k + wk * kWarpK;
      const uint32_t dst = stage + warp * kTileBytes;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int row = c * 4 + (lane >> 3), piece = lane & 7;
        const int k = k0 + piece * 32;
        const int bytes = n0 + row < a.n ? min(max((a.k - k + 1) >> 1, 0), 16) : 0;
        const uint8_t* src = a.weight + int64_t(bytes ? n0 + row : 0) * a.weight_stride + (bytes ? k >> 1 : 0);
        const uint32_t at = dst + row * 128 + ((piece ^ (row & 7)) << 4);
        if constexpr (Aligned) copy16(at, src, bytes);
        else sts128(at, load_any(src, bytes));
      }
      // the tokens' values of the whole stage, zeros beyond k
      const int pieces = stage_k / 8;
      for (int p = threadIdx.x; p < tokens * pieces; p += kThreads) {
        const int m = p / pieces, piece = p - m * pieces;
        const int k = k_first + i * stage_k + piece * 8;
        const int bytes = 2 * min(max(a.k - k, 0), 8);
        const T* src = xs + m * a.x_stride + (bytes ? k : 0);
        const uint32_t at = stage + kWeightBytes + m * x_row + piece * 16;
        if constexpr (Aligned) copy16(at, src, bytes);
        else sts128(at, keep(load_any(reinterpret_cast<const uint8_t*>(src), bytes), bytes >> 1));
      }
    }
    commit();
  };

  // scales (and zero points) of rows g and g + 8, one stage ahead of their use
  float scale_next[2][kRegs];
  uint32_t zero_next[2][kRegs];
  auto fetch_scales = [&](int i) {
    const int block0 = (k_first + i * stage_k + wk * kWarpK) / 32, per = a.group / 32;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int e = 0; e < kRegs; ++e) {
        const int block = block0 + (GB == 1 ? t + 4 * e : min(t, kGroups - 1) * GB);
        const int64_t at = int64_t(min(n0 + g + 8 * r, a.n - 1)) * a.groups + min(block / per, a.groups - 1);
        scale_next[r][e] = a.scales32 ? __ldg(static_cast<const float*>(a.scales) + at)
                                      : to_float(static_cast<const T*>(a.scales)[at]);
        zero_next[r][e] = Magic<T>::value | (a.zeros ? uint32_t(__ldg(a.zeros + at) & 15) * 0x10001u : 0x00080008u);
      }
  };

  float acc[NT][4] = {};
  if (n_stages) fetch_scales(0);
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(i);
  for (int i = 0; i < n_stages; ++i) {
    wait_groups<kStages - 2>();
    __syncthreads();                                     // stage i is there for all; stage i - 1 is read by all
    fetch(i + kStages - 1);
    float scale[2][kRegs];
    uint32_t zero[2][kRegs];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int e = 0; e < kRegs; ++e) scale[r][e] = scale_next[r][e], zero[r][e] = zero_next[r][e];
    if (i + 1 < n_stages) fetch_scales(i + 1);
    const uint32_t stage = ring + (i % kStages) * stage_bytes;
    const uint32_t w_at = stage + warp * kTileBytes + g * 128 + t * 4;
    const uint32_t x_at = stage + kWeightBytes + wk * (kWarpK * 2) + t * 16;
    float part[NT][4];
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      if (b % GB == 0) {
#pragma unroll
        for (int n = 0; n < NT; ++n) part[n][0] = part[n][1] = part[n][2] = part[n][3] = 0.0f;
      }
      const int from = (lane & ~3) | (GB == 1 ? b & 3 : b / GB);
      const int e = GB == 1 ? b >> 2 : 0;
      const uint32_t z0 = __shfl_sync(0xffffffffu, zero[0][e], from), z1 = __shfl_sync(0xffffffffu, zero[1][e], from);
      uint32_t p0[4], p1[4];
      unpack<T>(lds32(w_at + ((b ^ g) << 4)), z0, p0);
      unpack<T>(lds32(w_at + 8 * 128 + ((b ^ g) << 4)), z1, p1);
      const uint32_t a0[4] = {p0[0], p1[0], p0[1], p1[1]}, a1[4] = {p0[2], p1[2], p0[3], p1[3]};
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        // columns beyond the tokens repeat the last one: nothing reads their sums
        const uint4 x = lds128(x_at + min(n * 8 + g, tokens - 1) * x_row + b * 64);
        mma<T>(part[n], a0, __byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632));
        mma<T>(part[n], a1, __byte_perm(x.y, x.w, 0x5410), __byte_perm(x.y, x.w, 0x7632));
      }
      if (b % GB == GB - 1) {
        const float s0 = __shfl_sync(0xffffffffu, scale[0][e], from), s1 = __shfl_sync(0xffffffffu, scale[1][e], from);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          acc[n][0] += s0 * part[n][0];
          acc[n][1] += s0 * part[n][1];
          acc[n][2] += s1 * part[n][2];
          acc[n][3] += s1 * part[n][3];
        }
      }
    }
  }
  wait_groups<0>();
  __syncthreads();

  // sums of the warps along k, then of the cluster's CTAs: [wk][row][token] in shared memory
  constexpr int kCols = 8 * NT;
  float* red = reinterpret_cast<float*>(smem);
  const int rows = a.warps_n * 16;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float* at = red + ((wk * rows + wn * 16 + g) * kCols + n * 8 + 2 * t);
    at[0] = acc[n][0];
    at[1] = acc[n][1];
    at[8 * kCols] = acc[n][2];
    at[8 * kCols + 1] = acc[n][3];
  }
  __syncthreads();
  const int cells = rows * kCols;
  if (warps_k > 1) {
    for (int c = threadIdx.x; c < cells; c += kThreads) {
      float v = red[c];
      for (int w = 1; w < warps_k; ++w) v += red[w * cells + c];
      red[c] = v;
    }
  }
  const int ranks = gridDim.x;
  if (ranks > 1) cg::this_cluster().sync();
  else __syncthreads();
  if (blockIdx.x == 0) {
    T* y = static_cast<T*>(a.y) + int64_t(m0) * a.n;
    const int first = blockIdx.y * rows;
    for (int c = threadIdx.x; c < rows * tokens; c += kThreads) {
      const int m = c / rows, row = c - m * rows;
      if (first + row >= a.n) continue;
      float v = red[row * kCols + m];
      for (int r = 1; r < ranks; ++r) v += cg::this_cluster().map_shared_rank(red, r)[row * kCols + m];
      y[int64_t(m) * a.n + first + row] = from_float<T>(v);
    }
  }
  if (ranks > 1) cg::this_cluster().sync();              // a CTA's sums stay until rank 0 has them
}

// ---------------------------------------------------------------- launch
std::atomic<int> g_smem[2][2][4][2][kMaxDevices];

template <class T, int NT, int GB, bool Aligned>
cudaError_t launch_shape(W4Args a, int sms, cudaStream_t s) {
  // Rows of a CTA (16 to 128): as many as leave a CTA per SM, but at least 8
  // per token, so that the tokens' values, read again by every CTA, stay
  // within half of the weights' bytes.  Then the cluster's share of k: enough
  // CTAs for the SMs, each with at least 4 stages' worth of its warps' k.
  const int held = a.tokens < 8 * NT ? a.tokens : 8 * NT;
  int warps_n = 8;
  while (warps_n > 1 && (a.n + 16 * warps_n - 1) / (16 * warps_n) < sms && 16 * (warps_n / 2) >= 8 * held) warps_n /= 2;
  const int row_blocks = (a.n + 16 * warps_n - 1) / (16 * warps_n), stage_k = kWarps / warps_n * kWarpK;
  int ranks = 1;
  while (ranks < 8 && row_blocks * ranks < sms && a.k > 2 * ranks * stage_k) ranks *= 2;
  const int stages = (a.k + stage_k - 1) / stage_k;
  a.warps_n = warps_n;
  a.slice = (stages + ranks - 1) / ranks * stage_k;
  const size_t bytes = size_t(kStages) * (kWeightBytes + size_t(held) * (stage_k * 2 + kXPad));
  const auto kernel = w4_kernel<T, NT, GB, Aligned>;
  ensure_dynamic_smem(kernel, 1024, bytes, g_smem[std::is_same<T, fp16>::value][NT - 1][GB == 1 ? 0 : GB == 2 ? 1 : GB == 4 ? 2 : 3][Aligned]);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ranks, row_blocks, (a.tokens + 8 * NT - 1) / (8 * NT));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ranks > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <class T, int NT, bool Aligned>
cudaError_t launch_group(const W4Args& a, int sms, cudaStream_t s) {
  if (a.group == 64) return launch_shape<T, NT, 2, Aligned>(a, sms, s);
  if (a.group == 128) return launch_shape<T, NT, 4, Aligned>(a, sms, s);
  if (a.group % 256 == 0) return launch_shape<T, NT, 8, Aligned>(a, sms, s);
  return launch_shape<T, NT, 1, Aligned>(a, sms, s);
}

template <class T>
cudaError_t launch(const W4Args& a, int sms, cudaStream_t s) {
  const bool aligned_rows = aligned(a.weight, 16) && a.weight_stride % 16 == 0 && aligned(a.x, 16) && (a.x_stride % 8 == 0 || a.tokens == 1);
  if (a.tokens <= 8) return aligned_rows ? launch_group<T, 1, true>(a, sms, s) : launch_group<T, 1, false>(a, sms, s);
  return aligned_rows ? launch_group<T, 2, true>(a, sms, s) : launch_group<T, 2, false>(a, sms, s);
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
           j->x_stride, j->weight_stride, j->x, j->weight, j->scales, j->zeros, j->y, 0, 0};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = j->dtype == PM_DT_BF16 ? launch<bf16>(a, sms, s) : launch<fp16>(a, sms, s);
  return e == cudaSuccess ? PM_OK : cuda_fail(e, "pm_matvec_w4_device launch");
}
