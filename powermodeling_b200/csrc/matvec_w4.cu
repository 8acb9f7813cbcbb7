// The product of a few tokens with a matrix of 4-bit weights with a scale
// (and a zero point) per group:
//   y[m, n] = sum_g s[n, g] sum_{k in g} x[m, k] (q[n, k] - z[n, g]).
//
// The weights are read once and bound it.
//  * A warp owns 32 rows of weights and 256 (128) values of k at a time, 4 KB
//    that it copies into shared memory asynchronously, three stages deep.  The
//    8 warps of a CTA stand side by side along n or along k, so a stage is 32
//    KB whatever the matrix's shape: enough bytes in flight with two CTAs an SM.
//    The tokens' values for a stage are copied beside it, for all warps, and
//    each serves two tiles of 16 rows in registers: unpacking has to keep up
//    with the memory on the integer pipe, where every other instruction counts.
//  * A nibble is masked into a 16-bit float's mantissa, exactly.  The matrix
//    instruction multiplies 16 rows by 8 tokens with exact products and 32-bit
//    sums; the scale enters once a group, in 32 bits.  So nothing is rounded
//    to 16 bits before the output.
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

constexpr int kWarps = 8, kThreads = 256, kRows = 32;    // rows of a warp's tile
constexpr int kXPad = 64;                                // bytes after a token's values: neighbours in other banks

// Up to 8 tokens: tiles of 256 k, which halves what a stage costs besides its
// products; up to 16: of 128 k, as the tokens' values take the room.
template <int NT>
struct Tile {
  static constexpr int kK = NT == 1 ? 256 : 128, kStages = NT == 1 ? 3 : 4;
  static constexpr int kPitch = kK / 2, kPieces = kPitch / 16;                 // a row, in 16-byte pieces
  static constexpr int kBytes = kRows * kPitch, kStageBytes = kWarps * kBytes;
  // Pieces lie in an order of the row's own, so that 8 rows x 4 words meet all 32 banks.
  static __device__ __forceinline__ int turn(int row) { return kPieces == 8 ? row & 7 : row >> 1 & 3; }
};

// Bytes of a stage with the values of `tokens` tokens, a multiple of the 128 in which rows take turns.
template <int NT>
__host__ __device__ inline int stage_size(int tokens, int stage_k) {
  return Tile<NT>::kStageBytes + (tokens * (stage_k * 2 + kXPad) + 127) / 128 * 128;
}

struct W4Args {
  int tokens, n, k, group, groups, scales32;
  int64_t x_stride, weight_stride;
  const void* x;
  const uint8_t* weight;
  const void* scales;
  const uint8_t* zeros;
  void* y;
  int warps_n;                                           // warps along n; the others along k
  int vector_scales;                                     // scales 16-byte, zeros 4-byte aligned
  int x_shift;                                           // log2 of the 16-byte pieces of a token in a stage
  int group_shift;                                       // log2 of the 32-k blocks of a group, -1: no power of two
  int slice;                                             // k of one CTA of the cluster, a multiple of the stage's
};

constexpr uint32_t kOnes = 0x3f803f80u;                  // two bf16 ones

// (a & b) | c in one instruction.
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// The pairs (0,4), (1,5), (2,6), (3,7) of a word's nibbles as 16-bit floats.
// bf16: the mantissa takes a nibble as 128 + q; what is 128 + z too much of
// every product is taken off a group's sum, where the tokens' sums come from
// a matrix instruction with ones.  (Subtracting in the pairs costs 8
// instructions per 512 weights more, and issue slots are what is short.)
// The offset costs 32-bit sums of 2^5 times the size, 2^-19 of a result that
// is rounded to 2^-9.
// fp16: a mantissa holds a nibble as 1024 + q, and four bits further up as
// 1024 + 16 q; one subtraction and one fused multiply-add bring both to q - z
// exactly.  The offset would cost 2^-16 here, too near the output's 2^-12.
template <class T> struct Nibbles;
template <> struct Nibbles<bf16> {
  static constexpr bool kOffset = true;
  static __device__ __forceinline__ uint32_t zero(uint32_t) { return 0; }
  static __device__ __forceinline__ void unpack(uint32_t w, uint32_t, uint32_t (&p)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = and_or(w >> (4 * i), 0x000f000fu, 0x43004300u);
  }
};
template <> struct Nibbles<fp16> {
  static constexpr bool kOffset = false;
  static __device__ __forceinline__ uint32_t zero(uint32_t z) { return 0x64006400u | z * 0x10001u; }   // 1024 + z
  static __device__ __forceinline__ void unpack(uint32_t w, uint32_t zero, uint32_t (&p)[4]) {
    const __half2 z = *reinterpret_cast<const __half2*>(&zero);
    const uint32_t high = and_or(zero << 4, 0x00f000f0u, 0xd400d400u);                                  // -(64 + z)
    const uint32_t sixteenth = 0x2c002c00u;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t u = i ? w >> 8 : w;
      const uint32_t a = and_or(u, 0x000f000fu, 0x64006400u), b = and_or(u, 0x00f000f0u, 0x64006400u);
      const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), z);
      const __half2 y = __hfma2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&sixteenth),
                                *reinterpret_cast<const __half2*>(&high));
      p[2 * i] = *reinterpret_cast<const uint32_t*>(&x);
      p[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&y);
    }
  }
};
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

// GB: blocks of 32 k per scale within a tile (1 to all of them); 1 also serves
// the group sizes that the tile's k is no multiple of, or no divisor.
// Aligned: rows of weights and tokens start on 16-byte boundaries.
template <class T, int NT, int GB, bool Aligned>
__global__ void __launch_bounds__(kThreads, 2) w4_kernel(const __grid_constant__ W4Args a) {
  extern __shared__ __align__(128) uint8_t smem[];
  using L = Tile<NT>;
  constexpr int kStages = L::kStages, kGroups = L::kK / 32 / GB;               // scales of a row in a tile
  constexpr int kRowLanes = 32 / L::kPieces, kCopies = kRows / kRowLanes;      // rows that one round of copies takes
  constexpr bool kOffset = Nibbles<T>::kOffset;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int warps_k = kWarps / a.warps_n, wn = warp % a.warps_n, wk = warp / a.warps_n;
  const int stage_k = warps_k * L::kK;
  const int m0 = blockIdx.z * 8 * NT, tokens = min(a.tokens - m0, 8 * NT);
  const int x_row = stage_k * 2 + kXPad;
  const int stage_bytes = stage_size<NT>(min(a.tokens, 8 * NT), stage_k);
  const int k_first = blockIdx.x * a.slice, k_last = min(a.k, k_first + a.slice);
  const int n_stages = k_last > k_first ? (k_last - k_first + stage_k - 1) / stage_k : 0;
  const int n0 = (blockIdx.y * a.warps_n + wn) * kRows;
  const uint32_t ring = smem_addr(smem);

  // This lane's copies of its warp's tile: every kRowLanes-th row, one piece
  // each.  The sources move on by a stage at a time.
  const int w_row = lane / L::kPieces, w_piece = lane % L::kPieces;
  const int piece_k = k_first + wk * L::kK + w_piece * 32;
  const uint8_t* w_base = a.weight + int64_t(blockIdx.y) * a.warps_n * kRows * a.weight_stride;   // this CTA's rows: offsets of 32 bits
  uint32_t w_off = uint32_t(wn * kRows + w_row) * uint32_t(a.weight_stride) + uint32_t(piece_k >> 1);
  const uint32_t w_step = kRowLanes * uint32_t(a.weight_stride);
  const int w_rows = a.n - n0 - w_row;                   // rows below this one that there are
  uint32_t w_dst[2];                                     // the place in the ring, by the row's turn
#pragma unroll
  for (int c = 0; c < 2; ++c) w_dst[c] = ring + warp * L::kBytes + w_row * L::kPitch + ((w_piece ^ L::turn(w_row + c * kRowLanes)) * 16);
  int w_left = a.k - piece_k;                            // k from here on
  // ... and of the tokens' values of the whole stage, 8 at a time
  const int lg = a.x_shift, x_tokens = kThreads >> lg;   // pieces of a token: 2^lg; tokens that one round of copies serves
  const int x_piece = threadIdx.x & ((1 << lg) - 1), x_m = threadIdx.x >> lg;
  const T* x_src = static_cast<const T*>(a.x) + (int64_t(m0) + min(x_m, tokens - 1)) * a.x_stride + k_first + x_piece * 8;
  const uint32_t x_dst = ring + L::kStageBytes + x_m * x_row + x_piece * 16;
  int x_left = a.k - k_first - x_piece * 8;
  int next = 0;                                          // the next copies' stage

  auto fetch = [&](bool some) {
    if (some) {
      const uint32_t at = next * stage_bytes;
      const int bytes = min(max((w_left + 1) >> 1, 0), 16);
      if (Aligned && __all_sync(0xffffffffu, bytes == 16 && w_rows > (kCopies - 1) * kRowLanes)) {
#pragma unroll
        for (int c = 0; c < kCopies; ++c) copy16(w_dst[c & 1] + at + c * kRowLanes * L::kPitch, w_base + (w_off + c * w_step), 16);
      } else {
#pragma unroll
        for (int c = 0; c < kCopies; ++c) {
          const int n = kRowLanes * c < w_rows ? bytes : 0;
          const uint8_t* src = n ? w_base + (w_off + c * w_step) : a.weight;
          const uint32_t dst = w_dst[c & 1] + at + c * kRowLanes * L::kPitch;
          if constexpr (Aligned) copy16(dst, src, n);
          else sts128(dst, load_any(src, n));
        }
      }
      const int x_bytes = 2 * min(max(x_left, 0), 8);    // zeros beyond k
      for (int m = x_m; m < tokens; m += x_tokens) {
        const T* src = x_bytes ? x_src + (m - x_m) * a.x_stride : static_cast<const T*>(a.x);
        if constexpr (Aligned) copy16(x_dst + at + (m - x_m) * x_row, src, x_bytes);
        else sts128(x_dst + at + (m - x_m) * x_row, keep(load_any(reinterpret_cast<const uint8_t*>(src), x_bytes), x_bytes >> 1));
      }
      w_off += stage_k / 2;
      x_src += stage_k;
      w_left -= stage_k;
      x_left -= stage_k;
      next = next == kStages - 1 ? 0 : next + 1;
    }
    commit();
  };

  // Scales and zero points of row `lane`, one stage ahead of their use and as
  // they are in memory: converting them here would wait for them here.  A
  // tile's lie side by side, one access where that is aligned.
  constexpr int kZeroWords = kGroups > 4 ? 2 : 1;
  uint32_t scale_next[kGroups], zero_next[kGroups];
  const int per = a.group / 32;
  const int64_t scale_row = int64_t(min(n0 + lane, a.n - 1)) * a.groups;
  const bool side_by_side = kGroups > 1 && per == GB && a.groups % kGroups == 0 && a.vector_scales;
  auto fetch_scales = [&](int i) {
    const int block0 = (k_first + i * stage_k + wk * L::kK) / 32;
    if (side_by_side) {
      const int64_t at = scale_row + min(block0 / GB, a.groups - kGroups);
      auto words = [&](const void* from, uint32_t* to, int bytes) {
        if (bytes == 32) {
          *reinterpret_cast<uint4*>(to) = __ldg(static_cast<const uint4*>(from));
          *reinterpret_cast<uint4*>(to + 4) = __ldg(static_cast<const uint4*>(from) + 1);
        } else if (bytes == 16) {
          *reinterpret_cast<uint4*>(to) = __ldg(static_cast<const uint4*>(from));
        } else if (bytes == 8) {
          *reinterpret_cast<uint2*>(to) = __ldg(static_cast<const uint2*>(from));
        } else if (bytes == 4) {
          *to = __ldg(static_cast<const uint32_t*>(from));
        } else {
          *to = __ldg(static_cast<const uint16_t*>(from));
        }
      };
      if (a.scales32) words(static_cast<const float*>(a.scales) + at, scale_next, 4 * kGroups);
      else words(static_cast<const T*>(a.scales) + at, scale_next, 2 * kGroups);
      if (a.zeros) words(a.zeros + at, zero_next, kGroups);
    } else {
#pragma unroll
      for (int e = 0; e < kGroups; ++e) {
        const int block = block0 + e * GB, group = a.group_shift >= 0 ? block >> a.group_shift : block / per;
        const int64_t at = scale_row + min(group, a.groups - 1);
        scale_next[e] = a.scales32 ? __ldg(static_cast<const uint32_t*>(a.scales) + at) : __ldg(static_cast<const uint16_t*>(a.scales) + at);
        if (a.zeros) zero_next[e] = __ldg(a.zeros + at);
      }
    }
  };

  float acc[2][NT][4] = {};
  if (n_stages) fetch_scales(0);
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(i < n_stages);
  int stage_now = 0;
  for (int i = 0; i < n_stages; ++i) {
    wait_groups<kStages - 2>();
    __syncthreads();                                     // stage i is there for all; stage i - 1 is read by all
    fetch(i + kStages - 1 < n_stages);
    float scale[kGroups];
    uint32_t zero[kGroups];
#pragma unroll
    for (int e = 0; e < kGroups; ++e) {
      const uint16_t half = uint16_t(side_by_side ? scale_next[e / 2] >> (16 * (e & 1)) : scale_next[e]);
      scale[e] = a.scales32 ? __uint_as_float(scale_next[e]) : to_float(*reinterpret_cast<const T*>(&half));
      zero[e] = a.zeros ? (side_by_side ? zero_next[kZeroWords == 2 ? e / 4 : 0] >> (8 * (e & 3)) : zero_next[e]) & 15u : 8u;
    }
    if (i + 1 < n_stages) fetch_scales(i + 1);
    const uint32_t stage = ring + stage_now * stage_bytes;
    stage_now = stage_now == kStages - 1 ? 0 : stage_now + 1;
    const uint32_t w_at = stage + warp * L::kBytes + g * L::kPitch + L::turn(g) * 16 + t * 4;
    const uint32_t x_at = stage + L::kStageBytes + wk * (L::kK * 2) + t * 16;
    uint32_t x_of[NT];                                   // columns beyond the tokens repeat the last one: nothing reads their sums
#pragma unroll
    for (int n = 0; n < NT; ++n) x_of[n] = x_at + min(n * 8 + g, tokens - 1) * x_row;
#pragma unroll
    for (int e = 0; e < kGroups; ++e) {
      float part[2][NT][4], x_sum[NT][4];
      uint32_t z[4];
      if constexpr (!kOffset) {
#pragma unroll
        for (int r = 0; r < 4; ++r) z[r] = Nibbles<T>::zero(a.zeros ? __shfl_sync(0xffffffffu, zero[e], g + 8 * r) : 8u);
      }
#pragma unroll
      for (int b = e * GB; b < (e + 1) * GB; ++b) {
        uint32_t x[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint4 v = lds128(x_of[n] + b * 64);
          x[n][0] = __byte_perm(v.x, v.z, 0x5410);
          x[n][1] = __byte_perm(v.x, v.z, 0x7632);
          x[n][2] = __byte_perm(v.y, v.w, 0x5410);
          x[n][3] = __byte_perm(v.y, v.w, 0x7632);
          if constexpr (kOffset) {
            const uint32_t ones[4] = {kOnes, kOnes, kOnes, kOnes};
            if (b == e * GB) mma_first<T>(x_sum[n], ones, x[n][0], x[n][1]);
            else mma<T>(x_sum[n], ones, x[n][0], x[n][1]);
            mma<T>(x_sum[n], ones, x[n][2], x[n][3]);
          }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          uint32_t p0[4], p1[4];
          Nibbles<T>::unpack(lds32((w_at ^ (b * 16)) + (16 * r) * L::kPitch), z[2 * r], p0);
          Nibbles<T>::unpack(lds32((w_at ^ (b * 16)) + (16 * r + 8) * L::kPitch), z[2 * r + 1], p1);
          const uint32_t a0[4] = {p0[0], p1[0], p0[1], p1[1]}, a1[4] = {p0[2], p1[2], p0[3], p1[3]};
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (b == e * GB) mma_first<T>(part[r][n], a0, x[n][0], x[n][1]);
            else mma<T>(part[r][n], a0, x[n][0], x[n][1]);
            mma<T>(part[r][n], a1, x[n][2], x[n][3]);
          }
        }
      }
      const float offset = 128.0f + float(zero[e]);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float s0 = __shfl_sync(0xffffffffu, scale[e], g + 16 * r), s1 = __shfl_sync(0xffffffffu, scale[e], g + 16 * r + 8);
        float o0 = 136.0f, o1 = 136.0f;
        if (kOffset && a.zeros) {
          o0 = __shfl_sync(0xffffffffu, offset, g + 16 * r);
          o1 = __shfl_sync(0xffffffffu, offset, g + 16 * r + 8);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if constexpr (kOffset) {
            part[r][n][0] -= o0 * x_sum[n][0];
            part[r][n][1] -= o0 * x_sum[n][1];
            part[r][n][2] -= o1 * x_sum[n][2];
            part[r][n][3] -= o1 * x_sum[n][3];
          }
          acc[r][n][0] += s0 * part[r][n][0];
          acc[r][n][1] += s0 * part[r][n][1];
          acc[r][n][2] += s1 * part[r][n][2];
          acc[r][n][3] += s1 * part[r][n][3];
        }
      }
    }
  }
  wait_groups<0>();
  __syncthreads();

  // sums of the warps along k, then of the cluster's CTAs: [wk][row][token] in shared memory
  constexpr int kCols = 8 * NT;
  float* red = reinterpret_cast<float*>(smem);
  const int rows = a.warps_n * kRows;
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float* at = red + ((wk * rows + wn * kRows + 16 * r + g) * kCols + n * 8 + 2 * t);
      at[0] = acc[r][n][0];
      at[1] = acc[r][n][1];
      at[8 * kCols] = acc[r][n][2];
      at[8 * kCols + 1] = acc[r][n][3];
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
  // Rows of a CTA (32 to 256): as many as leave a CTA per SM, but at least 8
  // per token, so that the tokens' values, read again by every CTA, stay
  // within half of the weights' bytes.  Then the cluster's share of k: enough
  // CTAs for the SMs, each with at least two stages.
  const int held = a.tokens < 8 * NT ? a.tokens : 8 * NT;
  auto blocks_of = [&](int w) { return (a.n + kRows * w - 1) / (kRows * w); };
  int warps_n = 8;
  while (warps_n > 1 && blocks_of(warps_n) < sms && kRows * (warps_n / 2) >= 8 * held) warps_n /= 2;
  const int row_blocks = blocks_of(warps_n), stage_k = kWarps / warps_n * Tile<NT>::kK;
  int ranks = 1;
  while (ranks < 8 && row_blocks * ranks < sms && a.k > 2 * ranks * stage_k) ranks *= 2;
  const int stages = (a.k + stage_k - 1) / stage_k;
  a.warps_n = warps_n;
  a.x_shift = 31 - __builtin_clz(unsigned(stage_k / 8));
  const unsigned per = unsigned(a.group / 32);
  a.group_shift = per & (per - 1) ? -1 : 31 - __builtin_clz(per);
  a.slice = (stages + ranks - 1) / ranks * stage_k;
  const size_t bytes = size_t(Tile<NT>::kStages) * stage_size<NT>(held, stage_k);
  const auto kernel = w4_kernel<T, NT, GB, Aligned>;
  ensure_dynamic_smem(kernel, 1024, bytes, g_smem[std::is_same<T, fp16>::value][NT - 1][GB == 8 ? 3 : GB / 2][Aligned]);
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
  if (NT == 1 && a.group % 256 == 0) return launch_shape<T, NT, NT == 1 ? 8 : 4, Aligned>(a, sms, s);
  if (a.group == 128 || (NT == 2 && a.group % 128 == 0)) return launch_shape<T, NT, 4, Aligned>(a, sms, s);
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
  if (j->weight_stride > (1 << 23)) return fail(PM_E_LIMIT, "%s: weight rows lie at most 2^23 bytes apart", who);
  if (j->x_stride < j->k || j->weight_stride < (int64_t(j->k) + 1) / 2)
    return fail(PM_E_INVALID, "%s: strides must be at least a row", who);
  if (!j->x || !j->weight || !j->scales || !j->y) return fail(PM_E_INVALID, "%s: NULL buffer", who);
  if (!aligned(j->x, 2) || !aligned(j->y, 2) || !aligned(j->scales, type_bytes(j->scales_dtype)))
    return fail(PM_E_INVALID, "%s: a buffer is not aligned to its elements", who);
  int sms = 0;
  const int rc = sm_count(&sms);
  if (rc != PM_OK) return rc;
  W4Args a{j->tokens, j->n, j->k, j->group, int((int64_t(j->k) + j->group - 1) / j->group), j->scales_dtype == PM_DT_F32,
           j->x_stride, j->weight_stride, j->x, j->weight, j->scales, j->zeros, j->y, 0, aligned(j->scales, 16) && aligned(j->zeros, 4), 0, 0, 0};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = j->dtype == PM_DT_BF16 ? launch<bf16>(a, sms, s) : launch<fp16>(a, sms, s);
  return e == cudaSuccess ? PM_OK : cuda_fail(e, "pm_matvec_w4_device launch");
}
