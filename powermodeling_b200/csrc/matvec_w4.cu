// The product of a few tokens with a matrix of 4-bit weights with a scale
// (and a zero point) per group:
//   y[m, n] = sum_g s[n, g] sum_{k in g} x[m, k] (q[n, k] - z[n, g]).
//
// The weights are read once and bound it.
//  * A warp owns 32 rows of weights and 256 (128) values of k at a time, a
//    tile of 4 KB.  8 such warps stand side by side along n or along k, so a
//    stage is 32 KB whatever the matrix's shape: with three stages and two
//    CTAs an SM enough bytes are in flight.  A ninth warp fills the stages by
//    tensor copies, the tokens' values beside the weights (rows that start at
//    any byte: four warps that shift words into place), so the others do
//    nothing but unpack and multiply: issue slots, not bytes, are short.
//  * Each token pair serves two tiles of 16 rows in registers.
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
#include <cuda.h>

#include <cmath>

#include "blocks.cuh"

namespace cg = cooperative_groups;

namespace pm {
namespace blk {
namespace {

constexpr int kWarps = 8, kRows = 32;                    // warps that multiply; rows of a warp's tile
constexpr uint64_t kWaitNs = 2ull * 1000000000ull;       // bound on any single wait; a result that it poisons is NaN

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

// Bytes of a stage with the values of `tokens` tokens, a multiple of the
// swizzle's 1 KB: per warp along k its weights, then per warp along k its tokens' values.
template <int NT>
__host__ __device__ inline int stage_size(int tokens, int warps_k) {
  return Tile<NT>::kStageBytes + (warps_k * tokens * Tile<NT>::kK * 2 + 1023) / 1024 * 1024;
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
  int vector_scales;                                     // scales 16-byte, zeros 8-byte aligned
  int group_shift;                                       // log2 of the 32-k blocks of a group, -1: no power of two
  int stages;                                            // stages of a row block: its k over the stage's
  int ranks;                                             // CTAs of a cluster, which share each row block's stages
  float* part;                                           // ranks == 1: sums of cut row blocks, [2 * CTAs][rows][8 NT]
};

// (a & b) | c in one instruction.
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// The pairs (0,4), (1,5), (2,6), (3,7) of a word's nibbles, less the zero
// point and over kScale, as exact 16-bit floats.  Integer instructions are
// what the kernel has least of, so two nibble positions of a half are taken
// where they lie and one shift brings the other two: five and four fused
// multiply-adds a word.
// bf16: the bits of an integer below 256 are that integer times 2^-133 (the
// subnormals and the first binade are one even grid), so a nibble at bit 0 or
// bit 4 is n 2^-133 or n 2^-129, and n - z over 64 is one fma away.
// fp16: a nibble at bit 0 of 1024's mantissa is 1024 + n, at bit 4 1024 + 16 n.
template <class T> struct Nibbles;
template <> struct Nibbles<bf16> {
  static constexpr float kScale = 64.0f;
  static __device__ __forceinline__ uint32_t zero(uint32_t z) {
    const __nv_bfloat162 v = __float2bfloat162_rn(float(z) * -0.015625f);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ void unpack(uint32_t w, uint32_t zero, uint32_t (&p)[4]) {
    const uint32_t low = 0x7f007f00u, high = 0x7d007d00u;                      // 2^127, 2^123
    const __nv_bfloat162 z = *reinterpret_cast<const __nv_bfloat162*>(&zero);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t u = i ? w >> 8 : w, a = u & 0x000f000fu, b = u & 0x00f000f0u;
      const __nv_bfloat162 x = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&low), z);
      const __nv_bfloat162 y = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&b), *reinterpret_cast<const __nv_bfloat162*>(&high), z);
      p[2 * i] = *reinterpret_cast<const uint32_t*>(&x);
      p[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&y);
    }
  }
};
template <> struct Nibbles<fp16> {
  static constexpr float kScale = 1.0f;
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

__device__ __forceinline__ void barrier_init(uint32_t bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint32_t bar, int bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool barrier_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0;
}
__device__ __forceinline__ uint64_t nanoseconds() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// False when the wait runs out.
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity) {
  if (barrier_try(bar, parity)) return true;
  const uint64_t deadline = nanoseconds() + kWaitNs;
  while (!barrier_try(bar, parity))
    if (nanoseconds() > deadline) return false;
  return true;
}
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void multipliers_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// GB: blocks of 32 k per scale within a tile (1 to all of them); 1 also serves
// the group sizes that the tile's k is no multiple of, or no divisor.
// Copies: rows of weights and tokens start on 16-byte boundaries, and one lane
// of one warp copies boxes; else four warps copy words.
constexpr int kBoxThreads = 32, kWordThreads = 128;
template <class T, int NT, int GB, bool Boxes>
__global__ void __launch_bounds__(32 * kWarps + (Boxes ? kBoxThreads : kWordThreads), Boxes ? 2 : 1)
w4_kernel(const __grid_constant__ W4Args a, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x) {
  extern __shared__ uint8_t smem_raw[];
  using L = Tile<NT>;
  constexpr int kStages = L::kStages, kGroups = L::kK / 32 / GB, kCols = 8 * NT;
  __shared__ __align__(8) uint64_t bars[2 * kStages];    // a stage is full; it is read
  uint8_t* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int warps_k = kWarps / a.warps_n, wn = warp % a.warps_n, wk = warp / a.warps_n;
  const int stage_k = warps_k * L::kK, rows = a.warps_n * kRows;
  const int m0 = blockIdx.z * kCols, held = min(a.tokens, kCols), tokens = min(a.tokens - m0, kCols);
  const int stage_bytes = stage_size<NT>(held, warps_k);
  // The work is a line of stages, row block after row block.  A cluster's CTAs
  // each take a share of one block's; without clusters the line is cut into
  // equal runs.
  const int rank = blockIdx.x % a.ranks;
  int64_t first;
  int count;                                             // stages of this CTA: [first, first + count) of the line
  if (a.ranks > 1) {
    const int from = int(int64_t(a.stages) * rank / a.ranks);
    first = int64_t(blockIdx.x / a.ranks) * a.stages + from;
    count = int(int64_t(a.stages) * (rank + 1) / a.ranks) - from;
  } else {
    const int64_t total = int64_t((a.n + rows - 1) / rows) * a.stages;
    first = total * blockIdx.x / gridDim.x;
    count = int(total * (blockIdx.x + 1) / gridDim.x - first);
  }
  int block = int(first / a.stages), s = int(first - int64_t(block) * a.stages);
  const uint32_t ring = smem_addr(smem), full = smem_addr(bars), read = full + 8 * kStages;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      barrier_init(full + 8 * i, Boxes ? 1 : kWordThreads);
      barrier_init(read + 8 * i, kWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();

  if (warp >= kWarps) {
    // ------------------------------------------------ the copies
    const int me = threadIdx.x - 32 * kWarps;
    bool ok = true;
    for (int i = 0; i < count && ok; ++i) {
      const int place = i % kStages;
      const uint32_t stage = ring + place * stage_bytes, bar = full + 8 * place;
      const int k0 = s * stage_k;
      if (Boxes ? me == 0 : true) {
        if (i >= kStages) ok = barrier_wait(read + 8 * place, (i / kStages - 1) & 1);
        if (!ok) break;
        if constexpr (Boxes) {
          barrier_expect(bar, L::kStageBytes + warps_k * held * L::kK * 2);
          for (int w = 0; w < warps_k; ++w) {
            copy_box(stage + w * rows * L::kPitch, &map_w, (k0 + w * L::kK) / 2, block * rows, bar);
            copy_box(stage + L::kStageBytes + w * held * L::kK * 2, &map_x, k0 + w * L::kK, m0, bar);
          }
        } else {
          constexpr int kPieces = L::kStageBytes / 16 / kWordThreads;          // of a thread
#pragma unroll 16
          for (int c = 0; c < kPieces; ++c) {
            const int p = c * kWordThreads + me, tile = p / (kRows * L::kPieces), row = p / L::kPieces % kRows, piece = p % L::kPieces;
            const int n = block * rows + tile % a.warps_n * kRows + row, k = k0 + tile / a.warps_n * L::kK + piece * 32;
            const int bytes = n < a.n ? min(max((a.k - k + 1) >> 1, 0), 16) : 0;
            const uint8_t* src = a.weight + (bytes ? int64_t(n) * a.weight_stride + (k >> 1) : 0);
            sts128(stage + tile * L::kBytes + row * L::kPitch + ((piece ^ L::turn(row)) * 16), load_any(src, bytes));
          }
          for (int p = me; p < warps_k * tokens * (L::kK / 8); p += kWordThreads) {
            const int piece = p % (L::kK / 8), m = p / (L::kK / 8) % tokens, w = p / (L::kK / 8) / tokens;
            const int k = k0 + w * L::kK + piece * 8, left = min(max(a.k - k, 0), 8);
            const T* src = static_cast<const T*>(a.x) + (left ? int64_t(m0 + m) * a.x_stride + k : 0);
            sts128(stage + L::kStageBytes + ((w * held + m) * (L::kK / 8) + piece) * 16,
                   keep(load_any(reinterpret_cast<const uint8_t*>(src), 2 * left), left));
          }
          barrier_arrive(bar);
        }
      }
      if (++s == a.stages) s = 0, ++block;
    }
    if (Boxes && me == 0 && !ok)                         // copies under way land before the CTA goes
      for (int i = 0; i < kStages; ++i) barrier_wait(full + 8 * i, 0), barrier_wait(full + 8 * i, 1);
    if (a.ranks > 1) {
      cg::this_cluster().sync();
      cg::this_cluster().sync();
    }
    return;
  }

  // -------------------------------------------------- the products
  // Scales and zero points of row `lane`, one stage ahead of their use and as
  // they are in memory: converting them here would wait for them here.  A
  // tile's lie side by side, one access where that is aligned.
  constexpr int kZeroWords = kGroups > 4 ? 2 : 1;
  uint32_t scale_next[kGroups], zero_next[kGroups];
  const int per = a.group / 32;
  const bool side_by_side = kGroups > 1 && per == GB && a.groups % kGroups == 0 && a.vector_scales;
  auto fetch_scales = [&](int at_block, int at_s) {
    const int block0 = (at_s * stage_k + wk * L::kK) / 32;
    const int64_t scale_row = int64_t(min(at_block * rows + wn * kRows + lane, a.n - 1)) * a.groups;
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
        const int at_k = block0 + e * GB, group = a.group_shift >= 0 ? at_k >> a.group_shift : at_k / per;
        const int64_t at = scale_row + min(group, a.groups - 1);
        scale_next[e] = a.scales32 ? __ldg(static_cast<const uint32_t*>(a.scales) + at) : __ldg(static_cast<const uint16_t*>(a.scales) + at);
        if (a.zeros) zero_next[e] = __ldg(a.zeros + at);
      }
    }
  };

  float acc[2][NT][4] = {};
  bool ok = true;
  int s_first = s, place = 0;
  uint32_t parity = 0;
  float* red = nullptr;                                  // [wk][row][token], in the place of a row block's last stage
  // this lane's words of its tile (rows g + 8 r), and its tokens' values; columns beyond the tokens repeat the last one:
  // nothing reads their sums
  const int w_lane = warp * L::kBytes + g * L::kPitch + L::turn(g) * 16 + t * 4;
  int x_lane[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) x_lane[n] = L::kStageBytes + (wk * held + min(n * 8 + g, tokens - 1)) * (L::kK * 2) + t * 16;
  if (count) fetch_scales(block, s);
  for (int left = count; left > 0; --left) {
    float scale[kGroups];
    uint32_t zero[kGroups];
#pragma unroll
    for (int e = 0; e < kGroups; ++e) {
      const uint16_t half = uint16_t(side_by_side ? scale_next[e / 2] >> (16 * (e & 1)) : scale_next[e]);
      scale[e] = Nibbles<T>::kScale * (a.scales32 ? __uint_as_float(scale_next[e]) : to_float(*reinterpret_cast<const T*>(&half)));
      zero[e] = a.zeros ? (side_by_side ? zero_next[kZeroWords == 2 ? e / 4 : 0] >> (8 * (e & 3)) : zero_next[e]) & 15u : 8u;
    }
    const bool last = s + 1 == a.stages || left == 1;    // of this CTA in this row block
    if (left > 1) fetch_scales(s + 1 == a.stages ? block + 1 : block, s + 1 == a.stages ? 0 : s + 1);
    ok = ok && barrier_wait(full + 8 * place, parity);
    const int stage = place * stage_bytes;
    const int w_at = stage + w_lane;
#pragma unroll
    for (int e = 0; e < kGroups; ++e) {
      float part[2][NT][4];
      uint32_t z[4];
      {
        const uint32_t own = Nibbles<T>::zero(zero[e]);
#pragma unroll
        for (int r = 0; r < 4; ++r) z[r] = a.zeros ? __shfl_sync(0xffffffffu, own, g + 8 * r) : own;
      }
#pragma unroll
      for (int b = e * GB; b < (e + 1) * GB; ++b) {
        uint32_t x[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint4 v = *reinterpret_cast<const uint4*>(smem + stage + x_lane[n] + b * 64);
          x[n][0] = __byte_perm(v.x, v.z, 0x5410);
          x[n][1] = __byte_perm(v.x, v.z, 0x7632);
          x[n][2] = __byte_perm(v.y, v.w, 0x5410);
          x[n][3] = __byte_perm(v.y, v.w, 0x7632);
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          uint32_t p0[4], p1[4];
          const uint8_t* at = smem + (w_at ^ (b * 16)) + 16 * r * L::kPitch;
          Nibbles<T>::unpack(*reinterpret_cast<const uint32_t*>(at), z[2 * r], p0);
          Nibbles<T>::unpack(*reinterpret_cast<const uint32_t*>(at + 8 * L::kPitch), z[2 * r + 1], p1);
          const uint32_t a0[4] = {p0[0], p1[0], p0[1], p1[1]}, a1[4] = {p0[2], p1[2], p0[3], p1[3]};
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (b == e * GB) mma_first<T>(part[r][n], a0, x[n][0], x[n][1]);
            else mma<T>(part[r][n], a0, x[n][0], x[n][1]);
            mma<T>(part[r][n], a1, x[n][2], x[n][3]);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float s0 = __shfl_sync(0xffffffffu, scale[e], g + 16 * r), s1 = __shfl_sync(0xffffffffu, scale[e], g + 16 * r + 8);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          acc[r][n][0] += s0 * part[r][n][0];
          acc[r][n][1] += s0 * part[r][n][1];
          acc[r][n][2] += s1 * part[r][n][2];
          acc[r][n][3] += s1 * part[r][n][3];
        }
      }
    }
    ++s;
    if (last) {
      // the row block's sums over the warps along k, where nobody reads the stage any more
      multipliers_sync();
      red = reinterpret_cast<float*>(smem + stage);
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float* at = red + ((wk * rows + wn * kRows + 16 * r + g) * kCols + n * 8 + 2 * t);
          at[0] = ok ? acc[r][n][0] : NAN;
          at[1] = ok ? acc[r][n][1] : NAN;
          at[8 * kCols] = ok ? acc[r][n][2] : NAN;
          at[8 * kCols + 1] = ok ? acc[r][n][3] : NAN;
          acc[r][n][0] = acc[r][n][1] = acc[r][n][2] = acc[r][n][3] = 0.0f;
        }
      multipliers_sync();
      if (a.ranks == 1) {
        // a whole block to y, a cut one to scratch: at most one that this run ends within and one that it starts within
        const bool whole = s_first == 0 && s == a.stages;
        float* part = a.part + ((int64_t(blockIdx.z) * gridDim.x + blockIdx.x) * 2 + (s_first == 0 ? 1 : 0)) * rows * kCols;
        T* y = static_cast<T*>(a.y) + int64_t(m0) * a.n + int64_t(block) * rows;
        const int there = min(rows, a.n - block * rows);
        for (int c = threadIdx.x; c < rows * tokens; c += 32 * kWarps) {
          const int m = c / rows, row = c - m * rows;
          float v = 0.0f;
          for (int w = 0; w < warps_k; ++w) v += red[(w * rows + row) * kCols + m];
          if (!whole) part[m * rows + row] = v;
          else if (row < there) y[int64_t(m) * a.n + row] = from_float<T>(v);
        }
      }
      asm volatile("fence.proxy.async;" ::: "memory");   // these writes come before the copies that go there next
      if (s == a.stages) s = 0, ++block;
      s_first = s;
    }
    __syncwarp();
    if (lane == 0) barrier_arrive(read + 8 * place);
    if (++place == kStages) place = 0, parity ^= 1;
  }
  if (a.ranks == 1) return;

  // a cluster's sums, through distributed shared memory, in the ranks' order
  float* sums = reinterpret_cast<float*>(smem);          // one place for all ranks; red's own, or where no copy is under way
  for (int c = threadIdx.x; c < rows * kCols; c += 32 * kWarps) {
    float v = red[c];
    for (int w = 1; w < warps_k; ++w) v += red[w * rows * kCols + c];
    sums[c] = v;
  }
  cg::this_cluster().sync();
  if (rank == 0) {
    const int64_t first_row = int64_t(blockIdx.x / a.ranks) * rows;
    T* y = static_cast<T*>(a.y) + int64_t(m0) * a.n + first_row;
    for (int c = threadIdx.x; c < rows * tokens; c += 32 * kWarps) {
      const int m = c / rows, row = c - m * rows;
      if (first_row + row >= a.n) continue;
      float v = sums[row * kCols + m];
      for (int r = 1; r < a.ranks; ++r) v += cg::this_cluster().map_shared_rank(sums, r)[row * kCols + m];
      y[int64_t(m) * a.n + row] = from_float<T>(v);
    }
  }
  cg::this_cluster().sync();                             // a CTA's sums stay until rank 0 has them
}

// Joins the pieces of the row blocks that runs were cut within: CTA c takes
// the block in which run c starts, unless an earlier run starts there too.
constexpr int kJoinThreads = 256;
template <class T, int NT>
__global__ void __launch_bounds__(kJoinThreads) w4_join_kernel(const __grid_constant__ W4Args a, int runs) {
  constexpr int kCols = 8 * NT;
  const int rows = a.warps_n * kRows, c = blockIdx.x + 1;
  const int64_t total = int64_t((a.n + rows - 1) / rows) * a.stages;
  auto start = [&](int run) { return total * run / runs; };
  const int64_t block = start(c) / a.stages;
  asm volatile("griddepcontrol.wait;" ::: "memory");    // in every CTA: this kernel's end has to mean the first one's
  if (start(c) % a.stages == 0 || (start(c - 1) > block * a.stages)) return;
  const int m0 = blockIdx.z * kCols, tokens = min(a.tokens - m0, kCols);
  const float* part = a.part + int64_t(blockIdx.z) * runs * 2 * rows * kCols;
  T* y = static_cast<T*>(a.y) + int64_t(m0) * a.n + block * rows;
  const int there = int(min(int64_t(rows), a.n - block * rows));
  const int i = blockIdx.y * kJoinThreads + threadIdx.x, m = i / rows, row = i - m * rows;
  if (m >= tokens || row >= there) return;
  float v = __ldcg(part + (int64_t(c - 1) * 2 + 1) * rows * kCols + i);
  int last = c;
  while (last < runs && start(last) < (block + 1) * a.stages) ++last;
#pragma unroll 4
  for (int k = c; k < last; ++k) v += __ldcg(part + int64_t(k) * 2 * rows * kCols + i);
  y[int64_t(m) * a.n + row] = from_float<T>(v);
}

// ---------------------------------------------------------------- launch
// How a product is shared out.
struct Plan {
  int nt, warps_n, ranks, stages;
  int64_t ctas;
  bool cut;                              // runs end within row blocks: scratch and the second kernel
};

template <int NT>
Plan plan_for(int tokens, int n, int k, int sms) {
  constexpr int kK = Tile<NT>::kK;
  Plan p{NT, 8, 1, 0, 0, false};
  const int held = tokens < 8 * NT ? tokens : 8 * NT;
  // Rows of a CTA (32 to 256): few, as long as the warps along k all have some
  // and the tokens' values, read again by every CTA, stay within 4 (8) KB of a
  // stage: a quarter (half) of the weights' bytes, and two CTAs to an SM.
  const int need = NT == 1 ? held : 4;
  while (p.warps_n > 1 && p.warps_n / 2 >= need && kWarps / (p.warps_n / 2) * kK < k + kK) p.warps_n /= 2;
  const int rows = kRows * p.warps_n, stage_k = kWarps / p.warps_n * kK;
  const int64_t blocks = (int64_t(n) + rows - 1) / rows;
  p.stages = (k + stage_k - 1) / stage_k;
  const int64_t slots = 2 * int64_t(sms);                // CTAs resident at once
  if (blocks * p.stages >= 4 * slots) {
    // enough for every CTA to have four stages or more: equal runs
    p.ctas = slots;
    p.cut = blocks * p.stages % slots != 0 || blocks * p.stages / slots % p.stages != 0;
  } else {
    // a cluster for each row block, as long as the SMs hold more and every CTA has a stage
    while (p.ranks < 8 && blocks * p.ranks * 2 <= slots && p.ranks * 2 <= p.stages) p.ranks *= 2;
    p.ctas = p.ranks > 1 ? blocks * p.ranks : blocks;
  }
  return p;
}
Plan plan_of(int tokens, int n, int k, int sms) { return tokens <= 8 ? plan_for<1>(tokens, n, k, sms) : plan_for<2>(tokens, n, k, sms); }
size_t plan_scratch(const Plan& p, int tokens) {
  return p.cut ? size_t((tokens + 8 * p.nt - 1) / (8 * p.nt)) * p.ctas * 2 * (kRows * p.warps_n) * (8 * p.nt) * sizeof(float) : 0;
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encoder() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool found = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess;
    return found ? reinterpret_cast<EncodeTiled>(p) : nullptr;
  }();
  return fn;
}
// A matrix of rows x columns and boxes of it; what lies beyond reads as zeros.
bool make_map(CUtensorMap* map, CUtensorMapDataType type, CUtensorMapSwizzle swizzle, const void* base, int64_t columns, int64_t rows,
              int64_t stride_bytes, int box_columns, int box_rows) {
  const EncodeTiled encode = encoder();
  if (!encode) return false;
  const cuuint64_t dims[2] = {cuuint64_t(columns), cuuint64_t(rows)}, strides[1] = {cuuint64_t(stride_bytes)};
  const cuuint32_t box[2] = {cuuint32_t(box_columns), cuuint32_t(box_rows)}, step[2] = {1, 1};
  return encode(map, type, 2, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class T, int NT, int GB, bool Boxes>
cudaError_t launch_shape(W4Args a, const Plan& p, cudaStream_t s) {
  using L = Tile<NT>;
  const int held = a.tokens < 8 * NT ? a.tokens : 8 * NT, warps_k = kWarps / p.warps_n;
  a.warps_n = p.warps_n;
  a.stages = p.stages;
  a.ranks = p.ranks;
  const unsigned per = unsigned(a.group / 32);
  a.group_shift = per & (per - 1) ? -1 : 31 - __builtin_clz(per);
  CUtensorMap map_w{}, map_x{};
  if (Boxes) {
    const int64_t x_stride = a.tokens == 1 ? (int64_t(a.k) + 7) / 8 * 8 : a.x_stride;   // one token has no stride
    if (!make_map(&map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, L::kPitch == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                  a.weight, (int64_t(a.k) + 1) / 2, a.n, a.weight_stride, L::kPitch, kRows * p.warps_n) ||
        !make_map(&map_x, CU_TENSOR_MAP_DATA_TYPE_UINT16, CU_TENSOR_MAP_SWIZZLE_NONE, a.x, a.k, a.tokens, x_stride * 2, L::kK, held))
      return cudaErrorInvalidValue;
  }
  const size_t bytes = size_t(L::kStages) * stage_size<NT>(held, warps_k) + 1024;
  const auto kernel = w4_kernel<T, NT, GB, Boxes>;
  static std::atomic<int> limits[kMaxDevices];           // of this kernel
  ensure_dynamic_smem(kernel, 1024, bytes, limits);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(p.ctas), 1, (a.tokens + 8 * NT - 1) / (8 * NT));
  cfg.blockDim = dim3(32 * kWarps + (Boxes ? kBoxThreads : kWordThreads));
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  cfg.attrs = attr;
  if (p.ranks > 1) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  }
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a, map_w, map_x);
  if (e != cudaSuccess || !p.cut) return e;
  cfg.gridDim.x = unsigned(p.ctas - 1);
  cfg.gridDim.y = unsigned((kRows * p.warps_n * held + kJoinThreads - 1) / kJoinThreads);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.dynamicSmemBytes = 0;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, w4_join_kernel<T, NT>, a, int(p.ctas));
}

template <class T, int NT, bool Boxes>
cudaError_t launch_group(const W4Args& a, const Plan& p, cudaStream_t s) {
  if (a.group == 64) return launch_shape<T, NT, 2, Boxes>(a, p, s);
  if (NT == 1 && a.group % 256 == 0) return launch_shape<T, NT, NT == 1 ? 8 : 4, Boxes>(a, p, s);
  if (a.group == 128 || (NT == 2 && a.group % 128 == 0)) return launch_shape<T, NT, 4, Boxes>(a, p, s);
  return launch_shape<T, NT, 1, Boxes>(a, p, s);
}

template <class T>
cudaError_t launch(const W4Args& a, const Plan& p, cudaStream_t s) {
  const bool aligned_rows = aligned(a.weight, 16) && a.weight_stride % 16 == 0 && aligned(a.x, 16) && (a.x_stride % 8 == 0 || a.tokens == 1);
  if (a.tokens <= 8) return aligned_rows ? launch_group<T, 1, true>(a, p, s) : launch_group<T, 1, false>(a, p, s);
  return aligned_rows ? launch_group<T, 2, true>(a, p, s) : launch_group<T, 2, false>(a, p, s);
}

}  // namespace
}  // namespace blk
}  // namespace pm

using namespace pm;
using namespace pm::blk;

extern "C" size_t pm_matvec_w4_scratch_bytes(int32_t tokens, int32_t n, int32_t k) {
  int sms = 0;
  if (tokens < 1 || n < 1 || k < 1 || tokens > (1 << 16) || n > (1 << 24) || k > (1 << 24) || sm_count(&sms) != PM_OK) return 0;
  return plan_scratch(plan_of(tokens, n, k, sms), tokens);
}

extern "C" int pm_matvec_w4_device(const pm_matvec_w4* j, void* scratch, size_t scratch_bytes, void* stream) {
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
  const Plan plan = plan_of(j->tokens, j->n, j->k, sms);
  const size_t need = plan_scratch(plan, j->tokens);
  if (need && (!scratch || !aligned(scratch, 256) || scratch_bytes < need))
    return fail(PM_E_INVALID, "%s: needs %zu bytes of scratch, 256-byte aligned", who, need);
  W4Args a{j->tokens, j->n, j->k, j->group, int((int64_t(j->k) + j->group - 1) / j->group), j->scales_dtype == PM_DT_F32,
           j->x_stride, j->weight_stride, j->x, j->weight, j->scales, j->zeros, j->y, 0, aligned(j->scales, 16) && aligned(j->zeros, 8), 0, 0, 0, static_cast<float*>(scratch)};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = j->dtype == PM_DT_BF16 ? launch<bf16>(a, plan, s) : launch<fp16>(a, plan, s);
  return e == cudaSuccess ? PM_OK : cuda_fail(e, "pm_matvec_w4_device launch");
}
