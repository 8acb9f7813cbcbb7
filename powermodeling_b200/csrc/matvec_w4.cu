// The product of a few tokens with a matrix of 4-bit weights with a scale
// (and a zero point) per group:
//   y[m, n] = sum_g s[n, g] sum_{k in g} x[m, k] (q[n, k] - z[n, g]).
//
// The weights are read once; for one token their bytes bound it, beside a few
// tokens the instructions that unpack and scale them.
//  * A warp owns 32 rows of weights and 256 (128) values of k at a time, a
//    tile of 4 (2) KB.  8 such warps stand side by side along n or along k, so
//    a stage is 32 (16) KB whatever the matrix's shape, and with two CTAs an
//    SM enough bytes are in flight.  A ninth warp fills the stages by tensor
//    copies, a box to a lane, the tokens' values, scales and zero points
//    beside the weights, so the others do nothing but unpack and multiply.
//    Rows that start at any byte: two warps copy the 16-byte pieces that hold
//    them, and the readers shift two words into one.
//  * Each token pair serves two tiles of 16 rows in registers.
//  * A nibble is masked into a 16-bit float's mantissa, exactly.  The matrix
//    instruction multiplies 16 rows by 8 tokens with exact products and 32-bit
//    sums; the scale enters once a group, in 32 bits.  So nothing is rounded
//    to 16 bits before the output.
//  * k is summed in an order that suits the nibbles: a lane's word holds k =
//    0..7 of its eight, and the pairs (0,4), (1,5), (2,6), (3,7) are the
//    instruction's neighbours, for the weights and for the tokens alike.
//  * 8 tokens (16 in two halves) are the instruction's columns: mma.sync, which
//    takes the unpacked weights from the registers that they are in.  tcgen05
//    would have them written to tensor memory first, and its sums read back
//    for each group; that way is not built and not measured.
//  * Few stages: the CTAs of a cluster share k and add their sums through
//    distributed shared memory, in rank order.  Many: the line of all row
//    blocks' stages is cut into equal runs, and a second kernel adds the
//    pieces of the cut blocks in order.  So results do not vary.
// Measured (a copy runs at 6.55 TB/s): one token x 28672 x 8192 in groups of
// 128 32.4 us = 3.7 TB/s, 8 tokens 33 us; 16 tokens x 8192 x 28672 in groups
// of 32 with zero points 50.2 us = 2.8 TB/s; 1024 x 1024 for one token 4.2 us.
// The copies alone take 27 us of the first, in boxes 128 bytes wide; at the
// copy's rate its bytes would take 18.5.  For 16 tokens the issue slots are
// 60 % busy on the half of the pipes that unpacking needs, with 16 warps an SM;
// at 96 registers a thread these kernels spill up to 28 bytes.
#include <cooperative_groups.h>
#include <cuda.h>

#include <algorithm>
#include <cmath>

#include "blocks.cuh"

namespace cg = cooperative_groups;

namespace pm {
namespace blk {
namespace {

constexpr int kWarps = 8, kRows = 32;                    // warps that multiply; rows of a warp's tile
constexpr int kMaxRanks = 8;                             // CTAs of a cluster
constexpr int kLine = 8;                                 // stages of a CTA from which on runs are equal
constexpr int kLinePasses = 8;                           // passes over the tokens up to which they are: scratch is 5 MB a pass
constexpr uint64_t kWaitNs = 2ull * 1000000000ull;       // bound on any single wait, unless the caller sets another
std::atomic<uint64_t> g_wait_ns{kWaitNs};

// Rows lie in shared memory 256 k (128 bytes) wide, as a copy brings them: 64
// bytes a row and copy took 42 us where 128 took 27 (8192 x 28672).  Up to 8
// tokens a warp has all of its rows' 256 k, up to 16 half of them, as the
// tokens' values take the room.
constexpr int kBoxK = 256, kPitch = kBoxK / 2, kPieces = kPitch / 16;           // a row, in 16-byte pieces
constexpr int kRoom = 111 * 1024;                        // of a CTA's stages, two CTAs to an SM
template <int NT>
struct Tile {
  static constexpr int kK = NT == 1 ? 256 : 128, kShare = kBoxK / kK, kStages = NT == 1 ? 3 : 4;   // kShare: warps of a row
  static constexpr int kStageBytes = kWarps * kRows * kK / 2;
};
// Rows that start at any byte: the 16-byte pieces that hold them, as they lie in memory, nine for eight.
constexpr int kLoosePitch = kPitch + 16, kLoosePieces = kPieces + 1;
// Pieces lie in an order of the row's own, so that 8 rows x 4 words meet all 32 banks.
__device__ __forceinline__ int turn(int row) { return row & 7; }

// A stage: the weights (whole KBs, as their order wants), the tokens' values, and scales and zero points where copies
// bring them: `scale_box` and `zero_box` bytes a row.
struct Stage {
  int x, scales, zeros, bytes;
};
template <int NT>
__host__ __device__ inline Stage stage_of(int pitch, int tokens, int warps_n, int scale_box, int zero_box) {
  const int boxes = kWarps / warps_n / Tile<NT>::kShare, rows = kRows * warps_n;
  Stage s;
  s.x = Tile<NT>::kStageBytes / kPitch * pitch;
  s.scales = s.x + boxes * tokens * kBoxK * 2;
  s.zeros = s.scales + rows * scale_box;
  s.bytes = (s.zeros + rows * zero_box + 1023) / 1024 * 1024;
  return s;
}

struct W4Args {
  int tokens, n, k, group, groups, scales32;
  int64_t x_stride, weight_stride;
  const void* x;
  const uint8_t* weight;
  const void* scales;
  const uint8_t* zeros;
  void* y;
  uint64_t wait_ns;                                      // bound on a wait for a stage
  int warps_n;                                           // warps along n; the others along k
  int x_pieces;                                          // tokens start on 16-byte boundaries
  int scale_box, zero_box;                               // bytes of a row's scales and zero points in a stage, 0: not copied
  int group_shift;                                       // log2 of the 32-k blocks of a group, -1: no power of two
  int places;                                            // stages in shared memory
  int stages;                                            // stages of a row block: its k over the stage's
  int ranks;                                             // CTAs of a cluster, which share each row block's stages
  int runs, run_rest;                                    // ranks == 1: the line is cut into so many runs;
  int64_t run;                                           // total / runs and what is left
  float* part;                                           // ranks == 1: sums of cut row blocks, [2 * CTAs][rows][8 NT]
};

// The pairs (0,4), (1,5), (2,6), (3,7) of a word's nibbles, less the zero
// point and over kScale, as exact 16-bit floats.  Integer instructions are
// what the kernel has least of, so two nibble positions of a half are taken
// where they lie and one shift brings the other two: five and four fused
// multiply-adds a word.
// bf16: the bits of an integer below 256 are that integer times 2^-133 (the
// subnormals and the first binade are one even grid), so a nibble at bit 0 or
// bit 4 is n 2^-133 or n 2^-129, and n - z over 64 is one fma away.
// fp16: likewise n 2^-24 and n 2^-20, subnormal, and n - z over 512 is one fma away.
template <class T> struct Nibbles;
template <> struct Nibbles<bf16> {
  static constexpr float kScale = 64.0f;
  // of byte `at` of a word
  static __device__ __forceinline__ uint32_t zero(uint32_t word, int at) {
    const uint32_t bits = __byte_perm(word, 0u, 0x4040u + 0x0101u * at), high = 0xff00ff00u;   // -2^127
    const __nv_bfloat162 v = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&bits), *reinterpret_cast<const __nv_bfloat162*>(&high));
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
  static constexpr float kScale = 512.0f;
  static __device__ __forceinline__ uint32_t zero(uint32_t word, int at) {
    const uint32_t bits = __byte_perm(word, 0u, 0x4040u + 0x0101u * at), high = 0xf800f800u;   // -2^15
    const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&bits), *reinterpret_cast<const __half2*>(&high));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ void unpack(uint32_t w, uint32_t zero, uint32_t (&p)[4]) {
    const uint32_t low = 0x78007800u, high = 0x68006800u;                      // 2^15, 2^11
    const __half2 z = *reinterpret_cast<const __half2*>(&zero);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t u = i ? w >> 8 : w, a = u & 0x000f000fu, b = u & 0x00f000f0u;
      const __half2 x = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&low), z);
      const __half2 y = __hfma2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&high), z);
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

// Keeps what is done with a loaded value from moving up to the load, which it would wait for there.
__device__ __forceinline__ uint32_t late(uint32_t v) {
  asm volatile("" : "+r"(v));
  return v;
}
// A half of a word as a float.
template <class T>
__device__ __forceinline__ float half_of(uint32_t word, int high) {
  const uint16_t bits = uint16_t(high ? word >> 16 : word);
  return to_float(*reinterpret_cast<const T*>(&bits));
}
// 1 to 16 bytes of shared memory, a power of two and so aligned.
template <int Bytes>
__device__ __forceinline__ void load_words(uint32_t* to, const uint8_t* from) {
  if constexpr (Bytes == 16) {
    const uint4 v = *reinterpret_cast<const uint4*>(from);
    to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
  } else if constexpr (Bytes == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(from);
    to[0] = v.x, to[1] = v.y;
  } else if constexpr (Bytes == 4) {
    *to = *reinterpret_cast<const uint32_t*>(from);
  } else if constexpr (Bytes == 2) {
    *to = *reinterpret_cast<const uint16_t*>(from);
  } else {
    *to = *from;
  }
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
// Looks once.  The waiting form sleeps for up to milliseconds on its own account: limits that short are kept without it.
__device__ __forceinline__ bool barrier_try(uint32_t bar, uint32_t parity, uint64_t limit) {
  uint32_t done;
  if (limit < 20000000)
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0;
}
__device__ __forceinline__ uint64_t nanoseconds() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// False when the wait runs out, or has run out elsewhere in the CTA: `failed` says so to all of it.  A CTA that was not
// running in the meantime looks once more before it gives up.
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity, uint64_t limit, volatile int* failed) {
  if (barrier_try(bar, parity, limit)) return true;
  const uint64_t deadline = nanoseconds() + limit;
  while (!barrier_try(bar, parity, limit)) {
    if (*failed) return false;
    if (nanoseconds() > deadline) {
      if (barrier_try(bar, parity, limit)) return true;
      *failed = 1;
      return false;
    }
  }
  return true;
}
// The same without a way to give up early, for copies that have to have landed.
__device__ __forceinline__ void barrier_drain(uint32_t bar, uint32_t parity) {
  if (barrier_try(bar, parity, kWaitNs)) return;
  const uint64_t deadline = nanoseconds() + kWaitNs;
  while (!barrier_try(bar, parity, kWaitNs) && nanoseconds() < deadline) {}
}
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void multipliers_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// Where run `run` starts: total * run / runs without a 64-bit division.
__device__ __forceinline__ int64_t run_start(const W4Args& a, int run) { return a.run * run + uint32_t(a.run_rest * run) / uint32_t(a.runs); }

// GB: blocks of 32 k per scale within a tile (1 to all of them); 1 also serves
// the group sizes that the tile's k is no multiple of, or no divisor.
// Boxes: rows of weights and tokens start on 16-byte boundaries, and a lane
// copies a box; else the lanes copy 16-byte pieces of the weights as they lie,
// which the readers shift into place, and the tokens' values by words.
// Side: scales and zero points come with the stage too.
constexpr int kCopyThreads = 32, kLooseThreads = 64;       // copying boxes, pieces
template <class T, int NT, int GB, bool Boxes, bool Side>
__global__ void __launch_bounds__(32 * kWarps + (Boxes ? kCopyThreads : kLooseThreads), 2)
w4_kernel(const __grid_constant__ W4Args a, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
          const __grid_constant__ CUtensorMap map_s, const __grid_constant__ CUtensorMap map_z) {
  extern __shared__ uint8_t smem_raw[];
  using L = Tile<NT>;
  constexpr int kStages = L::kStages, kGroups = L::kK / 32 / GB, kCols = 8 * NT;
  __shared__ __align__(8) uint64_t bars[2 * kStages];    // a stage is full; it is read
  // A wait ran out.  Who gave up goes on without waiting: from then on nothing that this CTA sums counts.  Sums are
  // looked at only after a barrier that those who gave up come to as well.
  __shared__ int failed;
  uint8_t* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int warps_k = kWarps / a.warps_n, wn = warp % a.warps_n, wk = warp / a.warps_n;
  const int stage_k = warps_k * L::kK, boxes = warps_k / L::kShare, rows = a.warps_n * kRows;
  const int m0 = blockIdx.z * kCols, held = min(a.tokens, kCols), tokens = min(a.tokens - m0, kCols);
  constexpr int kRowBytes = Boxes ? kPitch : kLoosePitch, kCopies = Boxes ? kCopyThreads : kLooseThreads;
  const Stage at = stage_of<NT>(kRowBytes, held, a.warps_n, a.scale_box, a.zero_box);
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
    first = run_start(a, blockIdx.x);
    count = int(run_start(a, blockIdx.x + 1) - first);
  }
  int block = int(first >> 32 ? first / a.stages : int64_t(uint32_t(first) / uint32_t(a.stages))), s = int(first - int64_t(block) * a.stages);
  const uint32_t ring = smem_addr(smem), full = smem_addr(bars), read = full + 8 * kStages;
  if (threadIdx.x == 0) {
    failed = 0;
    for (int i = 0; i < a.places; ++i) {
      barrier_init(full + 8 * i, Boxes ? 1 : 2 * kCopies);
      barrier_init(read + 8 * i, kWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  // the first scale and zero point of a stage: their boxes start on 16-byte boundaries
  auto first_scale = [&](int at_s) { return (at_s * stage_k / 32 >> a.group_shift) & ~7; };
  auto first_zero = [&](int at_s) { return (at_s * stage_k / 32 >> a.group_shift) & ~15; };

  if (warp >= kWarps) {
    // ------------------------------------------------ the copies
    const int me = threadIdx.x - 32 * kWarps;
    bool ok = true;
    int place = 0, filled = 0;
    uint32_t parity = 1;
    for (int i = 0; i < count && ok; ++i) {
      const uint32_t stage = ring + place * at.bytes, bar = full + 8 * place;
      const int k0 = s * stage_k;
      // A place is filled again only if all eight readers waited for what it held: one that gave up said so before it
      // arrived.  (Copies to a place whose last ones are still under way would arrive twice in one phase of its barrier.)
      if (i >= a.places) ok = barrier_wait(read + 8 * place, parity, a.wait_ns, &failed) && !*static_cast<volatile int*>(&failed);
      if constexpr (Boxes) {
        // a lane for each box
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (me == 0) barrier_expect(bar, L::kStageBytes + boxes * held * kBoxK * 2 + rows * (a.scale_box + a.zero_box));
        __syncwarp();
        const int w = me & 7;
        if (me < 16) {
          if (w < boxes) {
            if (me < 8) copy_box(stage + w * rows * kPitch, &map_w, (k0 + w * kBoxK) / 2, block * rows, bar);
            else copy_box(stage + at.x + w * held * kBoxK * 2, &map_x, k0 + w * kBoxK, m0, bar);
          }
        } else if (Side && w == 0) {
          if (me == 16) copy_box(stage + at.scales, &map_s, first_scale(s), block * rows, bar);
          else if (me == 24 && a.zero_box) copy_box(stage + at.zeros, &map_z, first_zero(s), block * rows, bar);
        }
      } else {
        if (!ok) break;
        // Seven rows at a time, a lane for each piece.  What lies beyond the matrix is left as it is: its tokens' values
        // are zero, or nothing reads its sums.
        constexpr int kAtOnce = kCopies / kLoosePieces;
        const int sub = me / kLoosePieces, piece = me - sub * kLoosePieces, lines = min(rows, a.n - block * rows);
        for (int w = 0; w < boxes && sub < kAtOnce; ++w) {
          const int64_t at_byte = (k0 >> 1) + w * kPitch, left = ((int64_t(a.k) + 1) >> 1) - at_byte;
          const uint8_t* from = a.weight + int64_t(block * rows + sub) * a.weight_stride + at_byte;
          uint32_t dst = stage + (w * rows + sub) * kLoosePitch + piece * 16;
#pragma unroll 4
          for (int line = sub; line < lines; line += kAtOnce) {
            const int o = 16 * piece - int(reinterpret_cast<uintptr_t>(from) & 15);   // from the row's first byte here
            if (o < kPitch && o < left) copy16(dst, from + o, int(left - o < 16 ? left - o : 16));
            from += kAtOnce * a.weight_stride;
            dst += kAtOnce * kLoosePitch;
          }
        }
        // the tokens' values, zeros beyond k; by words where they lie anywhere
        for (int p = me; p < boxes * tokens * (kBoxK / 8); p += kCopies) {
          const int piece = p % (kBoxK / 8), m = p / (kBoxK / 8) % tokens, w = p / (kBoxK / 8) / tokens;
          const int k = k0 + w * kBoxK + piece * 8, left = min(max(a.k - k, 0), 8);
          const T* src = static_cast<const T*>(a.x) + (left ? int64_t(m0 + m) * a.x_stride + k : 0);
          const uint32_t to = stage + at.x + ((w * held + m) * (kBoxK / 8) + piece) * 16;
          if (a.x_pieces) copy16(to, src, 2 * left);
          else sts128(to, keep(load_any(reinterpret_cast<const uint8_t*>(src), 2 * left), left));
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" :: "r"(bar) : "memory");
        barrier_arrive(bar);
      }
      ++filled;
      if (++s == a.stages) s = 0, ++block;
      if (++place == a.places) place = 0, parity ^= 1;
    }
    // copies under way land before the CTA goes, whether its readers waited for them or not
    if (!Boxes) asm volatile("cp.async.wait_all;" ::: "memory");
    if (Boxes)
      for (int i = max(filled - a.places, 0); i < filled; ++i) barrier_drain(full + 8 * (i % a.places), i / a.places & 1);
    __syncwarp();
    if (a.ranks > 1) {
      cg::this_cluster().sync();
      cg::this_cluster().sync();
    }
    return;
  }

  // -------------------------------------------------- the products
  // Scales and zero points that no copy brings: row `lane`'s, one by one, one
  // stage ahead of their use and as they are in memory, as converting them
  // here would wait for them here.
  constexpr int kScaleWords = (kGroups + 1) / 2, kZeroWords = (kGroups + 3) / 4;
  uint32_t scale_next[Side ? 1 : kGroups], zero_next[Side ? 1 : kGroups];
  auto fetch_scales = [&](int at_block, int at_s) {
    const int block0 = (at_s * stage_k + wk * L::kK) / 32, per = a.group / 32;
    const int64_t scale_row = int64_t(min(at_block * rows + wn * kRows + lane, a.n - 1)) * a.groups;
#pragma unroll
    for (int e = 0; e < (Side ? 0 : kGroups); ++e) {
      const int at_k = block0 + e * GB, group = a.group_shift >= 0 ? at_k >> a.group_shift : at_k / per;
      const int64_t i = scale_row + min(group, a.groups - 1);
      scale_next[e] = a.scales32 ? __ldg(static_cast<const uint32_t*>(a.scales) + i) : __ldg(static_cast<const uint16_t*>(a.scales) + i);
      zero_next[e] = a.zeros ? __ldg(a.zeros + i) : 8u;
    }
  };

  float acc[2][NT][4] = {};
  int s_first = s, place = 0;
  uint32_t parity = 0;
  float* red = nullptr;                                  // [wk][row][token], in the place of a row block's last stage
  // this lane's words of its tile (rows g + 8 r), and its tokens' values; columns beyond the tokens repeat the last one:
  // nothing reads their sums
  const int box = wk / L::kShare, half = wk % L::kShare;
  const int w_lane = Boxes ? (box * rows + wn * kRows + g) * kPitch + ((half * (L::kK / 32)) ^ turn(g)) * 16 + t * 4
                           : (box * rows + wn * kRows + g) * kLoosePitch + half * (L::kK / 2) + t * 4;
  int x_lane[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) x_lane[n] = at.x + (box * held + min(n * 8 + g, tokens - 1)) * (kBoxK * 2) + half * (L::kK * 2) + t * 16;
  if (!Side && count) fetch_scales(block, s);
  for (int left = count; left > 0; --left) {
    uint32_t scale[Side ? 4 : 1][Side ? kScaleWords : kGroups], zero[Side ? 4 : 1][Side ? kZeroWords : kGroups];
    if constexpr (!Side) {
      const int blocks_left = (a.k + 31) / 32 - (s * stage_k + wk * L::kK) / 32;         // of 32 k, from the tile's start on
#pragma unroll
      for (int e = 0; e < kGroups; ++e) {
        // beyond the row zero, as the sums there are: an infinite scale is not to meet them
        scale[0][e] = e * GB < blocks_left ? late(scale_next[e]) : 0u;
        zero[0][e] = late(zero_next[e]) & 15u;
      }
    }
    const bool last = s + 1 == a.stages || left == 1;    // of this CTA in this row block
    if (left == 1 && a.ranks == 1) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the join's CTAs come and wait
    if (!Side && left > 1) fetch_scales(s + 1 == a.stages ? block + 1 : block, s + 1 == a.stages ? 0 : s + 1);
    barrier_wait(full + 8 * place, parity, a.wait_ns, &failed);
    const int stage = place * at.bytes;
    if constexpr (Side) {
      const int group = (s * stage_k + wk * L::kK) / 32 >> a.group_shift;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = wn * kRows + g + 8 * r;
        load_words<2 * kGroups>(scale[r], smem + stage + at.scales + row * a.scale_box + (group - first_scale(s)) * 2);
        if (a.zero_box) {
          load_words<kGroups>(zero[r], smem + stage + at.zeros + row * a.zero_box + (group - first_zero(s)));
#pragma unroll
          for (int e = 0; e < kZeroWords; ++e) zero[r][e] &= 0x0f0f0f0fu;
        } else {
#pragma unroll
          for (int e = 0; e < kZeroWords; ++e) zero[r][e] = 0x08080808u;
        }
      }
    }
    const int w_at = stage + w_lane;
    int skew[4];                                         // bytes of a row's start beyond a boundary; the same all along it
#pragma unroll
    for (int r = 0; r < 4; ++r)
      skew[r] = Boxes ? 0 : int(uint32_t(reinterpret_cast<uintptr_t>(a.weight)) + uint32_t(min(block * rows + wn * kRows + g + 8 * r, a.n - 1)) * uint32_t(a.weight_stride)) & 15;
    auto word_at = [&](int b, int r) {
      if constexpr (Boxes) return *reinterpret_cast<const uint32_t*>(smem + (w_at ^ (b * 16)) + 8 * r * kPitch);
      const uint32_t* at = reinterpret_cast<const uint32_t*>(smem + w_at + 8 * r * kLoosePitch + b * 16 + (skew[r] & 12));
      return __funnelshift_r(at[0], at[1], 8 * (skew[r] & 3));
    };
#pragma unroll
    for (int e = 0; e < kGroups; ++e) {
      float part[2][NT][4];
      uint32_t z[4];
      if constexpr (Side) {
#pragma unroll
        for (int r = 0; r < 4; ++r) z[r] = Nibbles<T>::zero(zero[r][e / 4], e & 3);
      } else {
        const uint32_t own = Nibbles<T>::zero(zero[0][e], 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) z[r] = __shfl_sync(0xffffffffu, own, g + 8 * r);
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
          Nibbles<T>::unpack(word_at(b, 2 * r), z[2 * r], p0);
          Nibbles<T>::unpack(word_at(b, 2 * r + 1), z[2 * r + 1], p1);
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
        float s0, s1;
        if constexpr (Side) {
          s0 = Nibbles<T>::kScale * half_of<T>(scale[2 * r][e / 2], e & 1);
          s1 = Nibbles<T>::kScale * half_of<T>(scale[2 * r + 1][e / 2], e & 1);
        } else {
          const float own = Nibbles<T>::kScale * (a.scales32 ? __uint_as_float(scale[0][e]) : half_of<T>(scale[0][e], 0));
          s0 = __shfl_sync(0xffffffffu, own, g + 16 * r), s1 = __shfl_sync(0xffffffffu, own, g + 16 * r + 8);
        }
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
          float* to = red + ((wk * rows + wn * kRows + 16 * r + g) * kCols + n * 8 + 2 * t);
          to[0] = acc[r][n][0];
          to[1] = acc[r][n][1];
          to[8 * kCols] = acc[r][n][2];
          to[8 * kCols + 1] = acc[r][n][3];
          acc[r][n][0] = acc[r][n][1] = acc[r][n][2] = acc[r][n][3] = 0.0f;
        }
      multipliers_sync();
      if (a.ranks == 1) {
        const bool lost = *static_cast<volatile int*>(&failed);
        // a whole block to y, a cut one to scratch: at most one that this run ends within and one that it starts within
        const bool whole = s_first == 0 && s == a.stages;
        float* part = a.part + ((int64_t(blockIdx.z) * gridDim.x + blockIdx.x) * 2 + (s_first == 0 ? 1 : 0)) * rows * kCols;
        T* y = static_cast<T*>(a.y) + int64_t(m0) * a.n + int64_t(block) * rows;
        const int there = min(rows, a.n - block * rows);
        for (int c = threadIdx.x; c < rows * (kCols / 4); c += 32 * kWarps) {
          const int q = c / rows, row = c - q * rows;    // four tokens of a row: 2 lanes to a bank where one would be 8 or 16
          if (4 * q >= tokens) break;
          float4 v = *reinterpret_cast<const float4*>(red + row * kCols + 4 * q);
          for (int w = 1; w < warps_k; ++w) {
            const float4 u = *reinterpret_cast<const float4*>(red + (w * rows + row) * kCols + 4 * q);
            v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
          }
          const float value[4] = {lost ? NAN : v.x, lost ? NAN : v.y, lost ? NAN : v.z, lost ? NAN : v.w};
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            if (4 * q + m >= tokens) continue;
            if (!whole) part[(4 * q + m) * rows + row] = value[m];
            else if (row < there) y[int64_t(4 * q + m) * a.n + row] = from_float<T>(value[m]);
          }
        }
      }
      asm volatile("fence.proxy.async;" ::: "memory");   // these writes come before the copies that go there next
      if (s == a.stages) s = 0, ++block;
      s_first = s;
    }
    __syncwarp();
    if (lane == 0) barrier_arrive(read + 8 * place);
    if (++place == a.places) place = 0, parity ^= 1;
  }
  if (a.ranks == 1) return;

  // a cluster's sums, through distributed shared memory, in the ranks' order; each rank has a share of the rows, and
  // all ranks' values are under way at once
  float* sums = reinterpret_cast<float*>(smem);          // one place for all ranks; red's own, or where no copy is under way
  for (int c = threadIdx.x; c < rows * kCols; c += 32 * kWarps) {
    float v = red[c];
    for (int w = 1; w < warps_k; ++w) v += red[w * rows * kCols + c];
    sums[c] = v;
  }
  cg::this_cluster().sync();
  bool lost = false;
  for (int r = 0; r < a.ranks; ++r) lost |= *static_cast<volatile int*>(cg::this_cluster().map_shared_rank(&failed, r)) != 0;
  const int64_t first_row = int64_t(blockIdx.x / a.ranks) * rows;
  T* y = static_cast<T*>(a.y) + int64_t(m0) * a.n + first_row;
  for (int c = rank * 32 * kWarps + threadIdx.x; c < rows * (kCols / 4); c += a.ranks * 32 * kWarps) {
    const int q = c / rows, row = c - q * rows;
    if (first_row + row >= a.n || 4 * q >= tokens) continue;
    float4 v[kMaxRanks];
#pragma unroll
    for (int r = 0; r < kMaxRanks; ++r)
      if (r < a.ranks) v[r] = *reinterpret_cast<const float4*>(cg::this_cluster().map_shared_rank(sums, r) + row * kCols + 4 * q);
#pragma unroll
    for (int r = 1; r < kMaxRanks; ++r)
      if (r < a.ranks) v[0].x += v[r].x, v[0].y += v[r].y, v[0].z += v[r].z, v[0].w += v[r].w;
    const float value[4] = {lost ? NAN : v[0].x, lost ? NAN : v[0].y, lost ? NAN : v[0].z, lost ? NAN : v[0].w};
#pragma unroll
    for (int m = 0; m < 4; ++m)
      if (4 * q + m < tokens) y[int64_t(4 * q + m) * a.n + row] = from_float<T>(value[m]);
  }
  cg::this_cluster().sync();                             // a CTA's sums stay until every rank has them
}

// Joins the pieces of the row blocks that runs were cut within: CTA c takes
// the block in which run c starts, unless an earlier run starts there too.  A
// thread adds four rows of a token; what it adds is known before the wait.
constexpr int kJoinThreads = 256;
template <class T, int NT>
__global__ void __launch_bounds__(kJoinThreads) w4_join_kernel(const __grid_constant__ W4Args a) {
  constexpr int kCols = 8 * NT;
  const int rows = a.warps_n * kRows, c = blockIdx.x + 1;
  const int64_t from = run_start(a, c);
  const int64_t block = from >> 32 ? from / a.stages : int64_t(uint32_t(from) / uint32_t(a.stages));
  const int64_t begin = block * a.stages;
  const bool first = from != begin && run_start(a, c - 1) <= begin;
  int last = c;                                          // the runs that start in the block end before this one
  while (first && last < a.runs && run_start(a, last) < begin + a.stages) ++last;
  asm volatile("griddepcontrol.wait;" ::: "memory");    // in every CTA: this kernel's end has to mean the first one's
  if (!first) return;
  const int m0 = blockIdx.z * kCols, tokens = min(a.tokens - m0, kCols);
  const int i = 4 * (blockIdx.y * kJoinThreads + threadIdx.x), m = i / rows, row = i - m * rows;
  const int there = int(min(int64_t(rows), a.n - block * rows));
  if (m >= tokens || row >= there) return;
  const float* part = a.part + int64_t(blockIdx.z) * a.runs * 2 * rows * kCols + i;
  float4 v = __ldcg(reinterpret_cast<const float4*>(part + (int64_t(c - 1) * 2 + 1) * rows * kCols));
#pragma unroll 4
  for (int k = c; k < last; ++k) {
    const float4 u = __ldcg(reinterpret_cast<const float4*>(part + int64_t(k) * 2 * rows * kCols));
    v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
  }
  T* y = static_cast<T*>(a.y) + int64_t(m0 + m) * a.n + block * rows + row;
  const float value[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (row + r < there) y[r] = from_float<T>(value[r]);
}

// ---------------------------------------------------------------- launch
// How a product is shared out.
struct Plan {
  int nt, warps_n, ranks, stages;
  int64_t ctas;
  bool cut;                              // runs end within row blocks: scratch and the second kernel
};

// Rules, each with what it gained (us): from kLine stages a CTA on, equal runs
// (one token x 28672 x 8192, 12 stages: 33.2, with row blocks as they come
// 37.4; below it the second kernel costs more: 16 tokens x 14336 x 4096 28.8
// by runs, 17.5 by clusters); row blocks of twice the rows where there are more
// than CTAs at once but less than two rounds (one token x 14336 x 4096 14.0,
// 11.4), of half where clusters of 8 leave half of the SMs idle (8 tokens x
// 4096 x 14336 19.6, 13.9).
template <int NT>
Plan plan_for(int tokens, int n, int k, int sms) {
  constexpr int kK = Tile<NT>::kK;
  Plan p{NT, kWarps / Tile<NT>::kShare, 1, 0, 0, false};
  const int held = tokens < 8 * NT ? tokens : 8 * NT;
  // Rows of a CTA (32 to 256): few, as long as the warps along k all have some
  // and the tokens' values, read again by every CTA, stay within 4 (8) KB of a
  // stage: a quarter (half) of the weights' bytes, and two CTAs to an SM.
  const int need = NT == 1 ? held : 4;
  while (p.warps_n > 1 && p.warps_n / 2 >= need && kWarps / (p.warps_n / 2) * kK < k + kK) p.warps_n /= 2;
  const int64_t slots = 2 * int64_t(sms);                // CTAs resident at once
  int64_t blocks;
  auto share = [&](int warps_n) {
    p.warps_n = warps_n;
    blocks = (int64_t(n) + kRows * warps_n - 1) / (kRows * warps_n);
    p.stages = (k + kWarps / warps_n * kK - 1) / (kWarps / warps_n * kK);
  };
  share(p.warps_n);
  const int64_t passes = (tokens + 8 * NT - 1) / (8 * NT);
  if (blocks * p.stages >= kLine * slots && passes <= kLinePasses) {
    // enough for every CTA to have kLine stages or more: equal runs
    p.ctas = slots;
    p.cut = blocks * p.stages % slots != 0 || blocks * p.stages / slots % p.stages != 0;
  } else {
    if (blocks > slots && p.warps_n < kWarps / Tile<NT>::kShare) share(p.warps_n * 2);
    else if (p.warps_n > 1 && blocks * kMaxRanks * 2 <= slots && p.stages > kMaxRanks) share(p.warps_n / 2);
    // a cluster for each row block, as long as the SMs hold more and every CTA has a stage
    while (p.ranks < kMaxRanks && blocks * p.ranks * 2 <= slots && p.ranks * 2 <= p.stages) p.ranks *= 2;
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
  auto made = [&] {
    return encode(map, type, 2, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  if (made()) return true;
  // a thread that has called nothing of the runtime yet has no context, and this driver call wants one
  int device = 0;
  return cudaGetDevice(&device) == cudaSuccess && cudaSetDevice(device) == cudaSuccess && made();
}

template <class T, int NT, int GB, bool Boxes, bool Side>
cudaError_t launch_shape(W4Args a, const Plan& p, cudaStream_t s) {
  using L = Tile<NT>;
  const int held = a.tokens < 8 * NT ? a.tokens : 8 * NT, warps_k = kWarps / p.warps_n;
  a.warps_n = p.warps_n;
  a.stages = p.stages;
  a.ranks = p.ranks;
  a.runs = int(p.ctas);
  const int64_t total = (int64_t(a.n) + kRows * p.warps_n - 1) / (kRows * p.warps_n) * p.stages;
  a.run = total / a.runs;
  a.run_rest = int(total % a.runs);
  const unsigned per = unsigned(a.group / 32);
  a.group_shift = per & (per - 1) ? -1 : 31 - __builtin_clz(per);
  CUtensorMap map_w{}, map_x{}, map_s{}, map_z{};
  if (Boxes) {
    const int64_t x_stride = a.tokens == 1 ? (int64_t(a.k) + 7) / 8 * 8 : a.x_stride;   // one token has no stride
    if (!make_map(&map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_128B, a.weight, (int64_t(a.k) + 1) / 2, a.n,
                  a.weight_stride, kPitch, kRows * p.warps_n) ||
        !make_map(&map_x, CU_TENSOR_MAP_DATA_TYPE_UINT16, CU_TENSOR_MAP_SWIZZLE_NONE, a.x, a.k, a.tokens, x_stride * 2, kBoxK, held))
      return cudaErrorInvalidValue;
  }
  if (Side) {
    const int groups = std::max(warps_k * L::kK / a.group, 1);                           // of a stage; a power of two
    a.scale_box = std::max(2 * groups, 16);
    a.zero_box = a.zeros ? std::max(groups, 16) : 0;
    if (!make_map(&map_s, CU_TENSOR_MAP_DATA_TYPE_UINT16, CU_TENSOR_MAP_SWIZZLE_NONE, a.scales, a.groups, a.n, int64_t(a.groups) * 2,
                  a.scale_box / 2, kRows * p.warps_n) ||
        (a.zeros && !make_map(&map_z, CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_NONE, a.zeros, a.groups, a.n, a.groups,
                              a.zero_box, kRows * p.warps_n)))
      return cudaErrorInvalidValue;
  }
  const int stage = stage_of<NT>(Boxes ? kPitch : kLoosePitch, held, p.warps_n, a.scale_box, a.zero_box).bytes;
  a.places = std::min(L::kStages, kRoom / stage);
  const size_t bytes = size_t(a.places) * stage + 1024;
  const auto kernel = w4_kernel<T, NT, GB, Boxes, Side>;
  static std::atomic<int> limits[kMaxDevices];           // of this kernel
  ensure_dynamic_smem(kernel, 1024, bytes, limits);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(p.ctas), 1, (a.tokens + 8 * NT - 1) / (8 * NT));
  cfg.blockDim = dim3(32 * kWarps + (Boxes ? kCopyThreads : kLooseThreads));
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
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a, map_w, map_x, map_s, map_z);
  if (e != cudaSuccess || !p.cut) return e;
  cfg.gridDim.x = unsigned(p.ctas - 1);
  cfg.gridDim.y = unsigned((kRows * p.warps_n * held + 4 * kJoinThreads - 1) / (4 * kJoinThreads));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.dynamicSmemBytes = 0;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, w4_join_kernel<T, NT>, a);
}

template <class T, int NT, int GB, bool Boxes>
cudaError_t launch_scales(const W4Args& a, const Plan& p, cudaStream_t s) {
  constexpr int kGroups = Tile<NT>::kK / 32 / GB;
  // copies bring rows of 16 bytes or more from 16-byte boundaries, in the tokens' type; a tile's scales are read as one
  // word, so they are its kGroups, or the one of a group of several tiles
  const bool whole = kGroups == 1 ? a.group % (32 * GB) == 0 && (a.group & (a.group - 1)) == 0 : a.group == 32 * GB;
  const bool side = Boxes && whole && !a.scales32 && aligned(a.scales, 16) && a.groups % 8 == 0 &&
                    (!a.zeros || (aligned(a.zeros, 16) && a.groups % 16 == 0));
  return side ? launch_shape<T, NT, GB, Boxes, Boxes>(a, p, s) : launch_shape<T, NT, GB, Boxes, false>(a, p, s);
}

// A kernel for each number of groups in a tile.  Scales by copies and by loads of each lane (us): one token x 28672 x
// 8192 in groups of 128 32.4 and 36.1, 16 tokens in groups of 64 46.8 and 74.7, of 32 (8192 x 28672) 50.2 and 141.
template <class T, int NT, bool Boxes>
cudaError_t launch_group(const W4Args& a, const Plan& p, cudaStream_t s) {
  if (a.group == 64) return launch_scales<T, NT, 2, Boxes>(a, p, s);
  if (NT == 1 && a.group % 256 == 0) return launch_scales<T, NT, NT == 1 ? 8 : 4, Boxes>(a, p, s);
  if (a.group == 128 || (NT == 2 && a.group % 128 == 0)) return launch_scales<T, NT, 4, Boxes>(a, p, s);
  return launch_scales<T, NT, 1, Boxes>(a, p, s);
}

// Copies of boxes need 16-byte rows; by pieces one token x 28672 x 8190 takes 62 us (8192 in boxes 32), 16 tokens 128 (45),
// 8 tokens x 4096 x 11006 24 (by four warps that shifted words into place 101, 174 and 48).  What the copying warps have to do for each piece, and two stages at a time, bound it.
template <class T>
cudaError_t launch(const W4Args& a, const Plan& p, cudaStream_t s) {
  const bool aligned_rows = aligned(a.weight, 16) && a.weight_stride % 16 == 0 && a.x_pieces;
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

extern "C" uint64_t pm_matvec_w4_wait_limit(uint64_t nanoseconds) {
  return g_wait_ns.exchange(nanoseconds ? std::min(nanoseconds, uint64_t(1) << 62) : kWaitNs);   // added to a clock
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
           j->x_stride, j->weight_stride, j->x, j->weight, j->scales, j->zeros, j->y, g_wait_ns.load(std::memory_order_relaxed), 0, aligned(j->x, 16) && (j->x_stride % 8 == 0 || j->tokens == 1), 0, 0, 0, 0, 0, 0, 0, 0, 0, static_cast<float*>(scratch)};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = j->dtype == PM_DT_BF16 ? launch<bf16>(a, plan, s) : launch<fp16>(a, plan, s);
  return e == cudaSuccess ? PM_OK : cuda_fail(e, "pm_matvec_w4_device launch");
}
