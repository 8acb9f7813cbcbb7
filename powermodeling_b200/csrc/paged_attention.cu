// Attention of one query token per sequence over a paged key-value cache:
//   out = softmax(scale q K^T) V over the live positions.
//
// The cache is read once for every 8 or 16 query heads of a key head and
// everything else is small, so the bytes of K and V over the memory's rate
// bound it; what the kernel has to do is to keep
// enough bytes in flight on every SM whatever the lengths are.
//  * Work is counted in tiles of 64 positions of one (sequence, key head).
//    All tiles of all sequences form one line, on which the start of each
//    (sequence, key head) counts as two tiles more (filling and draining the
//    copies takes about as long), and the line is cut into as many equal runs
//    as CTAs are resident: the CTAs read the lengths and find their run
//    themselves, so neither a long sequence nor a ragged batch leaves SMs
//    idle and the host needs no lengths.  A run that ends inside a sequence
//    leaves (maximum, sum, weighted values) in scratch, at most two such
//    pieces a CTA, and a second kernel joins them in the order of the runs.
//  * A warp takes 16 positions of a tile and has its own ring of 16-byte
//    asynchronous copies into shared memory, its own running maximum and sum:
//    no barrier inside a run.  Positions that are not live are filled with
//    zeros instead of being read, so nothing there (NaN included) counts.
//  * The query heads of one key head are the 8 columns of the matrix
//    instruction: S^T[16 positions x 8 heads] = K Q^T, and O^T[16 dims x 8
//    heads] += V^T P^T, K and V^T being the row operands straight from shared
//    memory.  A group of 8 costs no padding, and its keys are read once; two
//    groups go together where registers allow, further ones each read again.
//    mma.sync serves because 8 columns are all there is: the tensor core is
//    idle most of the time and tcgen05's 128-row tiles would be mostly empty.
//  * A weight enters the product as three 16-bit parts that add up to its 32
//    bits (fp16: to 2^-39 of the largest weight); sums and the running output
//    are 32-bit.  One sequence of 131072 positions takes 105 us so; with two
//    parts (2^-17 of a weight) summed in the instruction 103, and then 7 % of
//    the fp16 outputs over as many positive values were not the nearest to the
//    exact ones, where now 0.02 % are not.
// Measured (a copy runs at 6.55 TB/s): one sequence of 131072 positions, 8 key
// heads of 128, 105 us = 5.1 TB/s; 64 ragged sequences up to 8192, 186 us =
// 5.3 TB/s; 256 of 1024, 197 us = 5.5 TB/s; one of 77 positions 7.8 us, of
// which a copy's round trip, the reduction over the warps and the launch are
// nearly all.  At full length the copies' latency with three CTAs an SM bounds
// it (3.0 of 8.6 cycles between a warp's instructions wait for them), at a few
// tiles a sequence the start of each segment, about 2 us.
#include <climits>
#include <cmath>

#include "blocks.cuh"

namespace pm {
namespace blk {
namespace {

constexpr int kMaxRuns = 148 * 4;        // CTAs of the first kernel at most: sizes the scratch
constexpr int kSeam = 2;                 // what the start of a segment counts for, in tiles
constexpr int kWhole = 4;                // room for so many tiles at most, and a run for each segment: none is cut
constexpr int kWarps = 4, kThreads = 32 * kWarps, kSlice = 16, kTile = kSlice * kWarps;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnArgs {
  pm_paged_attention j;
  int page_shift;                        // log2 of the page size, -1: no power of two
  int whole;                             // runs end between segments: none is cut
  int share, blocks;                     // query heads per key head; groups of them that one pass serves
  float* part;                           // [2 * CTAs, kHeads, head_dim] weighted values of split segments
  float2* stat;                          // [2 * CTAs, kHeads] (maximum, sum), base 2
  struct Cut* cuts;                      // [CTAs]
};
// A segment that was cut, noted by the second run that has a piece of it.
struct Cut {
  int pieces, first_run;                 // 0 pieces: this run is no segment's second
  int row, rows;                         // query rows, from the start of out
};

__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// Weights are held times this: fp16 ends at 2^-24, where a weight then is 2^-39 of the largest.
template <class T> constexpr float lift = std::is_same<T, fp16>::value ? 32768.0f : 1.0f;
// Two floats as packed 16-bit values that add up to them: each is cut off where 16 bits end, the next holds what is
// left, the last one rounded.  bf16: 3 x 8 bits, all of a float's; fp16: 3 x 11, as far as they reach.
constexpr int kParts = 3;
__device__ __forceinline__ void split(bf16*, float x, float y, uint32_t (&part)[kParts]) {
#pragma unroll
  for (int i = 0; i < kParts; ++i) {
    const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
    part[i] = __byte_perm(a, b, 0x7632);
    x -= __uint_as_float(a & 0xffff0000u);
    y -= __uint_as_float(b & 0xffff0000u);
  }
}
__device__ __forceinline__ void split(fp16*, float x, float y, uint32_t (&part)[kParts]) {
#pragma unroll
  for (int i = 0; i < kParts; ++i) {
    __half2 h = __floats2half2_rn(x, y);
    if (i + 1 < kParts) {
      asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(part[i]) : "f"(y), "f"(x));
      h = *reinterpret_cast<const __half2*>(&part[i]);
      x -= __low2float(h);
      y -= __high2float(h);
    } else {
      part[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// What exponents are taken from: the largest score, unless it is infinite (then the sum is infinite, or zero).
__device__ __forceinline__ float base_of(float top) { return fabsf(top) == INFINITY ? 0.0f : top; }

// Positions [from, to) of a sequence and the tiles that they touch.
struct Span {
  uint32_t from, to, first;              // first: index of the first tile
  int tiles;
};
__device__ __forceinline__ Span span_of(const pm_paged_attention& j, int b) {
  Span s;
  const int length = max(j.lengths[b], 0);
  const int64_t room = int64_t(j.table_columns) * j.page_size;
  s.from = j.window && length > j.window ? length - j.window : 0;
  s.to = j.n_pages == 0 ? 0u : uint32_t(min(int64_t(length), room));
  s.first = s.from / kTile;
  s.tiles = s.to > s.from ? int((s.to + kTile - 1) / kTile - s.first) : 0;
  return s;
}
// What one key head of a sequence takes on the line; all the same where segments stay whole.
__device__ __forceinline__ int length_of(int tiles, int whole) { return tiles == 0 ? 0 : whole ? 1 : tiles + kSeam; }

// The sequences' lengths on the line, of one key head each, summed over the batch: thread t has the sum over the
// sequences before its `per` consecutive ones, prefix[Threads] all of them.
template <int Threads>
__device__ __forceinline__ int64_t scan_line(const pm_paged_attention& j, int whole, int per, int64_t* prefix) {
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  int64_t own = 0;
  for (int b = t * per; b < min(j.batch, (t + 1) * per); ++b) own += length_of(span_of(j, b).tiles, whole);
  int64_t sum = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += v;
  }
  __shared__ int64_t warp_sums[Threads / 32];
  if (lane == 31) warp_sums[warp] = sum;
  __syncthreads();
  int64_t before = 0;
#pragma unroll
  for (int w = 0; w < Threads / 32; ++w) before += w < warp ? warp_sums[w] : 0;
  prefix[t] = before + sum - own;
  if (t == Threads - 1) prefix[Threads] = before + sum;
  __syncthreads();
  return prefix[Threads];
}

// Infinite values.  A weight's parts may be zero, and zero times an infinity is not what the weight times it is; so
// outputs that are not finite are looked into again: an element is NaN where a live position's value is, where there
// are infinities of both signs, or where a score is -infinity beside an infinite value; else it has the infinity's sign.
// Positions [from, to) of one key head, nh query heads at q; a thread to a position.  found: [nh][head_dim], 1 for
// NaN, 2 and 4 for the infinities.
template <class T>
__device__ __noinline__ void look_into_values(const pm_paged_attention& j, int b, int kvh, uint32_t from, uint32_t to, uint32_t newest,
                                              const T* q, int nh, uint32_t* found) {
  const int D = j.head_dim;
  for (int i = threadIdx.x; i < nh * D; i += blockDim.x) found[i] = 0;
  __syncthreads();
  const int32_t* table = j.table + b * j.table_stride;
  for (uint32_t pos = from + threadIdx.x; pos < to; pos += blockDim.x) {
    const int page = table[pos / uint32_t(j.page_size)], entry = int(pos % uint32_t(j.page_size));
    if (page < 0 || page >= j.n_pages) continue;
    const bool is_new = pos == newest;
    const T* v = is_new ? static_cast<const T*>(j.new_v) + b * j.new_v_stride + kvh * j.new_v_head_stride
                        : static_cast<const T*>(j.v_cache) + page * j.v_page_stride + entry * j.v_token_stride + kvh * j.v_head_stride;
    const T* k = is_new ? static_cast<const T*>(j.new_k) + b * j.new_k_stride + kvh * j.new_k_head_stride
                        : static_cast<const T*>(j.k_cache) + page * j.k_page_stride + entry * j.k_token_stride + kvh * j.k_head_stride;
    bool any = false;
    for (int d = 0; d < D; ++d) any |= !(fabsf(to_float(v[d])) < INFINITY);
    if (!any) continue;
    for (int h = 0; h < nh; ++h) {
      float score = 0.0f;
      for (int d = 0; d < D; ++d) score += to_float(k[d]) * to_float(q[h * j.q_head_stride + d]);
      const bool nothing = score * j.scale == -INFINITY;
      for (int d = 0; d < D; ++d) {
        const float x = to_float(v[d]);
        if (!(fabsf(x) < INFINITY)) atomicOr(&found[h * D + d], x != x || nothing ? 1u : x > 0.0f ? 2u : 4u);
      }
    }
  }
  __syncthreads();
}

// ---------------------------------------------------------------- the runs
// DP: the head size that the kernel is built for, at least head_dim; NT: groups
// of 8 query heads served at once.  A row of shared memory is 16 bytes longer
// than a head, which puts 8 rows' pieces in 32 different banks at every DP.
template <class T, int DP, int NT>
struct Shape {
  static constexpr int kHeads = 8 * NT;
  static constexpr int kPitch = DP * 2 + 16;
  static constexpr int kSliceBytes = 2 * kSlice * kPitch;                       // K, then V
  // two to three slices in flight per warp; with 12 to 16 warps an SM, 90 to 190 KB
  static constexpr int kStages = DP <= 96 ? 3 : 2;
  static constexpr int kWarpBytes = kStages * kSliceBytes;
  static constexpr int kOutStride = DP + 4;                                     // floats; 8t + g: no two lanes in a bank
  static constexpr size_t kSmem = size_t(kWarps) * kWarpBytes;
  static_assert(kHeads * kOutStride * 4 <= kWarpBytes, "a warp's output fits in its ring, and so does what look_into_values finds");
};

template <class T, int DP, int NT>
__global__ void __launch_bounds__(kThreads) attention_runs_kernel(const __grid_constant__ AttnArgs a) {
  using S = Shape<T, DP, NT>;
  constexpr int kChunks = DP / 8;                        // 16-byte pieces of a row
  constexpr int kCopies = kSlice * kChunks / 32;         // per lane, for K and for V
  constexpr float kLift = lift<T>;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ int64_t prefix[kThreads + 1];
  __shared__ int64_t found_before;
  __shared__ int found_b;
  __shared__ uint32_t live_of[kWarps][S::kStages];
  __shared__ float2 warp_stat[kWarps][S::kHeads];
  __shared__ float factor[kWarps][S::kHeads];
  __shared__ float total_of[S::kHeads];

  const pm_paged_attention& j = a.j;
  asm volatile("griddepcontrol.launch_dependents;");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int D = j.head_dim, heads = j.kv_heads * a.blocks;
  const int per = (j.batch + kThreads - 1) / kThreads;
  const int64_t total = scan_line<kThreads>(j, a.whole, per, prefix) * heads;

  // sequences without a live position: zeros
  for (int b = blockIdx.x; b < j.batch; b += gridDim.x) {
    if (span_of(j, b).tiles) continue;
    T* out = static_cast<T*>(j.out) + int64_t(b) * j.q_heads * D;
    for (int64_t i = threadIdx.x; i < int64_t(j.q_heads) * D; i += kThreads) out[i] = from_float<T>(0.0f);
    if (j.lse)
      for (int i = threadIdx.x; i < j.q_heads; i += kThreads) j.lse[int64_t(b) * j.q_heads + i] = -INFINITY;
  }

  const int64_t runs = min(int64_t(gridDim.x), total);   // no run is empty
  if (threadIdx.x == 0) a.cuts[blockIdx.x].pieces = 0;
  if (blockIdx.x >= runs) return;
  int64_t cur = total * blockIdx.x / runs;
  const int64_t end = total * (blockIdx.x + 1) / runs;
  if (prefix[threadIdx.x] * heads <= cur && cur < prefix[threadIdx.x + 1] * heads) {
    int64_t before = prefix[threadIdx.x];
    int b = threadIdx.x * per;
    for (;; ++b) {
      const int n = length_of(span_of(j, b).tiles, a.whole);
      if (cur < (before + n) * heads) break;
      before += n;
    }
    found_b = b;
    found_before = before;
  }
  __syncthreads();
  int b = found_b;
  Span sp = span_of(j, b);
  int64_t base = found_before * heads;                   // where the sequence starts on the line

  // page and entry of a position
  auto page_at = [&](uint32_t pos) { return a.page_shift >= 0 ? pos >> a.page_shift : pos / uint32_t(j.page_size); };
  auto entry_of = [&](uint32_t pos) { return int(a.page_shift >= 0 ? pos & uint32_t(j.page_size - 1) : pos % uint32_t(j.page_size)); };
  // Slices that lie in one page, of heads without padding and with the same way from token to token in K and V, are
  // copied by these offsets (elements) of a lane's pieces
  const bool plain = D == DP && j.page_size % kSlice == 0 && j.k_token_stride == j.v_token_stride && j.k_token_stride < (1 << 26);
  uint32_t from_row[kCopies];
#pragma unroll
  for (int c = 0; c < kCopies; ++c) from_row[c] = uint32_t((c * 32 + lane) / kChunks) * uint32_t(j.k_token_stride) + (c * 32 + lane) % kChunks * 8;

  uint8_t* mine = ring + warp * S::kWarpBytes;
  const uint32_t mine_addr = smem_addr(mine);
  const float scale2 = j.scale * kLog2e;

  while (cur < end) {
    const int length = length_of(sp.tiles, a.whole);
    const uint64_t into = uint64_t(cur - base);
    // key head and group of query heads; a 64-bit division only where it takes one
    const int which = into >> 32 ? int(into / uint64_t(length)) : int(uint32_t(into) / uint32_t(length));
    const int kvh = which / a.blocks, hb = which - kvh * a.blocks;
    const int64_t s0 = base + int64_t(which) * length;   // the segment, and this run's part of it
    const int part0 = int(cur - s0), part1 = int(min(int64_t(length), part0 + (end - cur)));
    const int t0 = a.whole ? 0 : max(part0 - kSeam, 0), t1 = a.whole ? sp.tiles : max(part1 - kSeam, 0);
    const int h0 = kvh * a.share + hb * S::kHeads, nh = min(S::kHeads, a.share - hb * S::kHeads);
    if (t1 > t0) {
      const int n_slices = t1 - t0;                        // one slice of this warp in each tile
      const uint32_t pos0 = (sp.first + t0) * uint32_t(kTile) + warp * kSlice;
      const int32_t* table = j.table + b * j.table_stride;
      const T* kc = static_cast<const T*>(j.k_cache) + kvh * j.k_head_stride;
      const T* vc = static_cast<const T*>(j.v_cache) + kvh * j.v_head_stride;
      const T* nk = static_cast<const T*>(j.new_k) + b * j.new_k_stride + kvh * j.new_k_head_stride;
      const T* nv = static_cast<const T*>(j.new_v) + b * j.new_v_stride + kvh * j.new_v_head_stride;
      const uint32_t newest = j.new_k ? uint32_t(max(j.lengths[b], 0)) - 1u : 0xffffffffu;

      // the page of this lane's position (lanes 0-15) in slice i, -1 where it is not live
      auto page_of = [&](int i) {
        const uint32_t pos = pos0 + uint32_t(i) * kTile + lane;
        int page = -1;
        if (i < n_slices && lane < kSlice && pos >= sp.from && pos < sp.to) {
          page = table[page_at(pos)];
          if (page >= j.n_pages) page = -1;
        }
        return page;
      };
      auto fetch = [&](int i, int page) {
        const uint32_t live = i < n_slices ? __ballot_sync(0xffffffffu, page >= 0) & 0xffffu : 0u;
        if (live) {
          const uint32_t first_pos = pos0 + uint32_t(i) * kTile;
          const int off = entry_of(first_pos + lane), stage = i % S::kStages;
          if (lane == 0) live_of[warp][stage] = live;
          const uint32_t kdst = mine_addr + stage * S::kSliceBytes, vdst = kdst + kSlice * S::kPitch;
          // the new token's row, if it is here: read from its own tensors, and written to the cache by the first group
          const int new_row = newest - first_pos < uint32_t(kSlice) && live >> (newest - first_pos) & 1u ? int(newest - first_pos) : -1;
          if (new_row >= 0 && hb == 0) {
            const int new_page = __shfl_sync(0xffffffffu, page, new_row), new_off = __shfl_sync(0xffffffffu, off, new_row);
            if (lane * 8 < D) {
              T* ks = const_cast<T*>(kc) + new_page * j.k_page_stride + new_off * j.k_token_stride + lane * 8;
              T* vs = const_cast<T*>(vc) + new_page * j.v_page_stride + new_off * j.v_token_stride + lane * 8;
              *reinterpret_cast<uint4*>(ks) = *reinterpret_cast<const uint4*>(nk + lane * 8);
              *reinterpret_cast<uint4*>(vs) = *reinterpret_cast<const uint4*>(nv + lane * 8);
            }
          }
          if (plain) {
            // the slice is in one page: rows a fixed way apart
            const int some = __ffs(live) - 1;
            const int page0 = __shfl_sync(0xffffffffu, page, some), off0 = __shfl_sync(0xffffffffu, off, 0);
            const T* ks = kc + page0 * j.k_page_stride + off0 * j.k_token_stride;
            const T* vs = vc + page0 * j.v_page_stride + off0 * j.v_token_stride;
            if (live == 0xffffu && new_row < 0) {
#pragma unroll
              for (int c = 0; c < kCopies; ++c) {
                const int idx = c * 32 + lane, row = idx / kChunks, chunk = idx % kChunks;
                copy16(kdst + row * S::kPitch + chunk * 16, ks + from_row[c], 16);
                copy16(vdst + row * S::kPitch + chunk * 16, vs + from_row[c], 16);
              }
            } else {
#pragma unroll
              for (int c = 0; c < kCopies; ++c) {
                const int idx = c * 32 + lane, row = idx / kChunks, chunk = idx % kChunks;
                const int bytes = live >> row & 1u ? 16 : 0;
                copy16(kdst + row * S::kPitch + chunk * 16, row == new_row ? nk + chunk * 8 : ks + from_row[c], bytes);
                copy16(vdst + row * S::kPitch + chunk * 16, row == new_row ? nv + chunk * 8 : vs + from_row[c], bytes);
              }
            }
          } else {
#pragma unroll
            for (int c = 0; c < kCopies; ++c) {
              const int idx = c * 32 + lane, row = idx / kChunks, chunk = idx % kChunks;
              const int row_page = __shfl_sync(0xffffffffu, page, row), row_off = __shfl_sync(0xffffffffu, off, row);
              const bool read = row_page >= 0 && chunk * 8 < D;
              const T* ks = kc;
              const T* vs = vc;
              if (read) {
                ks = row == new_row ? nk + chunk * 8 : ks + (row_page * j.k_page_stride + row_off * j.k_token_stride + chunk * 8);
                vs = row == new_row ? nv + chunk * 8 : vs + (row_page * j.v_page_stride + row_off * j.v_token_stride + chunk * 8);
              }
              copy16(kdst + row * S::kPitch + chunk * 16, ks, read ? 16 : 0);
              copy16(vdst + row * S::kPitch + chunk * 16, vs, read ? 16 : 0);
            }
          }
        } else if (i < n_slices && lane == 0) {
          live_of[warp][i % S::kStages] = 0;
        }
        commit();
      };

      // queries as the column operand: head g, dims 2t, 2t+1 and 2t+8, 2t+9 of each 16
      uint32_t q[NT][DP / 16][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const bool have = n * 8 + g < nh;
        const T* qp = static_cast<const T*>(j.q) + b * j.q_stride + (h0 + (have ? n * 8 + g : 0)) * j.q_head_stride;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int d = k * 16 + e * 8 + 2 * t;
            q[n][k][e] = have && d < D ? *reinterpret_cast<const uint32_t*>(qp + d) : 0u;
          }
      }

      float o[NT][DP / 16][4] = {};
      float top[NT][2], sum[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) top[n][0] = top[n][1] = -INFINITY, sum[n][0] = sum[n][1] = 0.0f;

      int page = page_of(0);
#pragma unroll
      for (int i = 0; i < S::kStages - 1; ++i) {
        const int ahead = page_of(i + 1);
        fetch(i, page);
        page = ahead;
      }
      for (int i = 0; i < n_slices; ++i) {
        // the page index of the slice after the next fetch travels while this slice is computed
        const int ahead = page_of(i + S::kStages);
        fetch(i + S::kStages - 1, page);
        page = ahead;
        wait_groups<S::kStages - 1>();
        __syncwarp();
        const int stage = i % S::kStages;
        const uint32_t live = live_of[warp][stage];
        if (live) {
          const uint32_t kbase = mine_addr + stage * S::kSliceBytes, vbase = kbase + kSlice * S::kPitch;
          float s[NT][4];
          {
            // even and odd 16 dims apart: half as long a chain of sums
            float odd[NT][4];
            const uint32_t at = kbase + (lane & 15) * S::kPitch + (lane >> 4) * 16;
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
              uint32_t ka[4];
              ldsm(ka, at + k * 32);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                if (k == 0) mma_first<T>(s[n], ka, q[n][k][0], q[n][k][1]);
                else if (k == 1) mma_first<T>(odd[n], ka, q[n][k][0], q[n][k][1]);
                else if (k & 1) mma<T>(odd[n], ka, q[n][k][0], q[n][k][1]);
                else mma<T>(s[n], ka, q[n][k][0], q[n][k][1]);
              }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) s[n][e] = (s[n][e] + odd[n][e]) * scale2;
          }
          const bool live_a = live >> g & 1, live_b = live >> (g + 8) & 1;
          uint32_t w[NT][2][kParts];                       // weights of rows g and g + 8
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (live != 0xffffu) {
              s[n][0] = live_a ? s[n][0] : -INFINITY;
              s[n][1] = live_a ? s[n][1] : -INFINITY;
              s[n][2] = live_b ? s[n][2] : -INFINITY;
              s[n][3] = live_b ? s[n][3] : -INFINITY;
            }
            float m0 = fmaxf(s[n][0], s[n][2]), m1 = fmaxf(s[n][1], s[n][3]);
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
              m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, x));
              m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, x));
            }
            m0 = fmaxf(m0, top[n][0]);
            m1 = fmaxf(m1, top[n][1]);
            const float b0 = base_of(m0), b1 = base_of(m1);
            if (__any_sync(0xffffffffu, m0 != top[n][0] || m1 != top[n][1])) {
              const float c0 = exp2_fast(top[n][0] - b0), c1 = exp2_fast(top[n][1] - b1);
              sum[n][0] *= c0;
              sum[n][1] *= c1;
#pragma unroll
              for (int k = 0; k < DP / 16; ++k) {
                o[n][k][0] *= c0; o[n][k][1] *= c1; o[n][k][2] *= c0; o[n][k][3] *= c1;
              }
              top[n][0] = m0;
              top[n][1] = m1;
            }
            const float p0 = exp2_fast(s[n][0] - b0) * kLift, p1 = exp2_fast(s[n][1] - b1) * kLift;
            const float p2 = exp2_fast(s[n][2] - b0) * kLift, p3 = exp2_fast(s[n][3] - b1) * kLift;
            sum[n][0] += p0 + p2;
            sum[n][1] += p1 + p3;
            split(static_cast<T*>(nullptr), p0, p1, w[n][0]);
            split(static_cast<T*>(nullptr), p2, p3, w[n][1]);
#pragma unroll
            for (int i = 0; i < kParts; ++i) {
              w[n][0][i] = transpose8(w[n][0][i]);
              w[n][1][i] = transpose8(w[n][1][i]);
            }
          }
          {
            const uint32_t at = vbase + ((lane & 7) + (lane >> 4) * 8) * S::kPitch + (lane >> 3 & 1) * 16;
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
              uint32_t va[4];
              ldsm_t(va, at + k * 32);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                // the slice's own sum, smallest parts first: the instruction cuts its sums off, which over a long
                // sequence would add up (2^-14 of the output after 600 slices); the running one is rounded
                float slice[4];
                mma_first<T>(slice, va, w[n][0][kParts - 1], w[n][1][kParts - 1]);
#pragma unroll
                for (int i = kParts - 2; i >= 0; --i) mma<T>(slice, va, w[n][0][i], w[n][1][i]);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][k][e] += slice[e];
              }
            }
          }
        }
        __syncwarp();                                      // the slice is read before its place is filled again
      }
      wait_groups<0>();
      __syncwarp();

      // the warps' results through shared memory, each in its own ring
      float* ow = reinterpret_cast<float*>(mine);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          sum[n][0] += __shfl_xor_sync(0xffffffffu, sum[n][0], x);
          sum[n][1] += __shfl_xor_sync(0xffffffffu, sum[n][1], x);
        }
        if (g == 0) {
          warp_stat[warp][n * 8 + 2 * t] = make_float2(top[n][0], sum[n][0]);
          warp_stat[warp][n * 8 + 2 * t + 1] = make_float2(top[n][1], sum[n][1]);
        }
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          float* at = ow + (n * 8 + 2 * t) * S::kOutStride + k * 16 + g;
          at[0] = o[n][k][0];
          at[S::kOutStride] = o[n][k][1];
          at[8] = o[n][k][2];
          at[S::kOutStride + 8] = o[n][k][3];
        }
      }
      __syncthreads();
      const bool whole = t0 == 0 && t1 == sp.tiles;
      const int64_t slot = 2 * int64_t(blockIdx.x) + (t0 == 0 ? 1 : 0);
      if (threadIdx.x < S::kHeads) {
        const int h = threadIdx.x;
        if (h == 0 && t0 > 0) {
          // the run with the segment's first tile; the one after it notes the cut
          const int c0 = int(((s0 + kSeam + 1) * runs - 1) / total), c1 = int(((s0 + length) * runs - 1) / total);
          if (c0 + 1 == blockIdx.x) {
            a.cuts[blockIdx.x] = {c1 - c0 + 1, c0, b * j.q_heads + h0, nh};
          }
        }
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = fmaxf(m, warp_stat[w][h].x);
        const float mb = base_of(m);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float f = exp2_fast(warp_stat[w][h].x - mb);
          factor[w][h] = f;
          l += warp_stat[w][h].y * f;
        }
        total_of[h] = l;
        if (h < nh) {
          if (!whole) a.stat[slot * S::kHeads + h] = make_float2(m, l);
          else if (j.lse) j.lse[int64_t(b) * j.q_heads + h0 + h] = l == 0.0f ? -INFINITY : mb * kLn2 + logf(l / kLift);
        }
      }
      __syncthreads();
      auto put = [&](int h, int d, float v, float l) {
        if (whole) static_cast<T*>(j.out)[(int64_t(b) * j.q_heads + h0 + h) * D + d] = from_float<T>(l == 0.0f ? 0.0f : v / l);
        else a.part[(slot * S::kHeads + h) * D + d] = v;
      };
      bool odd = false;
      for (int h = 0; h < nh; ++h) {
        const float l = total_of[h];
        for (int d = threadIdx.x; d < D; d += kThreads) {
          float v = 0.0f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w)
            v += reinterpret_cast<const float*>(ring + w * S::kWarpBytes)[h * S::kOutStride + d] * factor[w][h];
          put(h, d, v, l);
          odd |= !(fabsf(v) < INFINITY);
        }
      }
      if (__syncthreads_or(odd)) {
        uint32_t* found = reinterpret_cast<uint32_t*>(ring);
        look_into_values<T>(j, b, kvh, max(sp.from, (sp.first + t0) * uint32_t(kTile)), min(sp.to, (sp.first + t1) * uint32_t(kTile)), newest,
                            static_cast<const T*>(j.q) + b * j.q_stride + h0 * j.q_head_stride, nh, found);
        for (int h = 0; h < nh; ++h) {
          const float l = total_of[h];
          if (!(l > 0.0f)) continue;                       // NaN for every element, or nothing but scores of -infinity
          for (int d = threadIdx.x; d < D; d += kThreads) {
            const uint32_t f = found[h * D + d];
            if (f) put(h, d, f == 2 ? INFINITY : f == 4 ? -INFINITY : NAN, l);
          }
        }
        __syncthreads();
      }
    }

    cur += part1 - part0;
    if (cur < end && cur == base + int64_t(length) * heads) {
      base = cur;
      do sp = span_of(j, ++b);                           // the line goes on: a later sequence has tiles
      while (!sp.tiles);
    }
  }
}

// Joins the pieces of each segment that was cut: one CTA per query head.  A
// thread has four neighbouring values; groups of threads take every so many
// pieces, whose factors were computed by a thread each.
constexpr int kJoinThreads = 256;
template <class T, int NT>
__global__ void __launch_bounds__(kJoinThreads) attention_join_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int kHeads = 8 * NT;
  __shared__ float factor[kMaxRuns], partial[8];
  __shared__ float4 sums[kJoinThreads];
  const pm_paged_attention& j = a.j;
  const int t = threadIdx.x, D = j.head_dim, row = blockIdx.y;
  asm volatile("griddepcontrol.wait;" ::: "memory");    // in every CTA: this kernel's end has to mean the first one's
  const int4 c = __ldcg(reinterpret_cast<const int4*>(&a.cuts[blockIdx.x + 1]));
  const int n = c.x;
  if (!n || row >= c.w) return;
  // a run's slots: first the piece that it starts within, then the one that it ends within, which is a segment's first
  auto slot_of = [&](int i) { return 2 * int64_t(c.y + i) + (i == 0 ? 1 : 0); };
  float m = -INFINITY;
  for (int i = t; i < n; i += kJoinThreads) {
    const float top = __ldcg(&a.stat[slot_of(i) * kHeads + row]).x;
    factor[i] = top;
    m = fmaxf(m, top);
  }
#pragma unroll
  for (int x = 16; x; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
  if ((t & 31) == 0) partial[t >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) m = fmaxf(m, partial[w]);
  const float mb = base_of(m);
  __syncthreads();
  float l = 0.0f;
  for (int i = t; i < n; i += kJoinThreads) {
    const float f = exp2_fast(factor[i] - mb);
    factor[i] = f;
    l += __ldcg(&a.stat[slot_of(i) * kHeads + row]).y * f;
  }
  l = warp_sum(l);
  if ((t & 31) == 0) partial[t >> 5] = l;
  __syncthreads();
  l = 0.0f;
#pragma unroll
  for (int w = 0; w < 8; ++w) l += partial[w];
  const int quads = D / 4, lanes = quads <= 16 ? 16 : quads <= 32 ? 32 : 64, lane = t % lanes, groups = kJoinThreads / lanes;
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (lane < quads) {
#pragma unroll 8
    for (int i = t / lanes; i < n; i += groups) {
      const float4 p = __ldcg(reinterpret_cast<const float4*>(a.part + (slot_of(i) * kHeads + row) * D) + lane);
      const float f = factor[i];
      auto part = [&](float x) { return fabsf(x) == INFINITY ? x : x * f; };               // f may be zero
      v.x += part(p.x); v.y += part(p.y); v.z += part(p.z); v.w += part(p.w);
    }
  }
  sums[t] = v;
  __syncthreads();
  if (t < quads) {
    for (int g = 1; g < groups; ++g) {
      const float4 p = sums[g * lanes + t];
      v.x += p.x; v.y += p.y; v.z += p.z; v.w += p.w;
    }
    T* out = static_cast<T*>(j.out) + int64_t(c.z + row) * D + 4 * t;
    out[0] = from_float<T>(l == 0.0f ? 0.0f : v.x / l);
    out[1] = from_float<T>(l == 0.0f ? 0.0f : v.y / l);
    out[2] = from_float<T>(l == 0.0f ? 0.0f : v.z / l);
    out[3] = from_float<T>(l == 0.0f ? 0.0f : v.w / l);
  }
  if (j.lse && t == 0) j.lse[c.z + row] = l == 0.0f ? -INFINITY : mb * kLn2 + logf(l / lift<T>);
}

// ---------------------------------------------------------------- launch
// Query heads in groups of 8, two groups at once where more than 8 share a
// key head and their registers allow it (head_dim up to 128): 32 sequences up
// to 8192, 4 key heads, with 16 query heads a key head of 128 76 us, group
// after group 94; 12 heads of 64 47 and 56 us.
int tiles_of_heads(int share, int head_dim) { return share > 8 && head_dim <= 128 ? 2 : 1; }

template <class T, int DP, int NT>
cudaError_t launch_shape(AttnArgs& a, uint8_t* scratch, int sms, cudaStream_t s) {
  using S = Shape<T, DP, NT>;
  static std::atomic<int> occupancy[kMaxDevices], limits[kMaxDevices];   // of this kernel
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const auto kernel = attention_runs_kernel<T, DP, NT>;
  std::atomic<int>& known = occupancy[device];
  int occ = known.load(std::memory_order_relaxed);
  if (!occ) {
    ensure_dynamic_smem(kernel, 4096, S::kSmem, limits);
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, kernel, kThreads, S::kSmem);
    if (e != cudaSuccess) return e;
    if (occ < 1) return cudaErrorInvalidConfiguration;
    known.store(occ, std::memory_order_relaxed);
  }
  const pm_paged_attention& j = a.j;
  a.blocks = (a.share + S::kHeads - 1) / S::kHeads;
  int64_t runs = int64_t(sms) * occ;
  if (runs > kMaxRuns) runs = kMaxRuns;
  // The tables' full length bounds the lengths.  Where every segment has a run to itself and few tiles, none is cut:
  // the join's launch costs more than the tiles in turn (us whole and cut: 8 sequences x 8 heads with 128 positions
  // 7.4 and 8.9, with 256 10.0 and 11.9, with 512 15.1 and 13.1; 128 x 8 segments of 256, more than runs, 38.5 and 36.8).
  const int64_t room = (int64_t(j.table_columns) * j.page_size + kTile - 1) / kTile;
  const int64_t segments = int64_t(j.batch) * j.kv_heads * a.blocks;
  a.whole = room <= 1 || (room <= kWhole && segments <= runs);
  const int64_t most = segments * (a.whole ? 1 : room < (1 << 20) ? room : (1 << 20));   // no more runs than work
  if (runs > most) runs = most;
  a.cuts = reinterpret_cast<Cut*>(scratch);
  a.stat = reinterpret_cast<float2*>(scratch + kMaxRuns * sizeof(Cut));
  a.part = reinterpret_cast<float*>(scratch + kMaxRuns * sizeof(Cut) + size_t(2) * kMaxRuns * S::kHeads * sizeof(float2));
  kernel<<<unsigned(runs), kThreads, S::kSmem, s>>>(a);
  e = cudaGetLastError();
  if (e != cudaSuccess || a.whole || runs <= 1) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(runs - 1), unsigned(a.share < S::kHeads ? a.share : S::kHeads));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = s;
  cudaLaunchAttribute early[1];
  early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = early;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, attention_join_kernel<T, NT>, a);
}

template <class T>
cudaError_t launch(const pm_paged_attention& j, void* scratch, int sms, cudaStream_t s) {
  AttnArgs a{};
  a.j = j;
  a.share = j.q_heads / j.kv_heads;
  a.page_shift = j.page_size & (j.page_size - 1) ? -1 : 31 - __builtin_clz(unsigned(j.page_size));
  uint8_t* f = static_cast<uint8_t*>(scratch);
  const int nt = tiles_of_heads(a.share, j.head_dim);
  // a head's own size in shared memory and registers, where it is usual: 32 sequences up to 8192, 8 key heads of 80 97 us
  // (by the kernel for 128 110), of 96 97 (110), of 192 155 (by the kernel for 256 359)
  if (j.head_dim > 64 && j.head_dim <= 80) return nt == 2 ? launch_shape<T, 80, 2>(a, f, sms, s) : launch_shape<T, 80, 1>(a, f, sms, s);
  if (j.head_dim > 80 && j.head_dim <= 96) return nt == 2 ? launch_shape<T, 96, 2>(a, f, sms, s) : launch_shape<T, 96, 1>(a, f, sms, s);
  if (j.head_dim <= 64) return nt == 2 ? launch_shape<T, 64, 2>(a, f, sms, s) : launch_shape<T, 64, 1>(a, f, sms, s);
  if (j.head_dim <= 128) return nt == 2 ? launch_shape<T, 128, 2>(a, f, sms, s) : launch_shape<T, 128, 1>(a, f, sms, s);
  return j.head_dim <= 192 ? launch_shape<T, 192, 1>(a, f, sms, s) : launch_shape<T, 256, 1>(a, f, sms, s);
}

}  // namespace
}  // namespace blk
}  // namespace pm

using namespace pm;
using namespace pm::blk;

extern "C" size_t pm_paged_attention_scratch_bytes(int32_t batch, int32_t q_heads, int32_t kv_heads, int32_t head_dim) {
  if (batch < 1 || q_heads < 1 || kv_heads < 1 || head_dim < 1 || q_heads % kv_heads) return 0;
  const size_t rows = size_t(2) * kMaxRuns * 8 * tiles_of_heads(q_heads / kv_heads, head_dim);
  return kMaxRuns * sizeof(Cut) + rows * sizeof(float2) + rows * size_t(head_dim) * sizeof(float);
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
  const cudaError_t e = j->dtype == PM_DT_BF16 ? launch<bf16>(*j, scratch, sms, s) : launch<fp16>(*j, scratch, sms, s);
  return e == cudaSuccess ? PM_OK : cuda_fail(e, "pm_paged_attention_device launch");
}
