// Attention over the 8-bit key/value cache (kv_cache.cuh) for the last `tokens` positions of
// each sequence: out_i = sum_j softmax_j(scale q_i . k_j) v_j over the positions
// j <= lengths - tokens + i, k_j = code * k_scale[block, head], v_j = code * v_scale[block, head].
// q, out: [batch][tokens][heads][dim]; query head h reads key/value head h / group. A row that
// sees nothing is zeros. No reference counterpart.
//
// Bound by HBM (measured: 4 sequences of up to 131072, 64/8 heads of 128, 107 us, 6.1 TB/s, 0.94 of measured copy bandwidth; 64 of up
// to 4096, 32/8 heads, 57 us, 5.8 TB/s; one of 777, 8/2 heads of 64, 7.8 us, latency): every code is read once,
// 2 dim bytes a token and key/value head, against 4 dim flops a token and query head. Each warp is a worker of its own: all tiles of 64 positions of all
// (sequence, key/value head) pairs are numbered in one line, and worker w takes the w-th equal part of it, so
// ragged lengths leave nobody idle, whatever they are (the host never reads them). A pair that lies
// in one part is finished there; of the others each worker leaves its maximum, sum and
// accumulator, which a second kernel joins in a fixed order. Within a warp:
//   * The codes arrive by bulk copies into the warp's own ring of slots (a tile of K, a tile of V, ...); a slot is
//     refilled as soon as the warp has read it, so there are no barriers between warps.
//   * The products run as D = A B with the codes as A and the few query rows as the 8 columns of B
//     (mma m16n8k16), S^T = K Q^T and O^T = V^T P^T: 8 query rows fill an instruction, with the
//     queries as A they would fill half of it. tcgen05.mma would take 64 rows at least and its operands
//     from shared memory, in 16 bits: the codes would be written back there once more.
//   * A code is exact in f16 (and in bf16, at twice the instructions): one byte permutation puts it into
//     the mantissa of 1024 + code + 128, one packed subtraction takes 1152 off. The dims
//     within a product, and the tokens within the second one, are taken in the order in which a thread finds
//     them in 16 consecutive bytes; P gets into that order by the choice of the token for each row of S^T.
//   * P carries V's scale: with t = score + log2(v_scale), P = 2^(t - max t) is at most 1 for every row,
//     whatever the sizes of the blocks' values. It is rounded to f16 (2^-11; from 2^10 down to 2^-24, so
//     nothing within 2^-34 of the row's largest is lost); the denominator is summed in f32 before that.
//   * f32 queries: Q and P as the sum of two f16 values each, two products in place of one, into fresh accumulators every 64
//     channels and every tile: the tensor core cuts its sums off, always towards zero, where f32 rounds them.
#include <cuda_fp16.h>
#include <math.h>

#include <mutex>

#include "kv_cache.cuh"
#include "umma_ptx.cuh"

namespace b200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTileTokens = 64;
constexpr float kHeadroom = 10.f;         // P = 2^(t - max + 10) ...
constexpr float kStale = 5.f;             // ... and the maximum may be 5 behind: at most 2^15 in f16
constexpr float kSmallestScale = 7.888609052210118e-31f;
constexpr int kErrCachedWait = 1024;

struct CachedParams {
  Cache cache;
  Table table;
  const void* q;
  void* out;  // contiguous
  int64_t q_batch, q_token, q_head;
  const int32_t* lengths;
  int32_t batch, tokens, heads, group;
  int32_t rows, row_tiles;  // query rows of a (sequence, key/value head): tokens * group, row = token * group + head within the group
  int32_t workers;
  int32_t q_vectors;  // q can be read as 16-byte vectors
  float scale_log2, q_sign;  // |scale| * log2(e) and the scale's sign, which the queries take (a scale of 0: 1 and 0)
  float* partial;  // [workers][2][rows of a tile x (2 + dim)]
  int32_t* status;
};

__device__ const float g_not_a_number = __builtin_nanf("");

__device__ __forceinline__ int64_t capacity_of(const CachedParams& p) {
  return static_cast<int64_t>(p.table.width) << p.cache.token_bits;
}
// Tiles of one (sequence, head, row tile). A sequence that its table cannot hold has none: it is answered with NaN.
__device__ __forceinline__ int32_t tiles_of(const CachedParams& p, int32_t b) {
  const int64_t length = p.lengths[b];
  return length <= 0 || length > capacity_of(p) ? 0 : static_cast<int32_t>((length + kTileTokens - 1) / kTileTokens);
}
// Tiles of all sequences (the launch made sure that 32 bits hold them), and of those before sequence `upto`.
__device__ __forceinline__ int32_t count_tiles(const CachedParams& p, int32_t upto, int32_t& before) {
  int32_t sum = 0;
  before = 0;
#pragma unroll 4
  for (int32_t b = threadIdx.x & 31; b < p.batch; b += 32) {
    const int32_t tiles = tiles_of(p, b);
    sum += tiles;
    if (b < upto) before += tiles;
  }
  const int32_t pairs = p.cache.heads * p.row_tiles;
  before = __reduce_add_sync(0xffffffffu, before) * pairs;
  return __reduce_add_sync(0xffffffffu, sum) * pairs;
}
__device__ __forceinline__ int32_t tiles_per_worker(const CachedParams& p, int32_t total) {
  return (total + p.workers - 1) / p.workers;
}
// What a worker leaves of a pair that it did not do alone: maximum and sum of each row, then the accumulator. In slot 1 if
// the pair began with this worker, in slot 0 otherwise (a worker has one of either at most).
template <int ROWS, int D>
__device__ __forceinline__ float* partial_of(const CachedParams& p, int32_t worker, int slot) {
  return p.partial + static_cast<int64_t>(worker * 2 + slot) * (ROWS * (2 + D));
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Of f32 values the part that f16 leaves over.
__device__ __forceinline__ uint32_t half2_rest(float lo, float hi, uint32_t rounded) {
  const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&rounded));
  return half2_bits(lo - r.x, hi - r.y);
}
// Four codes to f16: bytes 0, 1 and bytes 2, 3.
__device__ __forceinline__ void codes_to_half(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  const uint32_t biased = codes ^ 0x80808080u;
  lo = __byte_perm(biased, 0x64646464u, 0x4140);
  hi = __byte_perm(biased, 0x64646464u, 0x4342);
  const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
  const __half2 a = __hsub2(*reinterpret_cast<__half2*>(&lo), bias), b = __hsub2(*reinterpret_cast<__half2*>(&hi), bias);
  lo = *reinterpret_cast<const uint32_t*>(&a);
  hi = *reinterpret_cast<const uint32_t*>(&b);
}

// Codes are read once a call: they go first when L2 needs room (61 -> 57 us on 64 sequences of up to 4096: the lines
// that stay are whole blocks that the next step finds again).
__device__ __forceinline__ uint64_t read_once_policy() {
  uint64_t policy;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  return policy;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(bar), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void word_load(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// Arrives (without raising the expected count) when this thread's word_loads so far have landed.
__device__ __forceinline__ void word_loads_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// Where a worker stands in the line of tiles.
struct Cursor {
  int32_t b, h, rt, tile, tiles;
};
__device__ __forceinline__ void advance(const CachedParams& p, Cursor& c) {
  if (++c.tile < c.tiles) return;
  c.tile = 0;
  if (++c.rt < p.row_tiles) return;
  c.rt = 0;
  if (++c.h < p.cache.heads) return;
  c.h = 0;
  do {
    ++c.b;
    c.tiles = c.b < p.batch ? tiles_of(p, c.b) : 1;  // behind the last one: never used
  } while (c.tiles == 0);
}

template <int D>
struct Ring {
  static constexpr int kWarps = D == 64 ? 12 : 8;  // workers of a CTA, one CTA per SM
  // 4 of up to 131072 positions, heads of 128, 8 warps: 107.5 us with two slots, 116 with three, 128 with four for 6 warps;
  // 10 warps of two: 120.
  static constexpr int kSlots = D == 64 ? 4 : 2;
  // 64 tokens of a head, plus the gap between pages that keeps V's columns on different banks
  static constexpr uint32_t kSlotBytes = kTileTokens * D + 128;
  static constexpr uint32_t kScaleBytes = 4 * 8 * 4;  // of four tiles: four pages' K and V scales
  static constexpr uint32_t kWarpBytes = kSlots * kSlotBytes + kScaleBytes;
  static constexpr size_t kBytes = 128 + kWarps * (kWarpBytes + kSlots * 8) + 16;
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(32 * Ring<D>::kWarps, 1) cached_kernel(const CachedParams p) {
  constexpr bool kSplit = sizeof(T) == 4;
  constexpr int kRows = 8 * NT, kSteps = D / 16, kSlots = Ring<D>::kSlots;
  extern __shared__ uint8_t smem_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quad = lane & 3, octet = lane >> 2;  // fragment coordinates: column pair, row
  uint8_t* base = smem_raw + ((128u - (smem_u32(smem_raw) & 127u)) & 127u);
  uint8_t* ring = base + warp * Ring<D>::kWarpBytes;
  float* scales = reinterpret_cast<float*>(ring + kSlots * Ring<D>::kSlotBytes);
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + Ring<D>::kWarps * Ring<D>::kWarpBytes) + warp * kSlots;
  volatile int* abort_flag = reinterpret_cast<int*>(base + Ring<D>::kWarps * (Ring<D>::kWarpBytes + kSlots * 8));
  const uint32_t ring_addr = smem_u32(ring), scales_addr = smem_u32(scales), bars_addr = smem_u32(bars);
  if (lane == 0) {
    for (int s = 0; s < kSlots; ++s) mbar_init(bars_addr + 8 * s, 33);
    fence_barrier_init();
  }
  if (threadIdx.x == 0) *abort_flag = 0;
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;");  // the joining kernel may come up (it waits for this one's end)

  const Cache& c = p.cache;
  int32_t none_before;
  const int32_t total = count_tiles(p, 0, none_before), each = tiles_per_worker(p, total);
  // neighbouring workers on different SMs: little work spreads over all of them
  const int32_t worker = warp * gridDim.x + blockIdx.x;
  if (worker >= p.workers || static_cast<int64_t>(worker) * each >= total) return;
  const int32_t begin = worker * each, end = static_cast<int32_t>(min(static_cast<int64_t>(begin) + each, static_cast<int64_t>(total)));

  Cursor at;
  {
    const Piece piece = find_piece(p.batch, begin, [&](int32_t b) { return int64_t{tiles_of(p, b)} * c.heads * p.row_tiles; });
    at.b = piece.sequence;
    at.tiles = tiles_of(p, at.b);
    const int32_t index = static_cast<int32_t>(piece.index), pair = index / at.tiles;
    at.tile = index - pair * at.tiles;
    at.h = pair / p.row_tiles;
    at.rt = pair - at.h * p.row_tiles;
  }

  // -------------------------------------------------------------------- copies
  // Item 2u is the K tile of the worker's u-th unit, item 2u + 1 its V tile; item i goes to slot i % kSlots.
  // Items are issued in order; lane i copies the tile's i-th page.
  const int pages_full = kTileTokens >> c.token_bits;
  const uint32_t page_bytes = static_cast<uint32_t>(D) << c.token_bits;
  const uint32_t v_page_step = page_bytes + (c.token_bits == 4 ? 32u : 64u);
  const int32_t items = 2 * (end - begin);
  Cursor ahead = at;
  int32_t next_item = 0;
  uint32_t next_slot = 0;
  const uint64_t policy = read_once_policy();
  int64_t next_pair = 0;     // (block, head) of this lane's page
  bool next_held = false;    // whether a position of it exists
  bool next_there = false;   // and its block does
  auto look_up = [&]() {   // the block of this lane's page of the next unit
    const int64_t page = static_cast<int64_t>(ahead.tile) * pages_full + lane;
    const int64_t held = (static_cast<int64_t>(p.lengths[ahead.b]) + c.tokens - 1) >> c.token_bits;
    next_held = lane < pages_full && page < held;
    const int32_t block = next_held ? p.table.blocks[ahead.b * p.table.stride + page] : -1;
    next_there = block >= 0 && block < c.blocks;
    next_pair = static_cast<int64_t>(block) * c.heads + ahead.h;
  };
  auto issue = [&]() {
    const uint32_t bar = bars_addr + 8 * next_slot;
    const bool is_v = next_item & 1;
    const unsigned copies = __ballot_sync(0xffffffffu, next_there);
    if (lane == 0) mbar_expect_tx(bar, __popc(copies) * page_bytes);
    __syncwarp();
    if (next_there) {
      const uint32_t dst = ring_addr + next_slot * Ring<D>::kSlotBytes + lane * (is_v ? v_page_step : page_bytes);
      bulk_load(dst, (is_v ? c.v_codes : c.k_codes) + next_pair * page_bytes, page_bytes, bar, policy);
    }
    if (!is_v && next_held) {
      const uint32_t dst = scales_addr + (static_cast<uint32_t>(next_item >> 1) & 3u) * 32 + lane * 4;
      word_load(dst, next_there ? c.k_scales + next_pair : &g_not_a_number);
      word_load(dst + 16, next_there ? c.v_scales + next_pair : &g_not_a_number);
      if (!next_there && p.status) atomicOr(p.status, kErrBlocks);
    }
    word_loads_arrive(bar);
    if (++next_slot == kSlots) next_slot = 0;
    if ((++next_item & 1) == 0 && next_item < items) {
      advance(p, ahead);
      look_up();
    }
  };
  look_up();
  for (int i = 0; i < kSlots && next_item < items; ++i) issue();

  // -------------------------------------------------------------------- the work
  uint32_t slot = 0, parity = 0;
  auto arrived = [&]() {
    bool ok = mbar_wait(bars_addr + 8 * slot, parity, abort_flag, p.status, kErrCachedWait);
    return __all_sync(0xffffffffu, ok) != 0;
  };
  auto release = [&]() {
    __syncwarp();
    if (++slot == kSlots) {
      slot = 0;
      parity ^= 1u;
    }
    if (next_item < items) issue();
  };

  uint32_t q_hi[kSteps][NT][2], q_lo[kSplit ? kSteps : 1][kSplit ? NT : 1][2];
  float o[kSteps][NT][4], row_scale[NT][2], top[NT][2], sum[NT][2];
  int64_t limit[NT][2];  // positions that the row sees
  int32_t segment = begin - at.tile;  // where the pair in work began
  bool fresh = true;

  for (int32_t unit = begin; unit < end; ++unit) {
    if (fresh) {
      // Queries of this (sequence, head): row `octet` of each row tile, the 16 consecutive dims per 64 that
      // belong to this quad; scaled by a power of two that brings the row's largest to [1, 2).
      fresh = false;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int row = at.rt * kRows + n * 8 + octet;
        float x[D / 4];
        uint32_t largest = 0;
        const bool real = row < p.rows;
        const int token = row / p.group, head = at.h * p.group + row % p.group;
        const T* src = static_cast<const T*>(p.q) + at.b * p.q_batch + token * p.q_token + head * p.q_head;
        constexpr int kVec = Elem<T>::kVec;
        if (real && p.q_vectors) {
#pragma unroll
          for (int i = 0; i < D / 4; i += kVec) {
            float part[kVec];
            unpack16(ld_plain16(src + (i / 16) * 64 + quad * 16 + i % 16), part);
#pragma unroll
            for (int e = 0; e < kVec; ++e) x[i + e] = part[e];
          }
        } else {
#pragma unroll
          for (int i = 0; i < D / 4; ++i) x[i] = real ? Elem<T>::load(src + (i / 16) * 64 + quad * 16 + i % 16) : 0.f;
        }
#pragma unroll
        for (int i = 0; i < D / 4; ++i) largest = max(largest, __float_as_uint(x[i]) & 0x7fffffffu);
        largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
        largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
        const uint32_t power = min(max(largest & 0x7f800000u, 27u << 23), 253u << 23);
        const float down = __uint_as_float((254u << 23) - power) * p.q_sign;
        float up = __uint_as_float(power) * p.scale_log2;
        if (largest >= 0x7f800000u) up = __uint_as_float(0x7fc00000u);
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float lo = x[4 * s + 2 * e] * down, hi = x[4 * s + 2 * e + 1] * down;
            q_hi[s][n][e] = half2_bits(lo, hi);
            if (kSplit) q_lo[s][n][e] = half2_rest(lo, hi, q_hi[s][n][e]);
          }
        const int64_t length = p.lengths[at.b];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          row_scale[n][e] = __shfl_sync(0xffffffffu, up, (2 * quad + e) * 4);
          limit[n][e] = length - p.tokens + 1 + (at.rt * kRows + n * 8 + 2 * quad + e) / p.group;
          top[n][e] = -INFINITY;
          sum[n][e] = 0.f;
        }
      }
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[s][n][i] = 0.f;
    }

    // S^T = K Q^T. Row r of 16-row tile m is token 16 (r % 8 / 2) + 4 m + 2 (r / 8) + r % 2: what a thread
    // gets of a row is then, transposed, the four consecutive tokens that its bytes of V hold.
    if (!arrived()) break;
    const float* tile_scales = scales + (static_cast<uint32_t>(unit - begin) & 3u) * 8;
    const int page = (octet >> 1) >> (c.token_bits - 4);
    const float k_scale = tile_scales[page];
    const float v_raw = tile_scales[4 + page], v_scale = v_raw < kSmallestScale ? kSmallestScale : v_raw;
    float s[4][NT][4];
    {
      const uint8_t* tile = ring + slot * Ring<D>::kSlotBytes + (16 * (octet >> 1) + (octet & 1)) * D + quad * 16;
#pragma unroll
      for (int m = 0; m < 4; ++m) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[m][n][i] = 0.f;
#pragma unroll
        for (int half = 0; half < D / 64; ++half) {
          const uint4 first = *reinterpret_cast<const uint4*>(tile + 4 * m * D + half * 64);
          const uint4 second = *reinterpret_cast<const uint4*>(tile + (4 * m + 2) * D + half * 64);
          const uint32_t w0[4] = {first.x, first.y, first.z, first.w}, w1[4] = {second.x, second.y, second.z, second.w};
          float fresh[kSplit ? 2 : 1][NT][4] = {};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t a[4];
            codes_to_half(w0[i], a[0], a[2]);
            codes_to_half(w1[i], a[1], a[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma_f16(kSplit ? fresh[0][n] : s[m][n], a, q_hi[half * 4 + i][n][0], q_hi[half * 4 + i][n][1]);
              if (kSplit) mma_f16(fresh[kSplit][n], a, q_lo[half * 4 + i][n][0], q_lo[half * 4 + i][n][1]);
            }
          }
          if (kSplit) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) s[m][n][i] += fresh[0][n][i] + fresh[kSplit][n][i];
          }
        }
      }
    }
    release();

    // Softmax: this thread has 8 tokens of two rows for each row tile. With t = score + log2(v_scale), as long as no t is more
    // than kStale above the row's `top`, nothing has to be agreed on between the threads of a row.
    const bool cut = (at.tile + int64_t{1}) * kTileTokens > static_cast<int64_t>(p.lengths[at.b]) - p.tokens + 1;
    float factor[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) factor[n][e] = row_scale[n][e] * k_scale;
    if (cut) {
      const int64_t first_token = static_cast<int64_t>(at.tile) * kTileTokens + 16 * (octet >> 1) + (octet & 1);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int64_t seen = limit[n][e] - first_token;
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float& x = s[m][n][2 * h + e];
              x = 4 * m + 2 * h < seen ? x * factor[n][e] : -INFINITY;  // (a masked position's scale may be anything)
            }
          factor[n][e] = 1.f;
        }
    }
    const float v_log = __log2f(v_scale);
    float best[NT][2];
    bool higher = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = s[0][n][e];
#pragma unroll
        for (int i = 1; i < 8; ++i) x = fmaxf(x, s[i >> 1][n][2 * (i & 1) + e]);
        best[n][e] = fmaf(x, factor[n][e], v_log);
        higher |= best[n][e] > top[n][e] + kStale;
      }
    if (__any_sync(0xffffffffu, higher)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float now = fmaxf(best[n][e], top[n][e]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, d));
          const float keep = now == -INFINITY ? 1.f : fast_exp2(top[n][e] - now);
          top[n][e] = now;
          sum[n][e] *= keep;
#pragma unroll
          for (int i = 0; i < kSteps; ++i) {
            o[i][n][e] *= keep;
            o[i][n][2 + e] *= keep;
          }
        }
    }
    uint32_t p_hi[4][NT][2], p_lo[kSplit ? 4 : 1][kSplit ? NT : 1][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float shift = kHeadroom - (top[n][e] == -INFINITY ? 0.f : top[n][e]);
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float& x = s[m][n][2 * h + e];
            const bool masked = cut && x == -INFINITY;
            x = fast_exp2(fmaf(x, factor[n][e], shift));
            sum[n][e] += x;
            x = masked ? 0.f : x * v_scale;
          }
      }
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t pair = half2_bits(s[m][n][2 * h], s[m][n][2 * h + 1]);
          p_hi[m][n][h] = transpose_8x8(pair);
          if (kSplit) p_lo[m][n][h] = transpose_8x8(half2_rest(s[m][n][2 * h], s[m][n][2 * h + 1], pair));
        }
    }

    // O^T += V^T P^T: a thread's 16 bytes of a channel are 16 tokens, four for each of the four products.
    if (!arrived()) break;
    {
      const int in_page = quad & ((1 << (c.token_bits - 4)) - 1);
      const uint8_t* tile = ring + slot * Ring<D>::kSlotBytes + (quad >> (c.token_bits - 4)) * v_page_step + in_page * 16;
#pragma unroll
      for (int d = 0; d < kSteps; ++d) {
        const uint4 first = *reinterpret_cast<const uint4*>(tile + ((16 * d + octet) << c.token_bits));
        const uint4 second = *reinterpret_cast<const uint4*>(tile + ((16 * d + octet + 8) << c.token_bits));
        const uint32_t w0[4] = {first.x, first.y, first.z, first.w}, w1[4] = {second.x, second.y, second.z, second.w};
        float fresh[kSplit ? 2 : 1][NT][4] = {};
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          uint32_t a[4];
          codes_to_half(w0[m], a[0], a[2]);
          codes_to_half(w1[m], a[1], a[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_f16(kSplit ? fresh[0][n] : o[d][n], a, p_hi[m][n][0], p_hi[m][n][1]);
            if (kSplit) mma_f16(fresh[kSplit][n], a, p_lo[m][n][0], p_lo[m][n][1]);
          }
        }
        if (kSplit) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[d][n][i] += fresh[0][n][i] + fresh[kSplit][n][i];
        }
      }
    }
    release();

    if (at.tile + 1 == at.tiles || unit + 1 == end) {
      const bool whole = segment >= begin && at.tile + 1 == at.tiles;
      float* left = partial_of<kRows, D>(p, worker, segment >= begin ? 1 : 0);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float l = sum[n][e];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
          const int in_tile = n * 8 + 2 * quad + e, row = at.rt * kRows + in_tile;
          if (row >= p.rows) continue;
          if (whole) {
            const float inv = limit[n][e] <= 0 ? 0.f : 1.f / l;
            const int token = row / p.group, head = at.h * p.group + row % p.group;
            T* dst = static_cast<T*>(p.out) + ((static_cast<int64_t>(at.b) * p.tokens + token) * p.heads + head) * D;
#pragma unroll
            for (int d = 0; d < kSteps; ++d) {
              Elem<T>::store(dst + 16 * d + octet, o[d][n][e] * inv);
              Elem<T>::store(dst + 16 * d + octet + 8, o[d][n][2 + e] * inv);
            }
          } else {
            if (octet == 0) {
              left[in_tile] = top[n][e];
              left[kRows + in_tile] = l;
            }
            float* dst = left + 2 * kRows + in_tile * D;
#pragma unroll
            for (int d = 0; d < kSteps; ++d) {
              dst[16 * d + octet] = o[d][n][e];
              dst[16 * d + octet + 8] = o[d][n][2 + e];
            }
          }
        }
      fresh = true;
      segment = unit + 1;
    }
    if (unit + 1 < end) advance(p, at);
  }
  if (*abort_flag) {
    // A wait ran out: copies of this warp may still be in flight; give them (bounded) time to land.
    const unsigned long long start = global_ns();
    while (global_ns() - start < 2000000ull) {
    }
  }
}

// Joins what several workers left of a row: out = sum_w 2^(m_w - m) O_w / sum_w 2^(m_w - m) l_w, the workers in order. A CTA's
// eight warps take eight rows of one (sequence, head, row tile), or, where there are few of those (SPLIT 8), one row: each an
// eighth of the workers, added in order. It comes up while the first kernel runs and waits for its end before it reads.
template <typename T, int D, int NT, int SPLIT>
__global__ void __launch_bounds__(256) cached_join_kernel(const CachedParams p) {
  constexpr int kRows = 8 * NT, kPer = D / 32, kStride = kRows * (2 + D);
  __shared__ float best_of[8], sum_of[8], acc_of[SPLIT > 1 ? 8 : 1][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = SPLIT > 1 ? warp : 0, in_tile = SPLIT > 1 ? blockIdx.y : blockIdx.y * 8 + warp;
  const int32_t pairs = p.cache.heads * p.row_tiles;
  const int32_t b = blockIdx.x / pairs, pair = blockIdx.x - b * pairs;
  const int32_t h = pair / p.row_tiles, rt = pair - h * p.row_tiles;
  const int row = rt * kRows + in_tile;
  const int token = row / p.group;
  const int64_t length = p.lengths[b], limit = length - p.tokens + 1 + token;
  const int32_t tiles = tiles_of(p, b);
  int32_t before, first = 0, last = 0;
  const int32_t total = count_tiles(p, b, before);
  if (tiles > 0) {
    const int32_t each = tiles_per_worker(p, total), start = before + pair * tiles;
    first = start / each;
    last = (start + tiles - 1) / each;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (row >= p.rows || (tiles > 0 && first == last)) return;  // no such row, or finished by its worker (CTA-wide if SPLIT)
  T* dst = static_cast<T*>(p.out) + ((static_cast<int64_t>(b) * p.tokens + token) * p.heads + h * p.group + row % p.group) * D;
  if (tiles == 0) {
    const bool beyond = length > 0;
    if (beyond && lane == 0 && p.status) atomicOr(p.status, kErrBlocks);
    if (split == 0)
      for (int i = lane; i < D; i += 32) Elem<T>::store(dst + i, beyond ? __uint_as_float(0x7fc00000u) : 0.f);
    return;
  }
  const float* left = partial_of<kRows, D>(p, first, 1) + in_tile;  // of the first worker; the others' in slot 0
  auto left_by = [&](int32_t w) { return left + static_cast<int64_t>((w - first) * 2 - (w > first)) * kStride; };
  const int32_t count = last - first + 1;
  const int32_t from = count * split / SPLIT, to = count * (split + 1) / SPLIT;  // this warp's
  float best = -INFINITY;
  for (int32_t i = from + lane; i < to; i += 32) best = fmaxf(best, *left_by(first + i));
  best = warp_fmax(best);
  if (SPLIT > 1) {
    if (lane == 0) best_of[warp] = best;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) best = fmaxf(best, best_of[i]);
  }
  if (best == -INFINITY) best = 0.f;
  float sum = 0.f, acc[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) acc[i] = 0.f;
  for (int32_t base = from; base < to; base += 32) {
    float weight = 0.f;
    if (base + lane < to) {
      const float* mine = left_by(first + base + lane);
      weight = fast_exp2(mine[0] - best);
      sum = fmaf(mine[kRows], weight, sum);
    }
    const int here = min(32, to - base);
#pragma unroll 8
    for (int i = 0; i < here; ++i) {
      const float w = __shfl_sync(0xffffffffu, weight, i);
      const float* x = left_by(first + base + i) - in_tile + 2 * kRows + in_tile * D + lane * kPer;
#pragma unroll
      for (int e = 0; e < kPer; ++e) acc[e] = fmaf(x[e], w, acc[e]);
    }
  }
  sum = warp_sum(sum);
  if (SPLIT > 1) {
    if (lane == 0) sum_of[warp] = sum;
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc_of[warp][lane * kPer + i] = acc[i];
    __syncthreads();
    if (warp > 0) return;
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      sum += sum_of[w];
#pragma unroll
      for (int i = 0; i < kPer; ++i) acc[i] += acc_of[w][lane * kPer + i];
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) Elem<T>::store(dst + lane * kPer + i, limit <= 0 ? 0.f : acc[i] / sum);
}

// Query rows of a tile: 8, or 16 where a (sequence, head) has more than 8 (32 would not leave room in
// the registers for the accumulators beside the queries).
int row_tile(int64_t rows) { return rows <= 8 ? 8 : 16; }

struct CachedPlan {
  int64_t rows, row_tiles, pairs, most, workers;  // most: tiles, if every sequence filled its table
  int tile, grid;
};
CachedPlan plan_cached(const b200_cached_attention_desc& d, int sms) {
  CachedPlan plan{};
  plan.rows = d.tokens * (d.heads / d.cache.heads);
  plan.tile = row_tile(plan.rows);
  plan.row_tiles = ceil_div(plan.rows, plan.tile);
  plan.pairs = d.batch * d.cache.heads * plan.row_tiles;
  // no more workers than the longest possible sequences have tiles
  const int warps = d.cache.dim == 64 ? Ring<64>::kWarps : Ring<128>::kWarps;
  const int64_t most = plan.most = plan.pairs * (ceil_div(d.table_width * d.cache.block_tokens, kTileTokens) + 1);
  plan.grid = static_cast<int>(most < sms ? most : sms);
  plan.workers = most < static_cast<int64_t>(plan.grid) * warps ? most : static_cast<int64_t>(plan.grid) * warps;
  return plan;
}

std::once_flag g_cached_attr_once[64];

// The joining kernel as a programmatic dependent of the first: launched and set up while that one runs.
template <typename T, int D, int NT, int SPLIT>
cudaError_t launch_join(const CachedParams& p, const CachedPlan& plan, cudaStream_t s) {
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(plan.pairs), SPLIT > 1 ? 8 * NT : NT);
  config.blockDim = dim3(256);
  config.stream = s;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, cached_join_kernel<T, D, NT, SPLIT>, p);
}

template <typename T, int D, int NT>
int launch_cached(const CachedParams& p, const CachedPlan& plan, int sms, cudaStream_t s) {
  cached_kernel<T, D, NT><<<plan.grid, 32 * Ring<D>::kWarps, Ring<D>::kBytes, s>>>(p);
  const int code = check_launch();
  if (code) return finish(code);
  // A row has about workers / pairs partial results. With few pairs one warp would go over many of them.
  const cudaError_t err = plan.pairs >= 2 * sms ? launch_join<T, D, NT, 1>(p, plan, s) : launch_join<T, D, NT, 8>(p, plan, s);
  if (err != cudaSuccess) cudaGetLastError();
  return err == cudaSuccess ? launched() : finish(-static_cast<int>(err));
}
template <typename T>
void cached_attributes() {
  cudaFuncSetAttribute(cached_kernel<T, 64, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Ring<64>::kBytes));
  cudaFuncSetAttribute(cached_kernel<T, 64, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Ring<64>::kBytes));
  cudaFuncSetAttribute(cached_kernel<T, 128, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Ring<128>::kBytes));
  cudaFuncSetAttribute(cached_kernel<T, 128, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Ring<128>::kBytes));
}
template <typename T>
int launch_cached_any(const CachedParams& p, const CachedPlan& plan, int dim, int sms, cudaStream_t s) {
  if (dim == 64) return plan.tile == 8 ? launch_cached<T, 64, 1>(p, plan, sms, s) : launch_cached<T, 64, 2>(p, plan, sms, s);
  return plan.tile == 8 ? launch_cached<T, 128, 1>(p, plan, sms, s) : launch_cached<T, 128, 2>(p, plan, sms, s);
}

}  // namespace
}  // namespace b200

using namespace b200;

static size_t workspace_for(const CachedPlan& plan, int dim) {
  return static_cast<size_t>(plan.workers) * 2 * plan.tile * (2 + dim) * sizeof(float);
}

extern "C" int64_t b200_attention_cached_workspace_bytes(const b200_cached_attention_desc* desc) {
  if (!desc) return 0;
  const b200_cached_attention_desc& d = *desc;
  if (!valid_cache(&d.cache) || d.batch < 1 || d.tokens < 1 || d.heads < 1 || d.heads % d.cache.heads || d.table_width < 0 ||
      d.table_width > INT32_MAX)
    return 0;
  return static_cast<int64_t>(workspace_for(plan_cached(d, device_info().sm_count), d.cache.dim));
}

extern "C" int b200_attention_cached(const b200_cached_attention_desc* desc, void* stream) {
  if (!enabled()) return refuse(B200_E_DISABLED);
  if (!desc) return refuse(B200_E_NULL);
  const b200_cached_attention_desc& d = *desc;
  if (!valid_dtype(d.dtype)) return refuse(B200_E_DTYPE);
  if (!valid_cache(&d.cache) || d.batch < 0 || d.tokens < 0 || d.heads < 1 || d.heads % d.cache.heads ||
      d.batch > INT32_MAX / 8 || d.tokens > INT32_MAX / 8 || d.heads > INT32_MAX / 8)
    return refuse(B200_E_SHAPE);
  if (!(fabsf(d.scale) <= 3.0e38f)) return refuse(B200_E_ARG);
  if (d.batch == 0 || d.tokens == 0) return finish(0);
  if (!cache_pointers(&d.cache) || !d.q || !d.out || !d.lengths || (d.table_width > 0 && !d.block_table))
    return refuse(B200_E_NULL);
  if (d.table_width < 0 || d.table_width > INT32_MAX || (d.batch > 1 && d.table_stride < d.table_width))
    return refuse(B200_E_STRIDE);
  if (!cache_aligned(&d.cache) || !aligned(d.q, dtype_size(d.dtype)) || !aligned(d.out, dtype_size(d.dtype)) ||
      !aligned(d.block_table, 4) || !aligned(d.lengths, 4))
    return refuse(B200_E_ALIGN);
  const DeviceInfo& dev = device_info();
  if (dev.sm_count == 0) return refuse(B200_E_DEVICE);
  const CachedPlan plan = plan_cached(d, dev.sm_count);
  if (plan.rows > INT32_MAX / 2 || plan.pairs > INT32_MAX || plan.most > INT32_MAX) return refuse(B200_E_SHAPE);
  if (!d.workspace || d.workspace_bytes < static_cast<int64_t>(workspace_for(plan, d.cache.dim)) || !aligned(d.workspace, 16))
    return refuse(B200_E_WORKSPACE);
  CachedParams p{};
  p.cache = device_cache(&d.cache);
  p.table = Table{d.block_table, d.table_stride, static_cast<int32_t>(d.table_width)};
  p.q = d.q;
  p.out = d.out;
  p.q_batch = d.q_batch;
  p.q_token = d.q_token;
  p.q_head = d.q_head;
  p.lengths = d.lengths;
  p.batch = static_cast<int32_t>(d.batch);
  p.tokens = static_cast<int32_t>(d.tokens);
  p.heads = static_cast<int32_t>(d.heads);
  p.group = static_cast<int32_t>(d.heads / d.cache.heads);
  p.rows = static_cast<int32_t>(plan.rows);
  p.row_tiles = static_cast<int32_t>(plan.row_tiles);
  p.workers = static_cast<int32_t>(plan.workers);
  const int64_t vec = d.dtype == B200_F32 ? 4 : 8;
  p.q_vectors = aligned(d.q, 16) && d.q_batch % vec == 0 && d.q_token % vec == 0 && d.q_head % vec == 0;
  p.scale_log2 = d.scale == 0.f ? 1.f : fabsf(d.scale) * kLog2e;
  p.q_sign = d.scale == 0.f ? 0.f : (d.scale < 0.f ? -1.f : 1.f);
  p.partial = static_cast<float*>(d.workspace);
  p.status = kernel_status_word();
  std::call_once(g_cached_attr_once[dev.device], [] {
    cached_attributes<float>();
    cached_attributes<__nv_bfloat16>();
  });
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return d.dtype == B200_F32 ? launch_cached_any<float>(p, plan, d.cache.dim, dev.sm_count, s)
                             : launch_cached_any<__nv_bfloat16>(p, plan, d.cache.dim, dev.sm_count, s);
}
