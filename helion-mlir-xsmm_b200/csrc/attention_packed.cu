// Prompt attention over packed sequences: out_i = sum_j softmax_j(scale q_i . k_j) v_j for
// query row i of a sequence over that sequence's keys, causal or not, query head h reading
// key/value head h / (heads / kv_heads). q, out: [rows_q][heads][dim], k, v:
// [rows_k][kv_heads][dim], any row and head strides; sequence b owns the rows
// [offsets[b], offsets[b + 1]). Causal: the queries are the last positions of the keys, so
// row i sees keys j <= i + keys - queries. A row that sees no key is zeros, and so are the
// rows behind the last sequence. No reference counterpart.
#include <cuda.h>
#include <math.h>

#include <mutex>

#include "sequences.cuh"
#include "umma_ptx.cuh"

namespace b200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct PackedParams {
  const void *q, *k, *v;
  void* out;  // [rows_q][heads][dim], contiguous
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // strides in elements
  int64_t rows_q, rows_k;
  const int32_t *offsets, *k_offsets;
  int32_t batch, heads, group, dim;  // group: query heads that share a key/value head
  int32_t causal;
  int32_t vectors;   // rows can be read four values at a time
  float scale_log2;  // scale * log2(e)
  int32_t* status;
};

// ------------------------------------------------------------------------- any type, any head size
// Values that a row does not see must not reach it, but the tensor core multiplies them by P = 0, and 0 * infinity is NaN. So
// a row whose result is not finite looks whether a value that is not finite lies among the keys that were read and not
// seen ([sees, read)), and one thread computes its columns [from, to) again if so (`always`: in any case).
template <typename T>
__device__ __forceinline__ void packed_row_again(const PackedParams& p, const T* q, const T* k, const T* v, int64_t sees, int64_t read,
                                                 bool always, int from, int to, T* dst) {
  bool touched = always;
  for (int64_t j = sees; j < read && !touched; ++j)
    for (int d = from; d < to; ++d) touched |= !isfinite(Elem<T>::load(v + j * p.v_row + d));
  if (!touched) return;  // the row itself is not finite
#pragma unroll 1
  for (int chunk = from; chunk < to; chunk += 32) {
    float acc[32], top = -INFINITY, total = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) acc[i] = 0.f;
#pragma unroll 1
    for (int64_t j = 0; j < sees; ++j) {
      float s = 0.f;
#pragma unroll 4
      for (int d = 0; d < p.dim; ++d) s = fmaf(Elem<T>::load(q + d), Elem<T>::load(k + j * p.k_row + d), s);
      s *= p.scale_log2;
      const float best = fmaxf(top, s), base = best == -INFINITY ? 0.f : best;
      const float keep = fast_exp2(top - base), weight = fast_exp2(s - base);
      top = best;
      total = fmaf(total, keep, weight);
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (chunk + i < to) acc[i] = fmaf(weight, Elem<T>::load(v + j * p.v_row + chunk + i), acc[i] * keep);
    }
    const float inv = 1.f / total;
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (chunk + i < to) Elem<T>::store(dst + chunk + i, acc[i] * inv);
  }
}

// One CTA takes 64 query rows of one head and goes over the keys in tiles, with the running maximum and sum of the
// softmax in f32. Eight warps: four runs of 16 rows, two halves of each tile's keys, joined at the end. The products are
// mma m16n8k16 on bf16 pieces: an f32 value is the sum of three (8 bits each, the exponent range of f32, so nothing
// has to be scaled), and a product the six of their products that reach 2^-27; Q, K, V and P alike. That is f32's own
// accuracy at six instructions; FFMA tiles of 64 x 64 stood still on shared memory at a third of FFMA's rate. Five sequences of
// 300, 6 heads of 80, f32: 60 us and 84 with FFMA; one of 4096, 8 heads of 64: 547 and 775. What bounds it: mma.sync, and the loads
// of a tile, which nothing covers but the other CTA of the SM. bf16 values are one piece (2048 rows, 16/4 heads of 80: 201 us).
constexpr int kTile = 64, kMmaThreads = 256;

template <typename T, int DP>
struct MmaTile {
  static constexpr int kPieces = sizeof(T) == 4 ? 3 : 1;
  static constexpr int kKeys = sizeof(T) == 4 && DP > 128 ? 32 : 64;  // of a tile: as many as leave room in shared memory
  static constexpr int kStep = DP + 8;  // of a row: the 16-byte pieces of eight rows on different banks
  static constexpr uint32_t kQPiece = kTile * kStep, kKeyPiece = kKeys * kStep;  // elements
  static constexpr size_t kTiles = kPieces * (kQPiece + 2 * kKeyPiece) * 2;
  static constexpr size_t kJoin = 4 * 32 * (DP / 2 + 4) * 4;  // what four warps hand over at the end
  static constexpr size_t kBytes = kTiles > kJoin ? kTiles : kJoin;
};

__device__ __forceinline__ void ldmatrix(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two values as PIECES bf16 pairs, each what the ones before leave over, rounded to the nearest: the second is at most 2^-9 of the
// value, the third 2^-18 (of either sign: the products that are left out do not add up). An infinity, or a value that rounds to one,
// leaves NaN over.
template <int PIECES>
__device__ __forceinline__ void to_pieces(float lo, float hi, uint32_t (&piece)[PIECES]) {
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    piece[i] = pack_bf16x2(lo, hi);
    if (i + 1 < PIECES) {
      lo -= __uint_as_float(piece[i] << 16);
      hi -= __uint_as_float(piece[i] & 0xffff0000u);
    }
  }
}

// `rows` rows of `dim` values as pieces into shared memory; rows from `count` on and channels from dim on are zeros, whatever
// lies there.
template <typename T, int DP>
__device__ __forceinline__ void mma_load(__nv_bfloat16* dst, uint32_t piece_step, const T* src, int64_t row_step, int rows, int count,
                                         int dim, bool vectors) {
  using Tile = MmaTile<T, DP>;
#pragma unroll 4
  for (int i = threadIdx.x; i < rows * (DP / 4); i += kMmaThreads) {
    const int r = i / (DP / 4), d = i % (DP / 4) * 4;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (r < count && d < dim) {
      const T* at = src + r * row_step + d;
      if (vectors) {  // dim is a multiple of four then
        if (sizeof(T) == 4) {
          unpack16(ld_plain16(at), x);
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(at);
          x[0] = __uint_as_float(w.x << 16);
          x[1] = __uint_as_float(w.x & 0xffff0000u);
          x[2] = __uint_as_float(w.y << 16);
          x[3] = __uint_as_float(w.y & 0xffff0000u);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d + e < dim) x[e] = Elem<T>::load(at + e);
      }
    }
    uint32_t lo[Tile::kPieces], hi[Tile::kPieces];
    to_pieces<Tile::kPieces>(x[0], x[1], lo);
    to_pieces<Tile::kPieces>(x[2], x[3], hi);
#pragma unroll
    for (int e = 0; e < Tile::kPieces; ++e)
      *reinterpret_cast<uint2*>(dst + e * piece_step + r * Tile::kStep + d) = make_uint2(lo[e], hi[e]);
  }
}

template <typename T, int DP>
__global__ void __launch_bounds__(kMmaThreads, DP <= 96 || (sizeof(T) == 2 && DP <= 128) ? 2 : 1)
    packed_mma_kernel(const PackedParams p) {
  using Tile = MmaTile<T, DP>;
  constexpr int kPieces = Tile::kPieces, kKeys = Tile::kKeys, kStep = Tile::kStep;
  constexpr int kMine = kKeys / 2;  // keys of a tile that a warp takes
  constexpr int kRun = kPieces > 1 ? 32 : DP;  // channels between two additions to the scores
  extern __shared__ __align__(16) uint8_t smem_raw[];
  __nv_bfloat16* qs = reinterpret_cast<__nv_bfloat16*>(smem_raw);
  __nv_bfloat16* ks = qs + kPieces * Tile::kQPiece;
  __nv_bfloat16* vs = ks + kPieces * Tile::kKeyPiece;

  const int head = blockIdx.y, dim = p.dim;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Tiles with many keys first (causal): a long sequence's last rows would otherwise start last.
  const Piece piece = find_piece(p.batch, static_cast<int64_t>(gridDim.x) - 1 - blockIdx.x, [&](int32_t b) {
    return (rows_of(p.offsets, b, p.rows_q, p.status).count + kTile - 1) / kTile;
  });
  T* out = static_cast<T*>(p.out);
  if (piece.sequence < 0) {
    const Rows rest = rows_behind(p.offsets, p.batch, p.rows_q);
    const int64_t first = piece.index * kTile;
    for (int r = warp; r < kTile && first + r < rest.count; r += 8)
      for (int d = lane; d < dim; d += 32) Elem<T>::store(out + ((rest.begin + first + r) * p.heads + head) * dim + d, 0.f);
    return;
  }
  const Rows mine = rows_of(p.offsets, piece.sequence, p.rows_q, nullptr);
  const Rows theirs = rows_of(p.k_offsets, piece.sequence, p.rows_k, p.status);
  const int64_t row0 = piece.index * kTile;
  const int rows = static_cast<int>(mine.count - row0 < kTile ? mine.count - row0 : kTile);
  const int64_t shift = p.causal ? theirs.count - mine.count + 1 : 0;  // row i sees the keys below i + shift
  int64_t keys = theirs.count;
  if (p.causal && row0 + rows - 1 + shift < keys) keys = row0 + rows - 1 + shift;

  const T* q = static_cast<const T*>(p.q) + (mine.begin + row0) * p.q_row + head * p.q_head;
  const int kv_head = head / p.group;
  const T* k = static_cast<const T*>(p.k) + theirs.begin * p.k_row + kv_head * p.k_head;
  const T* v = static_cast<const T*>(p.v) + theirs.begin * p.v_row + kv_head * p.v_head;
  mma_load<T, DP>(qs, Tile::kQPiece, q, p.q_row, kTile, rows, dim, p.vectors);

  const int run = warp & 3, half = warp >> 2, quad = lane & 3, octet = lane >> 2;
  const uint32_t q_addr = smem_u32(qs + (run * 16 + (lane & 15)) * kStep + (lane >> 4) * 8);
  const uint32_t k_addr = smem_u32(ks + (half * kMine + (lane & 7) + (lane >> 4) * 8) * kStep + ((lane >> 3) & 1) * 8);
  const uint32_t v_addr = smem_u32(vs + (half * kMine + (lane & 15)) * kStep + (lane >> 4) * 8);
  int64_t sees[2];  // keys that this thread's two rows see
  float top[2], total[2], o[DP / 8][4];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int64_t row = row0 + run * 16 + octet + 8 * e;
    sees[e] = p.causal ? min(max(row + shift, int64_t{0}), theirs.count) : theirs.count;
    top[e] = -INFINITY;
    total[e] = 0.f;
  }
#pragma unroll
  for (int n = 0; n < DP / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[n][i] = 0.f;

  for (int64_t key0 = 0; key0 < keys; key0 += kKeys) {
    const int here = static_cast<int>(keys - key0 < kKeys ? keys - key0 : kKeys);
    __syncthreads();  // the last tile has been read
    mma_load<T, DP>(ks, Tile::kKeyPiece, k + key0 * p.k_row, p.k_row, kKeys, here, dim, p.vectors);
    mma_load<T, DP>(vs, Tile::kKeyPiece, v + key0 * p.v_row, p.v_row, kKeys, here, dim, p.vectors);
    __syncthreads();
    float s[kMine / 8][4];
#pragma unroll
    for (int n = 0; n < kMine / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] = 0.f;
    // The tensor core cuts its sums off where f32 rounds them, always towards zero: f32 products of pieces go into fresh
    // accumulators every 32 channels, the leading one apart from the others, and are added up by the FMA pipe.
#pragma unroll 1
    for (int d0 = 0; d0 < DP; d0 += kRun) {
      float lead[kMine / 8][4], rest[kMine / 8][4];
#pragma unroll
      for (int n = 0; n < kMine / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) lead[n][i] = rest[n][i] = 0.f;
#pragma unroll
      for (int d = d0; d < d0 + kRun; d += 16) {
        if (DP % kRun && d >= DP) break;
        uint32_t a[kPieces][4];
#pragma unroll
        for (int x = 0; x < kPieces; ++x) ldmatrix(a[x], q_addr + (x * Tile::kQPiece + d) * 2);
#pragma unroll
        for (int n = 0; n < kMine / 8; n += 2)
#pragma unroll
          for (int y = 0; y < kPieces; ++y) {
            uint32_t b[4];
            ldmatrix(b, k_addr + (y * Tile::kKeyPiece + n * 8 * kStep + d) * 2);
#pragma unroll
            for (int x = 0; x + y < kPieces; ++x) {
              mma_bf16(x + y ? rest[n] : lead[n], a[x], b[0], b[1]);
              mma_bf16(x + y ? rest[n + 1] : lead[n + 1], a[x], b[2], b[3]);
            }
          }
      }
#pragma unroll
      for (int n = 0; n < kMine / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i] += kPieces > 1 ? lead[n][i] + rest[n][i] : lead[n][i];
    }
    // Softmax of two rows, 2 * kMine / 8 keys each in this thread.
    float best[2] = {-INFINITY, -INFINITY}, kept[2];
    const int64_t first_key = key0 + half * kMine + 2 * quad;
    const int seen[2] = {static_cast<int>(min(sees[0] - first_key, int64_t{kKeys})),
                         static_cast<int>(min(sees[1] - first_key, int64_t{kKeys}))};
#pragma unroll
    for (int n = 0; n < kMine / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[n][i] = n * 8 + (i & 1) < seen[i >> 1] ? s[n][i] * p.scale_log2 : -INFINITY;
        best[i >> 1] = fmaxf(best[i >> 1], s[n][i]);
      }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      best[e] = fmaxf(best[e], __shfl_xor_sync(0xffffffffu, best[e], 1));
      best[e] = fmaxf(fmaxf(best[e], __shfl_xor_sync(0xffffffffu, best[e], 2)), top[e]);
      const float base = best[e] == -INFINITY ? 0.f : best[e];  // nothing seen yet: every term is 2^-inf
      const float keep = fast_exp2(top[e] - base);
      top[e] = best[e];
      total[e] *= keep;
      kept[e] = keep;
#pragma unroll
      for (int n = 0; n < kMine / 8; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          s[n][2 * e + i] = fast_exp2(s[n][2 * e + i] - base);
          total[e] += s[n][2 * e + i];
        }
    }
    uint32_t a[kMine / 16][kPieces][4];
#pragma unroll
    for (int key = 0; key < kMine; key += 16)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t pieces[kPieces];
        to_pieces<kPieces>(s[key / 8 + i / 2][2 * (i & 1)], s[key / 8 + i / 2][2 * (i & 1) + 1], pieces);
#pragma unroll
        for (int x = 0; x < kPieces; ++x) a[key / 16][x][i] = pieces[x];
      }
#pragma unroll
    for (int n = 0; n < DP / 8; n += 2) {
      float lead[2][4] = {}, rest[2][4] = {};  // of this tile
#pragma unroll
      for (int key = 0; key < kMine; key += 16)
#pragma unroll
        for (int y = 0; y < kPieces; ++y) {
          uint32_t b[4];
          ldmatrix_trans(b, v_addr + (y * Tile::kKeyPiece + key * kStep + n * 8) * 2);
#pragma unroll
          for (int x = 0; x + y < kPieces; ++x) {
            mma_bf16(x + y ? rest[0] : lead[0], a[key / 16][x], b[0], b[1]);
            mma_bf16(x + y ? rest[1] : lead[1], a[key / 16][x], b[2], b[3]);
          }
        }
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          o[n + m][i] = fmaf(o[n + m][i], kept[i >> 1], kPieces > 1 ? lead[m][i] + rest[m][i] : lead[m][i]);
    }
  }
  // The halves of the keys are joined: those of the second hand over maximum, sum and accumulator.
  __syncthreads();
  float* left = reinterpret_cast<float*>(smem_raw) + (run * 32 + lane) * (DP / 2 + 4);
  if (half == 1) {
#pragma unroll
    for (int n = 0; n < DP / 8; ++n) *reinterpret_cast<float4*>(left + 4 * n) = make_float4(o[n][0], o[n][1], o[n][2], o[n][3]);
    *reinterpret_cast<float4*>(left + DP / 2) = make_float4(top[0], top[1], total[0], total[1]);
  }
  __syncthreads();
  if (half == 1) return;
  float mine_by[2], theirs_by[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const float their_top = left[DP / 2 + e], best = fmaxf(top[e], their_top), base = best == -INFINITY ? 0.f : best;
    const float a = fast_exp2(top[e] - base), b = fast_exp2(their_top - base);
    float sum = total[e] * a + left[DP / 2 + 2 + e] * b;
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    const float inv = sees[e] > 0 ? 1.f / sum : 0.f;
    mine_by[e] = a * inv;
    theirs_by[e] = b * inv;
  }
  bool fine[2] = {true, true};
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) {
    const float4 more = *reinterpret_cast<const float4*>(left + 4 * n);
    const float other[4] = {more.x, more.y, more.z, more.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = i >> 1, r = run * 16 + octet + 8 * e, d = n * 8 + 2 * quad + (i & 1);
      const float value = sees[e] > 0 ? o[n][i] * mine_by[e] + other[i] * theirs_by[e] : 0.f;
      fine[e] &= isfinite(value);
      if (r < rows && d < dim) Elem<T>::store(out + ((mine.begin + row0 + r) * p.heads + head) * dim + d, value);
    }
  }
  __syncwarp();  // a row's columns, which four threads have stored, may be stored again by another of them
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = run * 16 + octet + 8 * e;
    const unsigned not_fine = __ballot_sync(0xffffffffu, !fine[e]);
    if ((not_fine >> (lane & ~3) & 15u) == 0 || r >= rows) continue;
    // Each of the four takes a quarter of the columns. f32: pieces turn infinities into NaN, so the row is always taken again.
    const int each = (dim + 3) / 4;
    packed_row_again<T>(p, q + r * p.q_row, k, v, sees[e], keys, kPieces > 1, min(quad * each, dim), min((quad + 1) * each, dim),
                        out + ((mine.begin + row0 + r) * p.heads + head) * dim);
  }
}

std::once_flag g_mma_attr_once[64];

template <typename T, int DP>
void launch_mma(const PackedParams& p, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(p.rows_q / kTile + p.batch + 1), static_cast<unsigned>(p.heads));
  packed_mma_kernel<T, DP><<<grid, kMmaThreads, MmaTile<T, DP>::kBytes, s>>>(p);
}
template <typename T, int DP>
void mma_attribute() {
  cudaFuncSetAttribute(packed_mma_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                       static_cast<int>(MmaTile<T, DP>::kBytes));
}
template <typename T>
void mma_attributes() {
  mma_attribute<T, 64>();
  mma_attribute<T, 80>();
  mma_attribute<T, 96>();
  mma_attribute<T, 128>();
  mma_attribute<T, 192>();
  mma_attribute<T, 256>();
}

template <typename T>
void launch_mma_any(const PackedParams& p, cudaStream_t s) {
  if (p.dim <= 64)
    launch_mma<T, 64>(p, s);
  else if (p.dim <= 80)
    launch_mma<T, 80>(p, s);
  else if (p.dim <= 96)
    launch_mma<T, 96>(p, s);
  else if (p.dim <= 128)
    launch_mma<T, 128>(p, s);
  else if (p.dim <= 192)
    launch_mma<T, 192>(p, s);
  else
    launch_mma<T, 256>(p, s);
}

// ------------------------------------------------------------------------- bf16, head size 64 or 128
// The tensor-core form. A CTA takes two tiles of 128 query rows over the same keys: the same rows of two
// query heads that share a key/value head, or, where the heads do not come in such pairs, 256
// rows of one head. Each block of 128 keys is loaded once for both.
//   warps 0-3, 4-7  softmax of tile 0, 1: thread = query row = TMEM lane. It takes its 128 scores from tensor memory,
//                   keeps the running maximum and sum, writes P = 2^(score - maximum) as bf16 pairs over the scores (tcgen05.st)
//                   in two halves, each signalled when it is there, and rescales its row of the output
//                   accumulator only when the maximum grew by more than 2^8 (a stale maximum
//                   scales numerator and denominator alike).
//   warp 8          TMA: lane 0 Q and the K blocks, lane 1 the V blocks
//   warp 9          MMA issue: for each block, tile 0 then tile 1: O += P V (A from tensor memory), then the next S = Q K^T
// The tiles run half a period apart: while the tensor core works for one, the other's exponentials are
// computed. A tile's period is softmax + P V + Q K^T, since P lies where its scores were (tensor memory is full:
// 2 x 128 columns of scores, 2 x 128 of output), so the softmax's own length counts in full. It is
// kept short by registers for the whole row (setmaxnreg), three-input maxima and by taking a part of the exponentials off the
// special-function unit (16 a cycle and SM: 1024 cycles a block, as long as the two products). What bounds it now is
// that softmax: of the 3210 cycles of a period a group works 1950 (maximum 250, exponentials 1420, the rest loads, stores
// and signals: one warp to a scheduler hides little of its own latencies) and waits 1250 for the products, which the other
// group's work covers only in part. One sequence of 8192, 32/8 heads of 128: 463 us, 1187 TFLOP/s in short runs, 1058 sustained
// under the power cap (0.72 and 0.76 of measured cuBLAS); 4099 tokens in nine sequences 54 us; eight prompts of 128 12.6 us. Measured and not kept there: P in columns of its own with blocks
// of 80 keys, which ends the waiting but costs more softmax and MMA time a key (519 against 482 us); 16 softmax warps, two to a
// row (496); taking turns at the exponentials (506); the maximum taken alongside stale exponentials (519); a cubic
// for 0, 1/4 or 3/8 of the exponentials in place of 1/8 (491, 482, 530 against 468); a CTA that goes on to further tiles, taken
// back from the launch hardware (503 against 471: the loop costs the softmax more than the saved set-up gives).
// Masks cost only the blocks that they cut.
constexpr int kQRows = 128, kKeys = 128;
constexpr int kUmmaThreads = 384, kUmmaProducerWarp = 8, kUmmaMmaWarp = 9;
constexpr uint32_t kUmmaScoreCols = 128, kUmmaOutCol = 256;
constexpr float kRescale = 8.0f;
constexpr int kErrPackedWait = 2048;

template <int D>
struct UmmaTile {
  static constexpr int kChunks = D / 64;  // 64-element column chunks
  static constexpr int kStages = D == 64 ? 4 : 2;
  static constexpr uint32_t kBytes = kChunks * 16384;  // 128 rows x D bf16
  static constexpr uint32_t kVHalf = kChunks * 8192;   // 64 keys x D bf16
};

struct __align__(8) UmmaBarriers {
  uint64_t q_full[2];
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
  uint64_t s_full[2], p_full[2][2], o_done[2];  // by tile (and half of the keys)
  uint32_t tmem_base;
  int abort_flag;
};
template <int D>
constexpr size_t umma_smem_bytes() {
  return 1024 + (2 + 2 * UmmaTile<D>::kStages) * UmmaTile<D>::kBytes + sizeof(UmmaBarriers);
}

struct UmmaParams {
  PackedParams p;
  int32_t pairs;       // pairs of tiles in a row of pieces: heads / 2, or heads
  int32_t head_pairs;  // 1: the two tiles are two heads; 0: two runs of rows
  uint32_t idesc_qk, idesc_pv;
};

// 2^x for two values on the FMA pipe, |relative error| < 8.6e-5 (P is rounded to 2^-9): x = n + r with n the whole number below
// (adding 1.5 * 2^23 rounded down), a cubic for 2^r over [0, 1) that is 1 at 0 and was fitted for the least
// largest relative error, and n added to the exponent bits. At and below -127 the result is exactly 0, so that
// a masked or vanishing score does not even carry a huge value along.
__device__ __forceinline__ void exp2_pair(uint64_t x, float& lo, float& hi) {
  float a, b;
  unpack_f32x2(x, a, b);
  x = pack_f32x2(fmaxf(a, -127.f), fmaxf(b, -127.f));
  const uint64_t magic = pack_f32x2(12582912.f, 12582912.f), back = pack_f32x2(-12582912.f, -12582912.f);
  uint64_t shifted;
  asm("add.rm.f32x2 %0, %1, %2;" : "=l"(shifted) : "l"(x), "l"(magic));
  const uint64_t r = fma_f32x2(add_f32x2(shifted, back), pack_f32x2(-1.f, -1.f), x);
  uint64_t y = fma_f32x2(r, pack_f32x2(0.077067241f, 0.077067241f), pack_f32x2(0.22764498f, 0.22764498f));
  y = fma_f32x2(y, r, pack_f32x2(0.69511664f, 0.69511664f));
  y = fma_f32x2(y, r, pack_f32x2(1.f, 1.f));
  float n0, n1;
  unpack_f32x2(shifted, n0, n1);
  unpack_f32x2(y, lo, hi);
  lo = __int_as_float(__float_as_int(lo) + (__float_as_int(n0) << 23));
  hi = __int_as_float(__float_as_int(hi) + (__float_as_int(n1) << 23));
}

// The larger of three, NaN if one is.
__device__ __forceinline__ float nan_fmax(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <int D>
__global__ void __launch_bounds__(kUmmaThreads, 1)
    packed_umma_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, const __grid_constant__ UmmaParams u) {
  constexpr int kChunks = UmmaTile<D>::kChunks, kStages = UmmaTile<D>::kStages;
  constexpr uint32_t kTileBytes = UmmaTile<D>::kBytes, kVHalfBytes = UmmaTile<D>::kVHalf;
  extern __shared__ uint8_t smem_raw[];
  const PackedParams& p = u.p;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t q_smem = smem_base;
  const uint32_t k_smem = q_smem + 2 * kTileBytes;
  const uint32_t v_smem = k_smem + kStages * kTileBytes;
  const uint32_t end_smem = v_smem + kStages * kTileBytes;
  UmmaBarriers* bars = reinterpret_cast<UmmaBarriers*>(smem_raw + (end_smem - smem_u32(smem_raw)));
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 32 * kUmmaProducerWarp) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(smem_u32(&bars->q_full[t]), 1);
      mbar_init(smem_u32(&bars->s_full[t]), 1);
      mbar_init(smem_u32(&bars->p_full[t][0]), 4);
      mbar_init(smem_u32(&bars->p_full[t][1]), 4);
      mbar_init(smem_u32(&bars->o_done[t]), 1);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(smem_u32(&bars->k_full[s]), 1);
      mbar_init(smem_u32(&bars->k_empty[s]), 1);
      mbar_init(smem_u32(&bars->v_full[s]), 1);
      mbar_init(smem_u32(&bars->v_empty[s]), 1);
    }
    bars->abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  __syncwarp();

  // Which piece: the last rows of a sequence, which see the most keys, come first.
  const int rows_each = u.head_pairs ? kQRows : 2 * kQRows;
  const int64_t pieces = gridDim.x / u.pairs;
  const int64_t place = blockIdx.x / u.pairs;
  const int pair = static_cast<int>(blockIdx.x - place * u.pairs);
  const Piece piece = find_piece(p.batch, pieces - 1 - place, [&](int32_t b) {
    return (rows_of(p.offsets, b, p.rows_q, p.status).count + rows_each - 1) / rows_each;
  });
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out);
  if (piece.sequence < 0) {
    const Rows rest = rows_behind(p.offsets, p.batch, p.rows_q);
    const int64_t first = piece.index * rows_each;
    const int heads_here = u.head_pairs ? 2 : 1, head0 = u.head_pairs ? 2 * pair : pair;
    for (int64_t i = threadIdx.x; i < static_cast<int64_t>(rows_each) * heads_here * (D / 8); i += kUmmaThreads) {
      const int64_t r = first + i / (heads_here * (D / 8));
      const int part = static_cast<int>(i % (heads_here * (D / 8)));
      if (r < rest.count)
        *reinterpret_cast<uint4*>(out + ((rest.begin + r) * p.heads + head0) * D + part * 8) = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  const Rows mine = rows_of(p.offsets, piece.sequence, p.rows_q, nullptr);
  const Rows theirs = rows_of(p.k_offsets, piece.sequence, p.rows_k, p.status);
  const int64_t shift = p.causal ? theirs.count - mine.count + 1 : 0;  // row i sees the keys below i + shift
  int64_t row0[2], keys[2];
  int rows[2], head[2], blocks[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    head[t] = u.head_pairs ? 2 * pair + t : pair;
    row0[t] = piece.index * rows_each + (u.head_pairs ? 0 : t * kQRows);
    const int64_t left = mine.count - row0[t];
    rows[t] = static_cast<int>(left < 0 ? 0 : (left < kQRows ? left : kQRows));
    keys[t] = theirs.count;
    if (p.causal && row0[t] + rows[t] - 1 + shift < keys[t]) keys[t] = row0[t] + rows[t] - 1 + shift;
    if (rows[t] == 0 || keys[t] < 0) keys[t] = 0;
    blocks[t] = static_cast<int>((keys[t] + kKeys - 1) / kKeys);
  }
  const int most = max(blocks[0], blocks[1]);
  const int kv_head = head[0] / p.group;

  // The first copies are on their way before tensor memory is allocated and the warps meet.
  const int key_begin = static_cast<int>(theirs.begin), ready = min(kStages, most);
  auto load_keys = [&](int j, uint32_t stage) {  // lane 0: block j of K, lane 1: of V
    const uint32_t full = smem_u32(lane == 0 ? &bars->k_full[stage] : &bars->v_full[stage]);
    mbar_expect_tx(full, kTileBytes);
    if (lane == 0) {
      for (int c = 0; c < kChunks; ++c)
        tma_load_3d(k_smem + stage * kTileBytes + c * 16384, &map_k, full, 64 * c, key_begin + j * kKeys, kv_head);
    } else {
      for (int h = 0; h < 2; ++h)
        for (int c = 0; c < kChunks; ++c)
          tma_load_3d(v_smem + stage * kTileBytes + h * kVHalfBytes + c * 8192, &map_v, full, 64 * c,
                      key_begin + j * kKeys + 64 * h, kv_head);
    }
  };
  if (warp == kUmmaProducerWarp && lane < 2) {
    if (lane == 0) {
      for (int t = 0; t < 2; ++t) {
        if (!blocks[t]) continue;
        const uint32_t qf = smem_u32(&bars->q_full[t]);
        mbar_expect_tx(qf, kTileBytes);
        for (int c = 0; c < kChunks; ++c)
          tma_load_3d(q_smem + t * kTileBytes + c * 16384, &map_q, qf, 64 * c, static_cast<int>(mine.begin + row0[t]), head[t]);
      }
    }
    for (int j = 0; j < ready; ++j) load_keys(j, j);
  }
  __syncwarp();
  if (warp == kUmmaMmaWarp) {
    tmem_alloc<1>(smem_u32(&bars->tmem_base), 512);
    tmem_relinquish<1>();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;

  if (warp >= 8) {
    // 384 threads x 168 registers at launch = 128 x (2 x 208 + 88)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == kUmmaProducerWarp && lane < 2) {
      // ---------------------------------------------------------------- TMA producers
      uint32_t stage = 0, parity = 0;
      for (int j = ready; j < most; ++j) {
        if (!mbar_wait(smem_u32(lane == 0 ? &bars->k_empty[stage] : &bars->v_empty[stage]), parity, abort_flag, p.status, kErrPackedWait))
          break;
        load_keys(j, stage);
        if (++stage == kStages) {
          stage = 0;
          parity ^= 1u;
        }
      }
      if (*abort_flag) {
        // Loads that were issued may still be in flight: give them (bounded) time to land.
        const unsigned long long start = global_ns();
        while (global_ns() - start < 2000000ull) {
        }
      }
    } else if (warp == kUmmaMmaWarp && lane == 0) {
      // ---------------------------------------------------------------- MMA issuer
      const uint32_t hi = desc_hi(1024);
      bool ok = true;
      auto scores = [&](int t, int j) {  // S_t = Q_t K_j^T, both K-major
        const uint64_t q_desc = make_desc(q_smem + t * kTileBytes, 1u, hi);
        const uint64_t k_desc = make_desc(k_smem + (j % kStages) * kTileBytes, 1u, hi);
        const uint32_t d_tmem = tmem_base + t * kUmmaScoreCols;
#pragma unroll
        for (int i = 0; i < kChunks * 4; ++i) {
          const uint64_t step = static_cast<uint64_t>(((i >> 2) * 16384 + (i & 3) * 32) >> 4);
          umma_bf16<1>(d_tmem, q_desc + step, k_desc + step, u.idesc_qk, i ? 1u : 0u);
        }
        umma_commit<1>(smem_u32(&bars->s_full[t]));
      };
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        ok = ok && mbar_wait(smem_u32(bar), parity, abort_flag, p.status, kErrPackedWait);
        tc_fence_after();
        return ok;
      };
      if (most > 0 && wait(&bars->k_full[0], 0)) {
        for (int t = 0; t < 2 && ok; ++t)
          if (blocks[t] && wait(&bars->q_full[t], 0)) scores(t, 0);
        umma_commit<1>(smem_u32(&bars->k_empty[0]));
      }
      for (int j = 0; j < most && ok; ++j) {
        const uint32_t st = j % kStages, next = (j + 1) % kStages;
        const uint64_t v_lo = make_desc(v_smem + st * kTileBytes, 8192u >> 4, hi);
        const uint64_t v_hi = make_desc(v_smem + st * kTileBytes + kVHalfBytes, 8192u >> 4, hi);
        if (!wait(&bars->v_full[st], (j / kStages) & 1)) break;
        if (j + 1 < most && !wait(&bars->k_full[next], ((j + 1) / kStages) & 1)) break;
        for (int t = 0; t < 2 && ok; ++t) {
          if (j >= blocks[t]) continue;
          const uint32_t d_tmem = tmem_base + kUmmaOutCol + t * D, p_tmem = tmem_base + t * kUmmaScoreCols;
          if (!wait(&bars->p_full[t][0], j & 1)) break;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            umma_bf16_ts(d_tmem, p_tmem + i * 8, v_lo + static_cast<uint64_t>((i * 2048) >> 4), u.idesc_pv, (j | i) ? 1u : 0u);
          if (!wait(&bars->p_full[t][1], j & 1)) break;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            umma_bf16_ts(d_tmem, p_tmem + 32 + i * 8, v_hi + static_cast<uint64_t>((i * 2048) >> 4), u.idesc_pv, 1u);
          umma_commit<1>(smem_u32(&bars->o_done[t]));
          // The next scores go where P lies; the tensor core runs what one thread issues in order.
          if (j + 1 < blocks[t]) scores(t, j + 1);
        }
        umma_commit<1>(smem_u32(&bars->v_empty[st]));
        if (j + 1 < most) umma_commit<1>(smem_u32(&bars->k_empty[next]));
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- softmax and output
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int t = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t score_addr = tmem_base + lane_addr + t * kUmmaScoreCols;
    const uint32_t out_addr = tmem_base + lane_addr + kUmmaOutCol + t * D;
    const int64_t my_row0 = t ? row0[1] : row0[0], my_keys = t ? keys[1] : keys[0];
    const int my_rows = t ? rows[1] : rows[0], my_blocks = t ? blocks[1] : blocks[0], my_head = t ? head[1] : head[0];
    // keys that this row sees, and those that every row of the tile sees
    int64_t sees = theirs.count, all_see = theirs.count;
    if (p.causal) {
      sees = min(max(my_row0 + row + shift, int64_t{0}), theirs.count);
      all_see = min(max(my_row0 + shift, int64_t{0}), theirs.count);
    }
    const uint32_t s_full = smem_u32(&bars->s_full[t]), o_done = smem_u32(&bars->o_done[t]);
    const uint32_t p_half0 = smem_u32(&bars->p_full[t][0]), p_half1 = smem_u32(&bars->p_full[t][1]);
    float top = -1.0e30f, total = 0.f;
    bool ok = true;
    for (int j = 0; j < my_blocks; ++j) {
      ok = mbar_wait(s_full, j & 1, abort_flag, p.status, kErrPackedWait);
      ok = __all_sync(0xffffffffu, ok) != 0;
      if (!ok) break;
      tc_fence_after();
      float s[kKeys];
      {
        uint32_t(&raw)[kKeys] = reinterpret_cast<uint32_t(&)[kKeys]>(s);
#pragma unroll
        for (int c = 0; c < kKeys / 32; ++c) tmem_ld_32x32(score_addr + c * 32, reinterpret_cast<uint32_t(&)[32]>(raw[c * 32]));
        tmem_ld_wait();
      }
      if (static_cast<int64_t>(j + 1) * kKeys > all_see) {
        const int64_t here = sees - static_cast<int64_t>(j) * kKeys;
        const int valid = static_cast<int>(here < kKeys ? here : kKeys);
#pragma unroll
        for (int i = 0; i < kKeys; ++i)
          if (i >= valid) s[i] = -INFINITY;
      }
      float part[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) part[i] = nan_fmax(s[i], s[i + 8], s[i + 16]);
#pragma unroll
      for (int i = 24; i < kKeys - 8; i += 16)
#pragma unroll
        for (int x = 0; x < 8; ++x) part[x] = nan_fmax(part[x], s[i + x], s[i + 8 + x]);
#pragma unroll
      for (int x = 0; x < 4; ++x) part[x] = nan_fmax(part[x], s[kKeys - 8 + x], s[kKeys - 4 + x]);
      part[0] = nan_fmax(part[0], part[1], part[2]);
      part[3] = nan_fmax(part[3], part[4], part[5]);
      part[6] = nan_fmax(part[6], part[7], part[0]);
      const float raw = nan_fmax(part[3], part[6], part[6]) * p.scale_log2, best = nan_fmax(top, raw, raw);
      if (__any_sync(0xffffffffu, !(best - top <= kRescale))) {
        // Some row of this warp outgrew its maximum, or is not finite (it stays NaN from here on).
        const float higher = best < INFINITY ? best : __uint_as_float(0x7fc00000u);
        const float alpha = fast_exp2(top - higher);
        total *= alpha;
        top = higher;
        if (j > 0) {
          ok = mbar_wait(o_done, (j - 1) & 1, abort_flag, p.status, kErrPackedWait);
          ok = __all_sync(0xffffffffu, ok) != 0;
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t raw[16];
            tmem_ld_32x16(out_addr + c * 16, raw);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) raw[i] = __float_as_uint(__uint_as_float(raw[i]) * alpha);
            tmem_st_32x16(out_addr + c * 16, raw);
          }
          tmem_st_wait();
        }
      }
      const uint64_t scale2 = pack_f32x2(p.scale_log2, p.scale_log2), neg_top2 = pack_f32x2(-top, -top);
      uint64_t sums[4] = {0, 0, 0, 0};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t packed[32];
#pragma unroll
        for (int i = 0; i < 64; i += 2) {
          const uint64_t x = fma_f32x2(pack_f32x2(s[h * 64 + i], s[h * 64 + i + 1]), scale2, neg_top2);
          float lo, hi;
          if ((i & 14) == 14) {  // one pair of eight on the FMA pipe
            exp2_pair(x, lo, hi);
          } else {
            unpack_f32x2(x, lo, hi);
            lo = fast_exp2(lo);
            hi = fast_exp2(hi);
          }
          sums[(i >> 1) & 3] = add_f32x2(sums[(i >> 1) & 3], pack_f32x2(lo, hi));
          packed[i >> 1] = pack_bf16x2(lo, hi);
        }
        tmem_st_32x32(score_addr + h * 32, packed);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(h ? p_half1 : p_half0);
      }
      float lo, hi;
      unpack_f32x2(add_f32x2(add_f32x2(sums[0], sums[1]), add_f32x2(sums[2], sums[3])), lo, hi);
      total += lo + hi;
    }
    if (ok && my_blocks > 0) {
      ok = mbar_wait(o_done, (my_blocks - 1) & 1, abort_flag, p.status, kErrPackedWait);
      ok = __all_sync(0xffffffffu, ok) != 0;
      tc_fence_after();
    }
    if (ok) {
      const float inv = sees > 0 ? 1.f / total : 0.f;
      __nv_bfloat16* dst = out + ((mine.begin + my_row0 + row) * p.heads + my_head) * D;
      uint32_t largest = 0;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t x[32];
        if (my_blocks > 0) {
          tmem_ld_32x32(out_addr + c * 32, x);
          tmem_ld_wait();
        }
        float o[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          o[i] = sees > 0 ? __uint_as_float(x[i]) * inv : 0.f;
          largest = max(largest, __float_as_uint(o[i]) & 0x7fffffffu);
        }
        if (row < my_rows) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {  // whole sectors: 32 bytes a thread (in 16: 14.6 in place of 12.6 us for eight prompts of 128)
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = pack_bf16x2(o[16 * i + 2 * e], o[16 * i + 2 * e + 1]);
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + c * 32 + 16 * i), "r"(w[0]), "r"(w[1]),
                         "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                         : "memory");
          }
        }
      }
      if (largest >= 0x7f800000u && row < my_rows) {
        const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(p.q) + (mine.begin + my_row0 + row) * p.q_row + my_head * p.q_head;
        const __nv_bfloat16* k = static_cast<const __nv_bfloat16*>(p.k) + theirs.begin * p.k_row + kv_head * p.k_head;
        const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(p.v) + theirs.begin * p.v_row + kv_head * p.v_head;
        const int64_t read = min(static_cast<int64_t>(my_blocks) * kKeys, p.rows_k - theirs.begin);
        packed_row_again<__nv_bfloat16>(p, q, k, v, sees, read, false, 0, D, dst);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kUmmaMmaWarp) {
    tc_fence_after();
    tmem_dealloc<1>(tmem_base, 512);
  }
}

uint32_t umma_idesc(int n, bool b_kmajor) {
  uint32_t d = 0;
  d |= 1u << 4;   // D format f32
  d |= 1u << 7;   // A format bf16
  d |= 1u << 10;  // B format bf16
  d |= (b_kmajor ? 0u : 1u) << 16;
  d |= static_cast<uint32_t>(n >> 3) << 17;
  d |= static_cast<uint32_t>(kQRows >> 4) << 24;
  return d;
}

std::once_flag g_umma_attr_once[64];

bool tma_strides(const void* base, int64_t row, int64_t head) {
  return aligned(base, 16) && row > 0 && head > 0 && row % 8 == 0 && head % 8 == 0 && row < (int64_t{1} << 38) &&
         head < (int64_t{1} << 38);
}
// The tensor-core form takes bf16 heads of 64 and 128 with a positive scale (its maximum is that of the raw scores) and
// strides that a TMA descriptor can hold.
bool umma_takes(const b200_packed_attention_desc& d) {
  return d.dtype == B200_BF16 && (d.dim == 64 || d.dim == 128) && d.scale > 0.f && d.rows_k > 0 &&
         tma_strides(d.q, d.q_row, d.q_head) && tma_strides(d.k, d.k_row, d.k_head) && tma_strides(d.v, d.v_row, d.v_head) &&
         aligned(d.out, 32);
}

template <int D>
int launch_umma(const PackedParams& p, const b200_packed_attention_desc& d, cudaStream_t s) {
  UmmaParams u{};
  u.p = p;
  // Pairs of heads share every key block and mask, and leave tiles of 128 rows; an odd group pairs rows instead.
  u.head_pairs = p.group % 2 == 0;
  u.pairs = u.head_pairs ? p.heads / 2 : p.heads;
  const int64_t pieces = p.rows_q / (u.head_pairs ? kQRows : 2 * kQRows) + p.batch + 1;
  if (pieces * u.pairs > INT32_MAX) return refuse(B200_E_SHAPE);
  u.idesc_qk = umma_idesc(kKeys, true);
  u.idesc_pv = umma_idesc(D, false);
  CUtensorMap map_q, map_k, map_v;
  if (!encode_map(&map_q, d.q, D, d.rows_q, d.heads, d.q_row, d.q_head, 64, kQRows) ||
      !encode_map(&map_k, d.k, D, d.rows_k, d.kv_heads, d.k_row, d.k_head, 64, kKeys) ||
      !encode_map(&map_v, d.v, D, d.rows_k, d.kv_heads, d.v_row, d.v_head, 64, 64))
    return refuse(B200_E_DEVICE);
  packed_umma_kernel<D><<<static_cast<unsigned>(pieces * u.pairs), kUmmaThreads, umma_smem_bytes<D>(), s>>>(map_q, map_k, map_v, u);
  return launched();
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_attention_packed(const b200_packed_attention_desc* desc, void* stream) {
  if (!enabled()) return refuse(B200_E_DISABLED);
  if (!desc) return refuse(B200_E_NULL);
  const b200_packed_attention_desc& d = *desc;
  if (!valid_dtype(d.dtype)) return refuse(B200_E_DTYPE);
  if (d.rows_q < 0 || d.rows_k < 0 || d.batch < 0 || d.heads < 1 || d.kv_heads < 1 || d.heads % d.kv_heads || d.dim < 1 ||
      d.dim > 256)
    return refuse(B200_E_SHAPE);
  if (!(fabsf(d.scale) <= 3.0e38f) || (d.causal & ~1)) return refuse(B200_E_ARG);
  if (d.rows_q == 0) return finish(0);
  if (!d.q || !d.out || !d.offsets || !d.k_offsets || (d.rows_k > 0 && (!d.k || !d.v))) return refuse(B200_E_NULL);
  if (d.rows_q > INT32_MAX || d.rows_k > INT32_MAX || d.batch > INT32_MAX / 2 || d.heads > 65535) return refuse(B200_E_SHAPE);
  const size_t size = dtype_size(d.dtype);
  if (!aligned(d.q, size) || !aligned(d.k, size) || !aligned(d.v, size) || !aligned(d.out, size) || !aligned(d.offsets, 4) ||
      !aligned(d.k_offsets, 4))
    return refuse(B200_E_ALIGN);
  const DeviceInfo& dev = device_info();
  if (dev.sm_count == 0) return refuse(B200_E_DEVICE);
  cudaStream_t s = static_cast<cudaStream_t>(stream);

  PackedParams p{};
  p.q = d.q;
  p.k = d.k;
  p.v = d.v;
  p.out = d.out;
  p.q_row = d.q_row;
  p.q_head = d.q_head;
  p.k_row = d.k_row;
  p.k_head = d.k_head;
  p.v_row = d.v_row;
  p.v_head = d.v_head;
  p.rows_q = d.rows_q;
  p.rows_k = d.rows_k;
  p.offsets = d.offsets;
  p.k_offsets = d.k_offsets;
  p.batch = static_cast<int32_t>(d.batch);
  p.heads = static_cast<int32_t>(d.heads);
  p.group = static_cast<int32_t>(d.heads / d.kv_heads);
  p.dim = static_cast<int32_t>(d.dim);
  p.causal = d.causal;
  const int64_t strides = d.q_row | d.q_head | d.k_row | d.k_head | d.v_row | d.v_head | d.dim;
  p.vectors = strides % 4 == 0 && aligned(d.q, 16) && aligned(d.k, 16) && aligned(d.v, 16);
  p.scale_log2 = d.scale * kLog2e;
  p.status = kernel_status_word();

  std::call_once(g_mma_attr_once[dev.device], [] {
    mma_attributes<float>();
    mma_attributes<__nv_bfloat16>();
  });
  std::call_once(g_umma_attr_once[dev.device], [] {
    cudaFuncSetAttribute(packed_umma_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                         static_cast<int>(umma_smem_bytes<64>()));
    cudaFuncSetAttribute(packed_umma_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                         static_cast<int>(umma_smem_bytes<128>()));
  });
  if (umma_takes(d)) return d.dim == 64 ? launch_umma<64>(p, d, s) : launch_umma<128>(p, d, s);
  if (d.dtype == B200_F32)
    launch_mma_any<float>(p, s);
  else
    launch_mma_any<__nv_bfloat16>(p, s);
  return launched();
}
