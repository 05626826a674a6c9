// Prompt attention over packed sequences: out_i = sum_j softmax_j(scale q_i . k_j) v_j for
// query row i of a sequence over that sequence's keys, causal or not, query head h reading
// key/value head h / (heads / kv_heads). q, out: [rows_q][heads][dim], k, v:
// [rows_k][kv_heads][dim], any row and head strides; sequence b owns the rows
// [offsets[b], offsets[b + 1]). Causal: the queries are the last positions of the keys, so
// row i sees keys j <= i + keys - queries. A row that sees no key is zeros, and so are the
// rows behind the last sequence. No reference counterpart.
#include <math.h>

#include <mutex>

#include "sequences.cuh"

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
  float scale_log2;  // scale * log2(e)
  int32_t* status;
};

// ------------------------------------------------------------------------- any type, any head size
// One CTA takes 64 query rows of one head and goes over the keys in tiles of 64 with the running
// maximum and sum of the softmax (f32 throughout, products by FFMA). 128 threads in an 8 x 16 grid:
// a thread has 8 rows and 4 keys of the scores, and 8 rows and DP / 16 columns of the output
// in registers; of the four LDS wavefronts per k the eight-row operand is a broadcast, so the
// inner loops are bound by FFMA issue (32 a step) and not by shared memory. Operands
// lie transposed ([dim][row]) so that both are read as 16-byte vectors.
constexpr int kTile = 64, kSimtThreads = 128, kPad = 4;

template <int DP>
constexpr size_t simt_smem_bytes() {
  return (2 * DP * (kTile + kPad) + kTile * (DP + kPad) + kTile * (kTile + kPad)) * sizeof(float);
}

template <typename T, int DP>
__global__ void __launch_bounds__(kSimtThreads) packed_simt_kernel(const PackedParams p) {
  extern __shared__ float smem[];
  float* qt = smem;                           // [DP][64 + pad]
  float* kt = qt + DP * (kTile + kPad);       // [DP][64 + pad]
  float* vs = kt + DP * (kTile + kPad);       // [64][DP + pad]
  float* ps = vs + kTile * (DP + kPad);       // [key][64 + pad]
  constexpr int kStep = kTile + kPad, kVStep = DP + kPad, kCols = DP / 64;

  const int head = blockIdx.y, dim = p.dim;
  // Tiles with many keys first (causal): a long sequence's last rows would otherwise start last.
  const Piece piece = find_piece(p.batch, static_cast<int64_t>(gridDim.x) - 1 - blockIdx.x, [&](int32_t b) {
    return (rows_of(p.offsets, b, p.rows_q, p.status).count + kTile - 1) / kTile;
  });
  T* out = static_cast<T*>(p.out);
  if (piece.sequence < 0) {
    const Rows rest = rows_behind(p.offsets, p.batch, p.rows_q);
    const int64_t first = piece.index * kTile;
    for (int r = 0; r < kTile && first + r < rest.count; ++r)
      for (int d = threadIdx.x; d < dim; d += kSimtThreads)
        Elem<T>::store(out + ((rest.begin + first + r) * p.heads + head) * dim + d, 0.f);
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

  for (int i = threadIdx.x; i < kTile * DP; i += kSimtThreads) {
    const int r = i / DP, d = i % DP;
    qt[d * kStep + r] = r < rows && d < dim ? Elem<T>::load(q + r * p.q_row + d) : 0.f;
  }
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  float top[8], total[8], acc[8][kCols * 4];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    top[i] = -INFINITY;
    total[i] = 0.f;
#pragma unroll
    for (int c = 0; c < kCols * 4; ++c) acc[i][c] = 0.f;
  }
  for (int64_t key0 = 0; key0 < keys; key0 += kTile) {
    const int here = static_cast<int>(keys - key0 < kTile ? keys - key0 : kTile);
    __syncthreads();
    for (int i = threadIdx.x; i < kTile * DP; i += kSimtThreads) {
      const int r = i / DP, d = i % DP;
      const bool in = r < here && d < dim;  // past the end: zeros, whatever lies there
      kt[d * kStep + r] = in ? Elem<T>::load(k + (key0 + r) * p.k_row + d) : 0.f;
      vs[r * kVStep + d] = in ? Elem<T>::load(v + (key0 + r) * p.v_row + d) : 0.f;
    }
    __syncthreads();
    float s[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 4
    for (int d = 0; d < DP; ++d) {
      const float4 a0 = *reinterpret_cast<const float4*>(qt + d * kStep + ty * 8);
      const float4 a1 = *reinterpret_cast<const float4*>(qt + d * kStep + ty * 8 + 4);
      const float4 b = *reinterpret_cast<const float4*>(kt + d * kStep + tx * 4);
      const float a[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s[i][0] = fmaf(a[i], b.x, s[i][0]);
        s[i][1] = fmaf(a[i], b.y, s[i][1]);
        s[i][2] = fmaf(a[i], b.z, s[i][2]);
        s[i][3] = fmaf(a[i], b.w, s[i][3]);
      }
    }
    // Whether some row of the tile sees only a part of these keys.
    const bool cut = p.causal && row0 + shift < key0 + here;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t limit = p.causal ? row0 + ty * 8 + i + shift - key0 : here;
      float best = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = tx * 4 + j;
        s[i][j] = key < here && key < limit ? s[i][j] * p.scale_log2 : -INFINITY;
        best = fmaxf(best, s[i][j]);
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
      best = fmaxf(best, top[i]);
      const float base = best == -INFINITY ? 0.f : best;  // nothing seen yet: every term is 2^-inf
      const float keep = fast_exp2(top[i] - base);
      top[i] = best;
      total[i] *= keep;
#pragma unroll
      for (int c = 0; c < kCols * 4; ++c) acc[i][c] *= keep;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = fast_exp2(s[i][j] - base);
        total[i] += s[i][j];
        ps[(tx * 4 + j) * kStep + ty * 8 + i] = s[i][j];
      }
    }
    __syncthreads();
    for (int key = 0; key < here; ++key) {
      const float4 a0 = *reinterpret_cast<const float4*>(ps + key * kStep + ty * 8);
      const float4 a1 = *reinterpret_cast<const float4*>(ps + key * kStep + ty * 8 + 4);
      const float a[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        const float4 b = *reinterpret_cast<const float4*>(vs + key * kVStep + c * 64 + tx * 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          // A masked value must not be read as 0 * value: it may be an infinity or NaN.
          if (cut && key0 + key >= row0 + ty * 8 + i + shift) continue;
          acc[i][c * 4] = fmaf(a[i], b.x, acc[i][c * 4]);
          acc[i][c * 4 + 1] = fmaf(a[i], b.y, acc[i][c * 4 + 1]);
          acc[i][c * 4 + 2] = fmaf(a[i], b.z, acc[i][c * 4 + 2]);
          acc[i][c * 4 + 3] = fmaf(a[i], b.w, acc[i][c * 4 + 3]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) total[i] += __shfl_xor_sync(0xffffffffu, total[i], o);
    const int r = ty * 8 + i;
    if (r >= rows) continue;
    const bool none = p.causal ? row0 + r + shift <= 0 || theirs.count == 0 : theirs.count == 0;
    const float inv = none ? 0.f : 1.f / total[i];
    T* dst = out + ((mine.begin + row0 + r) * p.heads + head) * dim;
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int d = c * 64 + tx * 4 + j;
        if (d < dim) Elem<T>::store(dst + d, none ? 0.f : acc[i][c * 4 + j] * inv);
      }
  }
}

std::once_flag g_simt_attr_once[64];

template <typename T, int DP>
void launch_simt(const PackedParams& p, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(p.rows_q / kTile + p.batch + 1), static_cast<unsigned>(p.heads));
  packed_simt_kernel<T, DP><<<grid, kSimtThreads, simt_smem_bytes<DP>(), s>>>(p);
}

template <typename T>
void simt_attributes() {
  cudaFuncSetAttribute(packed_simt_kernel<T, 64>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                       static_cast<int>(simt_smem_bytes<64>()));
  cudaFuncSetAttribute(packed_simt_kernel<T, 128>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                       static_cast<int>(simt_smem_bytes<128>()));
  cudaFuncSetAttribute(packed_simt_kernel<T, 256>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                       static_cast<int>(simt_smem_bytes<256>()));
}

template <typename T>
void launch_simt_any(const PackedParams& p, cudaStream_t s) {
  if (p.dim <= 64)
    launch_simt<T, 64>(p, s);
  else if (p.dim <= 128)
    launch_simt<T, 128>(p, s);
  else
    launch_simt<T, 256>(p, s);
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
  p.scale_log2 = d.scale * kLog2e;
  p.status = kernel_status_word();

  std::call_once(g_simt_attr_once[dev.device], [] {
    simt_attributes<float>();
    simt_attributes<__nv_bfloat16>();
  });
  if (d.dtype == B200_F32)
    launch_simt_any<float>(p, s);
  else
    launch_simt_any<__nv_bfloat16>(p, s);
  return launched();
}
