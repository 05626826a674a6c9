// Attention over the 8-bit key/value cache (kv_cache.cuh) for the last `tokens` positions of
// each sequence: out_i = sum_j softmax_j(scale q_i . k_j) v_j over the positions
// j <= lengths - tokens + i, k_j = code * k_scale[block, head], v_j = code * v_scale[block, head].
// q, out: [batch][tokens][heads][dim]; query head h reads key/value head h / group. A row that
// sees nothing is zeros. No reference counterpart.
#include <math.h>

#include "kv_cache.cuh"

namespace b200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kThreads = 128;

struct CachedParams {
  Cache cache;
  Table table;
  const void* q;
  void* out;  // contiguous
  int64_t q_batch, q_token, q_head;
  const int32_t* lengths;
  int32_t batch, tokens, heads, group;
  float scale_log2;
  int32_t* status;
};

// One CTA per (sequence, token, query head): a thread scores one position of a tile of 128, then sums
// one channel over the tile.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) cached_simple_kernel(const CachedParams p) {
  __shared__ float query[D], prob[kThreads], value_scale[kThreads], part[4];
  __shared__ int64_t where[kThreads];
  const Cache& c = p.cache;
  const int head = blockIdx.x, token = blockIdx.y, b = blockIdx.z, kv_head = head / p.group;
  T* out = static_cast<T*>(p.out) + ((static_cast<int64_t>(b) * p.tokens + token) * p.heads + head) * D;
  const int64_t limit = static_cast<int64_t>(p.lengths[b]) - p.tokens + token + 1;
  if (threadIdx.x < D)
    query[threadIdx.x] =
        Elem<T>::load(static_cast<const T*>(p.q) + b * p.q_batch + token * p.q_token + head * p.q_head + threadIdx.x);
  float top = -INFINITY, total = 0.f, acc = 0.f;
  for (int64_t tile = 0; tile < limit; tile += kThreads) {
    __syncthreads();
    const int64_t position = tile + threadIdx.x;
    float s = -INFINITY;
    if (position < limit) {
      const int64_t block = block_of(c, p.table, b, position >> c.token_bits, p.status);
      where[threadIdx.x] = block;
      value_scale[threadIdx.x] = __uint_as_float(0x7fc00000u);
      s = value_scale[threadIdx.x];
      if (block >= 0) {
        const int8_t* k = c.k_codes + (block * c.heads + kv_head) * c.tokens * D + (position & (c.tokens - 1)) * D;
        s = 0.f;
        for (int d = 0; d < D; ++d) s = fmaf(query[d], k[d], s);
        s *= c.k_scales[block * c.heads + kv_head] * p.scale_log2;
        value_scale[threadIdx.x] = c.v_scales[block * c.heads + kv_head];
      }
    }
    const float warp_best = warp_fmax(s);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = warp_best;
    __syncthreads();
    const float best = fmaxf(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])), top);
    const float base = best == -INFINITY ? 0.f : best;
    const float keep = fast_exp2(top - base);
    top = best;
    prob[threadIdx.x] = position < limit ? fast_exp2(s - base) : 0.f;
    __syncthreads();
    total *= keep;
    acc *= keep;
    const int here = static_cast<int>(limit - tile < kThreads ? limit - tile : kThreads);
    for (int j = 0; j < here; ++j) {
      total += prob[j];
      if (threadIdx.x >= D) continue;
      const int64_t at = (where[j] * c.heads + kv_head) * c.tokens * D + threadIdx.x * c.tokens + ((tile + j) & (c.tokens - 1));
      acc = fmaf(prob[j], (where[j] < 0 ? 1.f : static_cast<float>(c.v_codes[at])) * value_scale[j], acc);
    }
  }
  if (threadIdx.x < D) Elem<T>::store(out + threadIdx.x, limit <= 0 ? 0.f : acc / total);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" size_t b200_attention_cached_workspace_bytes(const b200_kv_cache* cache, int64_t batch, int64_t tokens,
                                                        int64_t heads, int64_t table_width) {
  return 0;
}

extern "C" int b200_attention_cached(const b200_kv_cache* cache, int32_t dtype, const void* q, int64_t q_batch,
                                     int64_t q_token, int64_t q_head, void* out, const int32_t* block_table,
                                     int64_t table_stride, int64_t table_width, const int32_t* lengths, int64_t batch,
                                     int64_t tokens, int64_t heads, float scale, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  if (!enabled()) return refuse(B200_E_DISABLED);
  if (!cache) return refuse(B200_E_NULL);
  if (!valid_dtype(dtype)) return refuse(B200_E_DTYPE);
  if (!valid_cache(cache) || batch < 0 || tokens < 0 || heads < 1 || heads % cache->heads || batch > 65535 || tokens > 65535)
    return refuse(B200_E_SHAPE);
  if (!(fabsf(scale) <= 3.0e38f)) return refuse(B200_E_ARG);
  if (batch == 0 || tokens == 0) return finish(0);
  if (!cache_pointers(cache) || !q || !out || !lengths) return refuse(B200_E_NULL);
  if (table_width < 0 || table_width > INT32_MAX || (batch > 1 && table_stride < table_width)) return refuse(B200_E_STRIDE);
  if (!cache_aligned(cache)) return refuse(B200_E_ALIGN);
  if (device_info().sm_count == 0) return refuse(B200_E_DEVICE);
  CachedParams p{};
  p.cache = device_cache(cache);
  p.table = Table{block_table, table_stride, static_cast<int32_t>(table_width)};
  p.q = q;
  p.out = out;
  p.q_batch = q_batch;
  p.q_token = q_token;
  p.q_head = q_head;
  p.lengths = lengths;
  p.batch = static_cast<int32_t>(batch);
  p.tokens = static_cast<int32_t>(tokens);
  p.heads = static_cast<int32_t>(heads);
  p.group = static_cast<int32_t>(heads / cache->heads);
  p.scale_log2 = scale * kLog2e;
  p.status = kernel_status_word();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(heads), static_cast<unsigned>(tokens), static_cast<unsigned>(batch));
  if (dtype == B200_F32 && cache->dim == 64)
    cached_simple_kernel<float, 64><<<grid, kThreads, 0, s>>>(p);
  else if (dtype == B200_F32)
    cached_simple_kernel<float, 128><<<grid, kThreads, 0, s>>>(p);
  else if (cache->dim == 64)
    cached_simple_kernel<__nv_bfloat16, 64><<<grid, kThreads, 0, s>>>(p);
  else
    cached_simple_kernel<__nv_bfloat16, 128><<<grid, kThreads, 0, s>>>(p);
  return launched();
}
