// Writing tokens into the 8-bit key/value cache and reading them back (kv_cache.cuh has the
// layout). Both are bound by HBM: a value is read and written once, held in registers in between.
//
// A write takes one CTA per (block of the cache, head, K or V). With x the new values of the block:
//   s = max(s_old, max|x| / 127, 2^-100),  s_old counting only if the block holds older tokens of the sequence
//   code = rint(x / s), ties to even;  older codes, where s > s_old: rint(code * s_old / s)
// so a block's scale never shrinks while it fills, and an older value moves by at most half
// a step each time the scale grows. A value that is not finite makes s NaN: everything that
// reads the block's head then answers NaN. No reference counterpart.
#include "kv_cache.cuh"

namespace b200 {
namespace {

constexpr float kSmallestScale = 7.888609052210118e-31f;  // 2^-100: rint's test products stay normal numbers
constexpr uint32_t kInfBits = 0x7f800000u;

// rint(x / s) to the last tie: a first guess from the reciprocal, which is off by at most one,
// moved by the exact signs of x - (r +- 1/2) s (one rounding of an exact product and sum: the
// sign is right, and zero is a tie, which goes to the even neighbour).
__device__ __forceinline__ int quotient_code(float x, float s, float inv) {
  float r = rintf(x * inv);
  const float over = fmaf(-(r + 0.5f), s, x), under = fmaf(-(r - 0.5f), s, x);
  const bool odd = static_cast<int>(r) & 1;
  if (over > 0.f || (over == 0.f && odd)) r += 1.f;
  if (under < 0.f || (under == 0.f && odd)) r -= 1.f;
  return static_cast<int>(r);
}
// rint(code * old / s): both sides of each comparison are exact in f64 (at most 33 bits).
__device__ __forceinline__ int rescaled_code(int code, float old, float s) {
  const double x = static_cast<double>(code) * old, step = s;
  double r = rint(x / step);
  const bool odd = static_cast<int>(r) & 1;
  const double over = x - (r + 0.5) * step, under = x - (r - 0.5) * step;
  if (over > 0. || (over == 0. && odd)) r += 1.;
  if (under < 0. || (under == 0. && odd)) r -= 1.;
  return static_cast<int>(r);
}

__device__ __forceinline__ uint32_t pack_codes(int a, int b, int c, int d) {
  return (a & 255) | (b & 255) << 8 | (c & 255) << 16 | static_cast<uint32_t>(d & 255) << 24;
}
__device__ __forceinline__ int code_at(uint32_t word, int i) { return static_cast<int8_t>(word >> (8 * i)); }

// 8 consecutive values.
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const uint4 lo = ld_plain16(p), hi = ld_plain16(p + 4);
  float a[4], b[4];
  unpack16(lo, a);
  unpack16(hi, b);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = a[i];
    v[4 + i] = b[i];
  }
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) { unpack16(ld_plain16(p), v); }
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  const float a[4] = {v[0], v[1], v[2], v[3]}, b[4] = {v[4], v[5], v[6], v[7]};
  *reinterpret_cast<uint4*>(p) = pack16(a);
  *reinterpret_cast<uint4*>(p + 4) = pack16(b);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) { *reinterpret_cast<uint4*>(p) = pack16(v); }

struct AppendParams {
  Cache cache;
  Table table;
  const void *k, *v;
  int64_t k_row, k_head, v_row, v_head;  // strides in elements
  const int32_t *lengths, *offsets;      // lengths before; offsets NULL: `each` new tokens per sequence
  int64_t rows;
  int32_t batch, each;
  int32_t* status;
};

// A thread holds 8 values of each of 4 consecutive tokens. Threads of a warp go along the head first
// for K (8 code bytes of a token next to each other) and along the tokens first for V (4 codes of a
// channel in one word, the words of a channel next to each other), so both leave in whole sectors.
template <typename T>
__global__ void kv_append_kernel(const AppendParams p) {
  const Cache& c = p.cache;
  const bool is_v = blockIdx.z;
  const int head = blockIdx.y;
  auto new_rows = [&](int32_t b) {
    if (p.offsets) return rows_of(p.offsets, b, p.rows, p.status);
    return Rows{static_cast<int64_t>(b) * p.each, p.each};
  };
  Piece piece{static_cast<int32_t>(blockIdx.x), 0};
  if (p.offsets || p.each != 1)
    piece = find_piece(p.batch, blockIdx.x, [&](int32_t b) {
      const int64_t n = new_rows(b).count, length = max(p.lengths[b], 0);
      return n == 0 ? int64_t{0} : ((length + n - 1) >> c.token_bits) - (length >> c.token_bits) + 1;
    });
  if (piece.sequence < 0) return;
  const Rows rows = new_rows(piece.sequence);
  const int64_t length = max(p.lengths[piece.sequence], 0);
  const int64_t page = (length >> c.token_bits) + piece.index;
  const int64_t block = block_of(c, p.table, piece.sequence, page, p.status);
  if (block < 0) return;
  const int64_t start = page << c.token_bits;
  const int first = static_cast<int>(max(length, start) - start);  // slots [first, stop) are new
  const int stop = static_cast<int>(min(length + rows.count, start + c.tokens) - start);
  const int64_t row = rows.begin + start - length;  // of slot 0

  const int parts = c.dim / 8, groups = c.tokens / 4;
  const int part = is_v ? threadIdx.x / groups : threadIdx.x % parts;
  const int slot0 = 4 * (is_v ? threadIdx.x % groups : threadIdx.x / parts);
  const T* src = static_cast<const T*>(is_v ? p.v : p.k) + head * (is_v ? p.v_head : p.k_head) + part * 8;
  const int64_t step = is_v ? p.v_row : p.k_row;
  float x[4][8];
  uint32_t largest = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int slot = slot0 + j;
    if (slot >= first && slot < stop) {
      load8(src + (row + slot) * step, x[j]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[j][i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) largest = max(largest, __float_as_uint(x[j][i]) & 0x7fffffffu);  // NaN above infinity
  }
  __shared__ uint32_t warp_largest[8];
  __shared__ float old_scale;
  float* scale = (is_v ? c.v_scales : c.k_scales) + block * c.heads + head;
  largest = __reduce_max_sync(0xffffffffu, largest);
  if ((threadIdx.x & 31) == 0) warp_largest[threadIdx.x >> 5] = largest;
  if (threadIdx.x == 0) old_scale = first > 0 ? *scale : 0.f;
  __syncthreads();
  largest = warp_largest[0];
  for (unsigned w = 1; w < blockDim.x / 32; ++w) largest = max(largest, warp_largest[w]);
  const float before = old_scale;
  float s = fmaxf(fmaxf(__fdiv_rn(__uint_as_float(largest), 127.f), kSmallestScale), before);
  const bool finite = largest < kInfBits && before == before;
  if (!finite) s = __uint_as_float(0x7fc00000u);
  if (threadIdx.x == 0 && !(s == before)) *scale = s;

  int8_t* codes = (is_v ? c.v_codes : c.k_codes) + (block * c.heads + head) * c.tokens * c.dim;
  if (first > 0 && finite && s > before) {
    // The older tokens' codes follow the scale: rare (a running maximum over a block's tokens).
    for (int i = threadIdx.x; i < c.dim * first; i += blockDim.x) {
      int8_t* at = codes + (is_v ? (i / first) * c.tokens + i % first : i);
      *at = static_cast<int8_t>(rescaled_code(*at, before, s));
    }
  }
  const float inv = __frcp_rn(s);
  uint32_t word[8];  // K: two words of each token; V: one word of each channel
#pragma unroll
  for (int i = 0; i < 8; ++i) word[i] = 0;
  if (finite) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      int code[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) code[i] = quotient_code(x[j][i], s, inv);
      if (is_v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) word[i] |= static_cast<uint32_t>(code[i] & 255) << (8 * j);
      } else {
        word[2 * j] = pack_codes(code[0], code[1], code[2], code[3]);
        word[2 * j + 1] = pack_codes(code[4], code[5], code[6], code[7]);
      }
    }
  }
  if (!is_v) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (slot0 + j >= first && slot0 + j < stop)
        *reinterpret_cast<uint2*>(codes + (slot0 + j) * c.dim + part * 8) = make_uint2(word[2 * j], word[2 * j + 1]);
  } else if (slot0 >= first && slot0 + 4 <= stop) {
#pragma unroll
    for (int i = 0; i < 8; ++i) *reinterpret_cast<uint32_t*>(codes + (part * 8 + i) * c.tokens + slot0) = word[i];
  } else if (slot0 + 4 > first && slot0 < stop) {
    // A word that older or later slots share: only the new slots' bytes are touched.
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (slot0 + j >= first && slot0 + j < stop)
          codes[(part * 8 + i) * c.tokens + slot0 + j] = static_cast<int8_t>(code_at(word[i], j));
  }
}

struct ReadParams {
  Cache cache;
  Table table;
  void *k_out, *v_out;  // [rows][heads][dim]
  const int32_t *starts, *lengths, *offsets;
  int64_t rows;
  int32_t batch;
  int32_t* status;
};

// The same division of a block among threads as in the write, the other way round.
template <typename T>
__global__ void kv_read_kernel(const ReadParams p) {
  const Cache& c = p.cache;
  const bool is_v = blockIdx.z;
  const int head = blockIdx.y;
  const int parts = c.dim / 8, groups = c.tokens / 4;
  const int part = is_v ? threadIdx.x / groups : threadIdx.x % parts;
  const int slot0 = 4 * (is_v ? threadIdx.x % groups : threadIdx.x / parts);
  T* out = static_cast<T*>(is_v ? p.v_out : p.k_out) + static_cast<int64_t>(head) * c.dim + part * 8;
  const int64_t step = static_cast<int64_t>(c.heads) * c.dim;
  const Piece piece = find_piece(p.batch, blockIdx.x, [&](int32_t b) {
    const int64_t n = rows_of(p.offsets, b, p.rows, p.status).count, start = max(p.starts[b], 0);
    return n == 0 ? int64_t{0} : ((start + n - 1) >> c.token_bits) - (start >> c.token_bits) + 1;
  });
  const float none[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (piece.sequence < 0) {
    const Rows rest = rows_behind(p.offsets, p.batch, p.rows);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t r = (piece.index << c.token_bits) + slot0 + j;
      if (r < rest.count) store8(out + (rest.begin + r) * step, none);
    }
    return;
  }
  const Rows rows = rows_of(p.offsets, piece.sequence, p.rows, nullptr);
  const int64_t from = max(p.starts[piece.sequence], 0), page = (from >> c.token_bits) + piece.index;
  const int64_t start = page << c.token_bits;
  const int first = static_cast<int>(max(from, start) - start);
  const int stop = static_cast<int>(min(from + rows.count, start + c.tokens) - start);
  const int held = static_cast<int>(min(max(p.lengths[piece.sequence] - start, int64_t{0}), int64_t{stop}));
  const int64_t row = rows.begin + start - from;  // of slot 0
  float s = 0.f;
  uint32_t word[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) word[i] = 0;
  if (held > first) {
    const int64_t block = block_of(c, p.table, piece.sequence, page, p.status);
    if (block < 0) {
      s = __uint_as_float(0x7fc00000u);
    } else {
      s = (is_v ? c.v_scales : c.k_scales)[block * c.heads + head];
      const int8_t* codes = (is_v ? c.v_codes : c.k_codes) + (block * c.heads + head) * c.tokens * c.dim;
      if (is_v) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          word[i] = __ldg(reinterpret_cast<const uint32_t*>(codes + (part * 8 + i) * c.tokens + slot0));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint2 w = __ldg(reinterpret_cast<const uint2*>(codes + (slot0 + j) * c.dim + part * 8));
          word[2 * j] = w.x;
          word[2 * j + 1] = w.y;
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (slot0 + j < first || slot0 + j >= stop) continue;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int code = is_v ? code_at(word[i], j) : code_at(word[2 * j + i / 4], i & 3);
      x[i] = slot0 + j < held ? static_cast<float>(code) * s : 0.f;
    }
    store8(out + (row + slot0 + j) * step, x);
  }
}

bool table_ok(const int32_t* table, int64_t batch, int64_t stride, int64_t width) {
  return width >= 0 && width <= INT32_MAX && (batch <= 1 || stride >= width) && (table || width == 0);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_kv_append(const b200_kv_append_desc* desc, void* stream) {
  if (!enabled()) return refuse(B200_E_DISABLED);
  if (!desc) return refuse(B200_E_NULL);
  const b200_kv_append_desc& d = *desc;
  if (!valid_dtype(d.dtype)) return refuse(B200_E_DTYPE);
  if (!valid_cache(&d.cache) || d.batch < 0 || d.rows < 0 || d.rows > INT32_MAX || d.batch > INT32_MAX / 8)
    return refuse(B200_E_SHAPE);
  if (!d.offsets && d.batch > 0 && d.rows % d.batch) return refuse(B200_E_SHAPE);
  if (d.batch == 0 || d.rows == 0) return finish(0);
  if (!cache_pointers(&d.cache) || !d.k || !d.v || !d.lengths) return refuse(B200_E_NULL);
  if (!table_ok(d.block_table, d.batch, d.table_stride, d.table_width)) return refuse(B200_E_STRIDE);
  const int64_t vec = d.dtype == B200_F32 ? 4 : 8;
  if (d.k_row % vec || d.k_head % vec || d.v_row % vec || d.v_head % vec) return refuse(B200_E_STRIDE);
  if (!cache_aligned(&d.cache) || !aligned(d.k, 16) || !aligned(d.v, 16) || !aligned(d.block_table, 4) ||
      !aligned(d.lengths, 4) || !aligned(d.offsets, 4))
    return refuse(B200_E_ALIGN);
  if (device_info().sm_count == 0) return refuse(B200_E_DEVICE);
  AppendParams p{};
  p.cache = device_cache(&d.cache);
  p.table = Table{d.block_table, d.table_stride, static_cast<int32_t>(d.table_width)};
  p.k = d.k;
  p.v = d.v;
  p.k_row = d.k_row;
  p.k_head = d.k_head;
  p.v_row = d.v_row;
  p.v_head = d.v_head;
  p.lengths = d.lengths;
  p.offsets = d.offsets;
  p.rows = d.rows;
  p.batch = static_cast<int32_t>(d.batch);
  p.each = d.offsets ? 0 : static_cast<int32_t>(d.rows / d.batch);
  p.status = kernel_status_word();
  // n new tokens touch at most (n - 2) / tokens + 2 blocks; one token each, one block each
  const int64_t pieces = !d.offsets && d.rows == d.batch ? d.batch : d.rows / d.cache.block_tokens + 2 * d.batch;
  const dim3 grid(static_cast<unsigned>(pieces), static_cast<unsigned>(d.cache.heads), 2);
  const unsigned threads = static_cast<unsigned>(d.cache.block_tokens / 4 * (d.cache.dim / 8));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d.dtype == B200_F32)
    kv_append_kernel<float><<<grid, threads, 0, s>>>(p);
  else
    kv_append_kernel<__nv_bfloat16><<<grid, threads, 0, s>>>(p);
  return launched();
}

extern "C" int b200_kv_read(const b200_kv_read_desc* desc, void* stream) {
  if (!enabled()) return refuse(B200_E_DISABLED);
  if (!desc) return refuse(B200_E_NULL);
  const b200_kv_read_desc& d = *desc;
  if (!valid_dtype(d.dtype)) return refuse(B200_E_DTYPE);
  if (!valid_cache(&d.cache) || d.batch < 0 || d.rows < 0 || d.rows > INT32_MAX || d.batch > INT32_MAX / 8)
    return refuse(B200_E_SHAPE);
  if (d.rows == 0) return finish(0);
  if (!cache_pointers(&d.cache) || !d.k_out || !d.v_out || !d.offsets || (d.batch > 0 && (!d.starts || !d.lengths)))
    return refuse(B200_E_NULL);
  if (!table_ok(d.block_table, d.batch, d.table_stride, d.table_width)) return refuse(B200_E_STRIDE);
  if (!cache_aligned(&d.cache) || !aligned(d.k_out, 16) || !aligned(d.v_out, 16) || !aligned(d.block_table, 4) ||
      !aligned(d.starts, 4) || !aligned(d.lengths, 4) || !aligned(d.offsets, 4))
    return refuse(B200_E_ALIGN);
  if (device_info().sm_count == 0) return refuse(B200_E_DEVICE);
  ReadParams p{};
  p.cache = device_cache(&d.cache);
  p.table = Table{d.block_table, d.table_stride, static_cast<int32_t>(d.table_width)};
  p.k_out = d.k_out;
  p.v_out = d.v_out;
  p.starts = d.starts;
  p.lengths = d.lengths;
  p.offsets = d.offsets;
  p.rows = d.rows;
  p.batch = static_cast<int32_t>(d.batch);
  p.status = kernel_status_word();
  // two partial blocks a sequence at most, and the rows behind the last sequence
  const int64_t pieces = d.rows / d.cache.block_tokens + 2 * d.batch + 1;
  const dim3 grid(static_cast<unsigned>(pieces), static_cast<unsigned>(d.cache.heads), 2);
  const unsigned threads = static_cast<unsigned>(d.cache.block_tokens / 4 * (d.cache.dim / 8));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d.dtype == B200_F32)
    kv_read_kernel<float><<<grid, threads, 0, s>>>(p);
  else
    kv_read_kernel<__nv_bfloat16><<<grid, threads, 0, s>>>(p);
  return launched();
}
