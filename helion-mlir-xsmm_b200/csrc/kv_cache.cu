// Writing tokens into the 8-bit key/value cache and reading them back (kv_cache.cuh has the
// layout). Both should be bound by HBM: a value is read and written once, held in registers in between. Measured (one B200, 8
// heads of 128): reading 12 prefixes of up to 4096 as bf16 35 us (5.3 TB/s, 0.80 of measured copy bandwidth); writing 10600 prompt
// tokens 28 us (2.4 TB/s: bound by the chain of dependent loads at the start of each CTA, four CTAs to an SM); writing one
// token for each of 128 sequences 5.3 us (latency).
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

// Conversions by the bits of 1.5 * 2^23 + n: cvt and rint run at a quarter of the rate of the FMA pipe and set the time
// of both kernels otherwise (a write of 10600 tokens, 8 heads of 128: 55 us with them, 40 without).
constexpr float kWhole = 12582912.f;
// x / s to the nearest, as the bits of kWhole + code (the low byte is the code): `inv` is within 2^-23 of 1 / s, so the result can
// only be wrong next to a tie, where the remainder is near s / 2 (`rest` keeps the largest).
__device__ __forceinline__ float quotient(float x, float s, float inv, float& rest) {
  const float shifted = fmaf(x, inv, kWhole);
  rest = fmaxf(rest, fabsf(fmaf(kWhole - shifted, s, x)));
  return shifted;
}
constexpr float kNearTie = 0.4999f;
// rint(x / s), ties to even: the guess moved by the exact signs of x - (r +- 1/2) s (one rounding of an exact product and
// sum: the sign is right, and zero is a tie).
__device__ __forceinline__ float quotient_at_tie(float x, float s, float shifted) {
  float r = shifted - kWhole;
  const float over = fmaf(-(r + 0.5f), s, x), under = fmaf(-(r - 0.5f), s, x);
  const bool odd = static_cast<int>(r) & 1;
  if (over > 0.f || (over == 0.f && odd)) r += 1.f;
  if (under < 0.f || (under == 0.f && odd)) r -= 1.f;
  return r + kWhole;
}
// rint(code * old / s), old <= s: as above, with both sides of the comparison exact in f64 (32 bits at most), which is
// looked at only where the quotient is near a tie.
__device__ __forceinline__ float code_value(uint32_t word, int i) {  // of byte i: 2^23 + 128 + code, less 2^23 + 128
  return __uint_as_float(__byte_perm(word ^ 0x80808080u, 0x4B000000u, 0x7440 + i)) - 8388736.f;
}
__device__ __forceinline__ float rescaled(float code, float old, float s, float ratio) {
  const float q = code * ratio, shifted = q + kWhole;
  if (fabsf(fabsf(q - (shifted - kWhole)) - 0.5f) > 1e-3f) return shifted;
  const double low = floor(static_cast<double>(q));
  const double off = static_cast<double>(code) * old - (low + 0.5) * s;  // above or below the tie that is near
  const bool odd = static_cast<int>(low) & 1;
  return static_cast<float>(low) + (off > 0. || (off == 0. && odd) ? 1.f : 0.f) + kWhole;
}
// Byte `i` of `word` replaced by the low byte of `code`'s bits.
__device__ __forceinline__ uint32_t with_code(uint32_t word, int i, float code) {
  return __byte_perm(word, __float_as_uint(code), i == 0 ? 0x3214 : (i == 1 ? 0x3240 : (i == 2 ? 0x3410 : 0x4210)));
}

// A thread's eight channels of a token: 16 bytes next to each other for bf16, and for f32 16 bytes in either half of the head, so
// that neighbouring threads always touch neighbouring 16 bytes. channel_of is the i-th.
template <typename T>
__device__ __forceinline__ int channel_of(int part, int i, int dim) {
  return sizeof(T) == 2 ? part * 8 + i : (i >> 2) * (dim >> 1) + part * 4 + (i & 3);
}
template <typename T>
struct Eight {
  uint4 raw[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* token, int part, int dim) {
#pragma unroll
    for (unsigned i = 0; i < sizeof(T) / 2; ++i) raw[i] = ld_stream16(token + channel_of<T>(part, i * Elem<T>::kVec, dim));
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (unsigned i = 0; i < sizeof(T) / 2; ++i) raw[i] = make_uint4(0, 0, 0, 0);
  }
  // The largest magnitude's bits as f32 (infinities above all numbers, NaN above them).
  __device__ __forceinline__ uint32_t largest() const {
    uint32_t m = 0;
#pragma unroll
    for (unsigned i = 0; i < sizeof(T) / 2; ++i) {
      const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (sizeof(T) == 4)
          m = max(m, w[e] & 0x7fffffffu);
        else
          m = __vmaxu2(m, w[e] & 0x7fff7fffu);
      }
    }
    return sizeof(T) == 4 ? m : max(m << 16, m & 0xffff0000u);
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
    float part[Elem<T>::kVec];
#pragma unroll
    for (unsigned i = 0; i < sizeof(T) / 2; ++i) {
      unpack16(raw[i], part);
#pragma unroll
      for (int e = 0; e < Elem<T>::kVec; ++e) v[i * Elem<T>::kVec + e] = part[e];
    }
  }
};
__device__ __forceinline__ void store8(float* token, int part, int dim, const float (&v)[8]) {
  const float a[4] = {v[0], v[1], v[2], v[3]}, b[4] = {v[4], v[5], v[6], v[7]};
  st_stream16(token + channel_of<float>(part, 0, dim), pack16(a));
  st_stream16(token + channel_of<float>(part, 4, dim), pack16(b));
}
__device__ __forceinline__ void store8(__nv_bfloat16* token, int part, int dim, const float (&v)[8]) {
  st_stream16(token + part * 8, pack16(v));
}
// Those channels' codes of a token of K: two words.
template <typename T>
__device__ __forceinline__ uint2 load_codes(const int8_t* token, int part, int dim) {
  if (sizeof(T) == 2) return *reinterpret_cast<const uint2*>(token + part * 8);
  return make_uint2(*reinterpret_cast<const uint32_t*>(token + channel_of<T>(part, 0, dim)),
                    *reinterpret_cast<const uint32_t*>(token + channel_of<T>(part, 4, dim)));
}
template <typename T>
__device__ __forceinline__ void store_codes(int8_t* token, int part, int dim, uint32_t lo, uint32_t hi) {
  if (sizeof(T) == 2) {
    *reinterpret_cast<uint2*>(token + part * 8) = make_uint2(lo, hi);
  } else {
    *reinterpret_cast<uint32_t*>(token + channel_of<T>(part, 0, dim)) = lo;
    *reinterpret_cast<uint32_t*>(token + channel_of<T>(part, 4, dim)) = hi;
  }
}
// A block of V in shared memory, as words of four tokens: word g of channel r. Every run of channels that one thread holds starts
// a bank further on, so that neighbouring threads' words do not collide.
constexpr int kTurnWords = 64 / 4 * 128 + 128 / 4;
template <typename T>
__device__ __forceinline__ int turn_at(int r, int g, int groups) {
  constexpr int kRun = Elem<T>::kVec;
  return r / kRun * (kRun * groups + 1) + r % kRun * groups + g;
}

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

// Which block a CTA writes, and the slots [first, stop) of it that are new; `row` is the packed row of slot 0.
struct AppendPlace {
  int32_t sequence;
  int64_t page, row;
  int first, stop;
};
__device__ __forceinline__ bool find_append(const AppendParams& p, AppendPlace& at) {
  const Cache& c = p.cache;
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
  if (piece.sequence < 0) return false;
  const Rows rows = new_rows(piece.sequence);
  const int64_t length = max(p.lengths[piece.sequence], 0);
  at.sequence = piece.sequence;
  at.page = (length >> c.token_bits) + piece.index;
  const int64_t start = at.page << c.token_bits;
  at.first = static_cast<int>(max(length, start) - start);
  at.stop = static_cast<int>(min(length + rows.count, start + c.tokens) - start);
  at.row = rows.begin + start - length;
  return true;
}
// The block's scale from the largest new magnitude (its bits) and the scale before.
__device__ __forceinline__ float new_scale(uint32_t largest, float before, bool& finite) {
  finite = largest < kInfBits && before == before;
  const float s = fmaxf(fmaxf(__fdiv_rn(__uint_as_float(largest), 127.f), kSmallestScale), before);
  return finite ? s : __uint_as_float(0x7fc00000u);
}

// A thread holds 8 values of each of 4 consecutive tokens; the threads of a warp go along the head first, so values are read
// and K's codes written in whole lines. V's codes lie the other way round: a block that is written whole is turned
// in shared memory (words of four tokens) and leaves as one run of lines; of one that is not, each thread
// writes its words. A CTA is one chain of
// dependent loads (lengths, then its values and the table, then the block's scale and codes): what counts is how many
// are on an SM, so registers are held to four CTAs of 256 threads.
template <typename T, bool is_v>
__device__ __forceinline__ void append_block(const AppendParams& p, uint32_t* turn) {
  const Cache& c = p.cache;
  AppendPlace place;
  if (!find_append(p, place)) return;
  const int first = place.first, stop = place.stop;
  const int head = blockIdx.y, parts = c.dim / 8, groups = c.tokens / 4;
  const int part = threadIdx.x % parts, slot0 = threadIdx.x / parts * 4;
  const int64_t step = is_v ? p.v_row : p.k_row;
  const T* src = static_cast<const T*>(is_v ? p.v : p.k) + place.row * step + head * (is_v ? p.v_head : p.k_head);
  auto is_new = [&](int j) { return slot0 + j >= first && slot0 + j < stop; };
  const bool any_new = slot0 + 4 > first && slot0 < stop, all_new = slot0 >= first && slot0 + 4 <= stop;
  const bool any_old = slot0 < first;

  Eight<T> here[4];  // on their way while the block is looked up
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (is_new(j))
      here[j].load(src + (slot0 + j) * step, part, c.dim);
    else
      here[j].clear();
  }
  const int64_t block = block_of(c, p.table, place.sequence, place.page, p.status);
  if (block < 0) return;
  float* scale = (is_v ? c.v_scales : c.k_scales) + block * c.heads + head;
  const float before = first > 0 ? *scale : 0.f;
  int8_t* codes = (is_v ? c.v_codes : c.k_codes) + (block * c.heads + head) * c.tokens * c.dim;
  // K: two words of each token; V: one word of each channel. What is there counts only where older
  // tokens or bytes of other slots share a word.
  uint32_t word[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) word[i] = 0;
  if (is_v ? (any_old || any_new) && !all_new : any_old) {
    if (is_v) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        word[i] = *reinterpret_cast<const uint32_t*>(codes + channel_of<T>(part, i, c.dim) * c.tokens + slot0);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint2 w = load_codes<T>(codes + (slot0 + j) * c.dim, part, c.dim);
        word[2 * j] = w.x;
        word[2 * j + 1] = w.y;
      }
    }
  }
  __shared__ uint32_t warp_largest[8];
  uint32_t largest = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) largest = max(largest, here[j].largest());
  largest = __reduce_max_sync(0xffffffffu, largest);
  if ((threadIdx.x & 31) == 0) warp_largest[threadIdx.x >> 5] = largest;
  __syncthreads();
  largest = warp_largest[0];
  for (unsigned w = 1; w < blockDim.x / 32; ++w) largest = max(largest, warp_largest[w]);
  bool finite;
  const float s = new_scale(largest, before, finite);
  if (threadIdx.x == 0 && !(s == before)) *scale = s;  // (every thread has read it before the barrier)

  const bool grew = finite && first > 0 && s > before;
  if (grew && any_old) {
    // The older tokens' codes follow the scale: rare (a running maximum over a block's tokens).
    const float ratio = __fdiv_rn(before, s);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (slot0 + j >= first) continue;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint32_t& w = word[is_v ? i : 2 * j + i / 4];
        const int at = is_v ? j : i & 3;
        w = with_code(w, at, rescaled(code_value(w, at), before, s, ratio));
      }
    }
  }
  if (!finite) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (is_new(j))
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint32_t& w = word[is_v ? i : 2 * j + i / 4];
          w = with_code(w, is_v ? j : i & 3, kWhole);
        }
  } else if (any_new) {
    const float inv = __frcp_rn(s);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (!is_new(j)) continue;
      float x[8], code[8], rest = 0.f;
      here[j].values(x);
#pragma unroll
      for (int i = 0; i < 8; ++i) code[i] = quotient(x[i], s, inv, rest);
      if (rest > kNearTie * s) {
#pragma unroll
        for (int i = 0; i < 8; ++i) code[i] = quotient_at_tie(x[i], s, code[i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint32_t& w = word[is_v ? i : 2 * j + i / 4];
        w = with_code(w, is_v ? j : i & 3, code[i]);
      }
    }
  }
  if (!is_v) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (is_new(j) || (grew && slot0 + j < first))
        store_codes<T>(codes + (slot0 + j) * c.dim, part, c.dim, word[2 * j], word[2 * j + 1]);
  } else if (first == 0 && stop == c.tokens) {
#pragma unroll
    for (int i = 0; i < 8; ++i) turn[turn_at<T>(channel_of<T>(part, i, c.dim), slot0 / 4, groups)] = word[i];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int at = 4 * (threadIdx.x + n * blockDim.x), r = at / groups, g = at % groups;
      uint4 w;
      w.x = turn[turn_at<T>(r, g, groups)];
      w.y = turn[turn_at<T>(r, g + 1, groups)];
      w.z = turn[turn_at<T>(r, g + 2, groups)];
      w.w = turn[turn_at<T>(r, g + 3, groups)];
      *reinterpret_cast<uint4*>(codes + 4 * at) = w;
    }
  } else if (any_new || (grew && any_old)) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      *reinterpret_cast<uint32_t*>(codes + channel_of<T>(part, i, c.dim) * c.tokens + slot0) = word[i];
  }
}

template <typename T>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 3) kv_append_kernel(const AppendParams p) {
  __shared__ uint32_t turn[kTurnWords];
  if (blockIdx.z)
    append_block<T, true>(p, turn);
  else
    append_block<T, false>(p, turn);
}

// The same write when the blocks get few tokens each (single tokens of many sequences): a warp for each (block, head,
// K or V), whose lanes hold dim / 32 channels of a token. A CTA of the kernel above would be up to 256 threads for
// one token (128 tokens into blocks of 64: 23.5 us, and 5.3 here).
template <typename T, int PER>
__device__ __forceinline__ void load_channels(const T* p, float (&v)[PER]) {  // dim / 32 = 2 or 4 channels
  if (sizeof(T) * PER == 16) {
    const uint4 w = ld_stream16(p);
    v[0] = __uint_as_float(w.x);
    v[1] = __uint_as_float(w.y);
    v[PER - 2] = __uint_as_float(w.z);
    v[PER - 1] = __uint_as_float(w.w);
  } else if (sizeof(T) == 4) {
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
    v[0] = __uint_as_float(w.x);
    v[1] = __uint_as_float(w.y);
  } else if (PER == 4) {
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
    v[0] = __uint_as_float(w.x << 16);
    v[1] = __uint_as_float(w.x & 0xffff0000u);
    v[PER - 2] = __uint_as_float(w.y << 16);
    v[PER - 1] = __uint_as_float(w.y & 0xffff0000u);
  } else {
    const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(p));
    v[0] = __uint_as_float(w << 16);
    v[1] = __uint_as_float(w & 0xffff0000u);
  }
}

template <typename T, int PER>
__global__ void __launch_bounds__(256) kv_append_few_kernel(const AppendParams p) {
  const Cache& c = p.cache;
  const int lane = threadIdx.x & 31;
  const int task = blockIdx.y * 8 + (threadIdx.x >> 5), head = task >> 1;
  const bool is_v = task & 1;
  AppendPlace at;
  if (!find_append(p, at) || head >= c.heads) return;
  const int first = at.first, stop = at.stop;
  const int64_t step = is_v ? p.v_row : p.k_row;
  const T* src = static_cast<const T*>(is_v ? p.v : p.k) + at.row * step + head * (is_v ? p.v_head : p.k_head) + lane * PER;
  float x[PER];
  load_channels<T, PER>(src + first * step, x);  // of the first token: often the only one
  const int64_t block = block_of(c, p.table, at.sequence, at.page, p.status);
  if (block < 0) return;
  float* scale = (is_v ? c.v_scales : c.k_scales) + block * c.heads + head;
  const float before = first > 0 ? *scale : 0.f;
  uint32_t largest = 0;
  for (int slot = first; slot < stop; ++slot) {
    float y[PER];
    if (slot == first) {
#pragma unroll
      for (int i = 0; i < PER; ++i) y[i] = x[i];
    } else {
      load_channels<T, PER>(src + slot * step, y);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) largest = max(largest, __float_as_uint(y[i]) & 0x7fffffffu);
  }
  largest = __reduce_max_sync(0xffffffffu, largest);
  bool finite;
  const float s = new_scale(largest, before, finite);
  if (lane == 0 && !(s == before)) *scale = s;
  int8_t* codes = (is_v ? c.v_codes : c.k_codes) + (block * c.heads + head) * c.tokens * c.dim;
  if (finite && first > 0 && s > before) {
    const float ratio = __fdiv_rn(before, s);
    const int words = is_v ? (first + 3) / 4 : c.dim / 4;  // of a channel's old tokens, or of a token
    const int rows = is_v ? c.dim : first;
    for (int i = lane; i < rows * words; i += 32) {
      const int row = i / words, word = i - row * words;
      uint32_t* where = reinterpret_cast<uint32_t*>(codes + row * (is_v ? c.tokens : c.dim) + word * 4);
      const uint32_t old = *where;
      uint32_t w = old;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (!is_v || word * 4 + e < first) w = with_code(w, e, rescaled(code_value(w, e), before, s, ratio));
      *where = w;
    }
    __syncwarp();  // a word of V may hold new tokens too: they are written after it
  }
  const float inv = __frcp_rn(s);
  for (int slot = first; slot < stop; ++slot) {
    if (slot > first) load_channels<T, PER>(src + slot * step, x);
    float code[PER], rest = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) code[i] = quotient(x[i], s, inv, rest);
    if (rest > kNearTie * s) {
#pragma unroll
      for (int i = 0; i < PER; ++i) code[i] = quotient_at_tie(x[i], s, code[i]);
    }
    if (is_v) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        codes[(lane * PER + i) * c.tokens + slot] = static_cast<int8_t>(finite ? __float_as_uint(code[i]) & 255 : 0);
    } else {
      uint32_t w = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) w = with_code(w, i, finite ? code[i] : kWhole);
      int8_t* where = codes + slot * c.dim + lane * PER;
      if (PER == 4)
        *reinterpret_cast<uint32_t*>(where) = w;
      else
        *reinterpret_cast<uint16_t*>(where) = static_cast<uint16_t>(w);
    }
  }
}

struct ReadParams {
  Cache cache;
  Table table;
  void *k_out, *v_out;  // [rows][heads][dim]
  const int32_t *starts, *lengths, *offsets;
  int64_t rows;
  int32_t batch;
  int32_t heads_each;
  int32_t* status;
};

// The same division of a block among threads as in the write, the other way round; a CTA goes over several heads with the next
// one's codes on their way, so that finding the block is done once.
template <typename T, bool is_v>
__device__ __forceinline__ void read_block(const ReadParams& p, uint32_t* turn) {
  const Cache& c = p.cache;
  const int parts = c.dim / 8, groups = c.tokens / 4;
  const int part = threadIdx.x % parts, slot0 = threadIdx.x / parts * 4;
  const int head0 = blockIdx.y * p.heads_each, head_end = min(head0 + p.heads_each, c.heads);
  T* out = static_cast<T*>(is_v ? p.v_out : p.k_out);
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
      if (r < rest.count)
        for (int head = head0; head < head_end; ++head) store8(out + (rest.begin + r) * step + head * c.dim, part, c.dim, none);
    }
    return;
  }
  const Rows rows = rows_of(p.offsets, piece.sequence, p.rows, nullptr);
  const int64_t from = max(p.starts[piece.sequence], 0), page = (from >> c.token_bits) + piece.index;
  const int64_t start = page << c.token_bits;
  const int first = static_cast<int>(max(from, start) - start);
  const int stop = static_cast<int>(min(from + rows.count, start + c.tokens) - start);
  const int held = static_cast<int>(min(max(p.lengths[piece.sequence] - start, int64_t{0}), int64_t{stop}));
  out += (rows.begin + start - from) * step;
  int64_t block = -1;
  if (held > first) block = block_of(c, p.table, piece.sequence, page, p.status);
  const bool any = slot0 + 4 > first && slot0 < held;

  uint32_t next[8];  // K: two words of each token; V: eight words of the block as it lies, to be turned
  float next_scale = held > first ? __uint_as_float(0x7fc00000u) : 0.f;  // (a bad block)
#pragma unroll
  for (int i = 0; i < 8; ++i) next[i] = 0;
  auto fetch = [&](int head) {
    if (block < 0) return;
    next_scale = (is_v ? c.v_scales : c.k_scales)[block * c.heads + head];
    const int8_t* codes = (is_v ? c.v_codes : c.k_codes) + (block * c.heads + head) * c.tokens * c.dim;
    if (is_v) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const uint4 w = ld_stream16(codes + 16 * (threadIdx.x + n * blockDim.x));
        next[4 * n] = w.x;
        next[4 * n + 1] = w.y;
        next[4 * n + 2] = w.z;
        next[4 * n + 3] = w.w;
      }
    } else if (any) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint2 w = load_codes<T>(codes + (slot0 + j) * c.dim, part, c.dim);
        next[2 * j] = w.x;
        next[2 * j + 1] = w.y;
      }
    }
  };
  fetch(head0);
  for (int head = head0; head < head_end; ++head) {
    uint32_t word[8];
    if (is_v) {
      if (head > head0) __syncthreads();  // the last head's words have been taken
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = 4 * (threadIdx.x + (i >> 2) * blockDim.x) + (i & 3);
        turn[turn_at<T>(at / groups, at % groups, groups)] = next[i];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) word[i] = turn[turn_at<T>(channel_of<T>(part, i, c.dim), slot0 / 4, groups)];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) word[i] = next[i];
    }
    const float s = next_scale;
    if (head + 1 < head_end) fetch(head + 1);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (slot0 + j < first || slot0 + j >= stop) continue;
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float code = is_v ? code_value(word[i], j) : code_value(word[2 * j + i / 4], i & 3);
        x[i] = slot0 + j < held ? code * s : 0.f;
      }
      store8(out + (slot0 + j) * step + head * c.dim, part, c.dim, x);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) kv_read_kernel(const ReadParams p) {
  __shared__ uint32_t turn[kTurnWords];
  if (blockIdx.z)
    read_block<T, true>(p, turn);
  else
    read_block<T, false>(p, turn);
}

// Heads for one CTA of a read: as many as leave nine CTAs to an SM (a power of two, so that little is left over). One head
// each against this: 51 and 35 us for twelve prefixes of 4096 (bf16), 25.5 and 22 us for six of 2731 (f32); eight
// heads each, 36 us for the former.
int heads_for(int64_t pieces, int heads, int sms) {
  int each = 1;
  while (each < heads && pieces * 2 * ceil_div(heads, 2 * each) >= 9LL * sms) each *= 2;
  return each;
}

// New tokens a sequence, on average, up to which a warp takes a block. 64 sequences: 3 tokens each 8.4 against 13.9 us (blocks
// of 64), 7 tokens each 15.7 against 15.3 and, in blocks of 16, 10.7 against 8.1.
constexpr int64_t kFewTokens = 4;

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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d.rows <= kFewTokens * d.batch) {
    const dim3 grid(static_cast<unsigned>(pieces), static_cast<unsigned>(ceil_div(2 * d.cache.heads, 8)));
    if (d.dtype == B200_F32 && d.cache.dim == 64)
      kv_append_few_kernel<float, 2><<<grid, 256, 0, s>>>(p);
    else if (d.dtype == B200_F32)
      kv_append_few_kernel<float, 4><<<grid, 256, 0, s>>>(p);
    else if (d.cache.dim == 64)
      kv_append_few_kernel<__nv_bfloat16, 2><<<grid, 256, 0, s>>>(p);
    else
      kv_append_few_kernel<__nv_bfloat16, 4><<<grid, 256, 0, s>>>(p);
    return launched();
  }
  const dim3 grid(static_cast<unsigned>(pieces), static_cast<unsigned>(d.cache.heads), 2);
  const unsigned threads = static_cast<unsigned>(d.cache.block_tokens / 4 * (d.cache.dim / 8));
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
  p.heads_each = heads_for(pieces, d.cache.heads, device_info().sm_count);
  const dim3 grid(static_cast<unsigned>(pieces), static_cast<unsigned>(ceil_div(d.cache.heads, p.heads_each)), 2);
  const unsigned threads = static_cast<unsigned>(d.cache.block_tokens / 4 * (d.cache.dim / 8));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d.dtype == B200_F32)
    kv_read_kernel<float><<<grid, threads, 0, s>>>(p);
  else
    kv_read_kernel<__nv_bfloat16><<<grid, threads, 0, s>>>(p);
  return launched();
}
