// Ragged sequences whose lengths lie in device memory: which sequence a block of the grid
// works on. The host knows only totals, so grids are sized by a bound on the number of
// pieces and every block finds its own piece (or that there is none for it) from the
// lengths. A warp scans 32 sequences at a time; one load of the lengths is all that a
// batch of up to 32 sequences costs.
#pragma once

#include "common.cuh"

namespace b200 {
namespace {

// Bits of the kernel status word raised by the operators on ragged sequences.
constexpr int kErrOffsets = 256;  // offsets that decrease or leave the packed tensor
constexpr int kErrBlocks = 512;   // a block number outside the cache, or a length beyond the block table

struct Piece {
  int32_t sequence;  // -1: none
  int64_t index;     // of the piece within its sequence
};

// The `target`-th piece when sequence b consists of count(b) >= 0 pieces, one sequence after the
// other. All 32 lanes call it together and get the same answer. Each lane first sums a 32nd of the
// sequences (independent loads: one memory latency, whatever the batch), then the lanes go through the
// 32nd that the piece lies in.
template <class Count>
__device__ __forceinline__ Piece find_piece(int32_t batch, int64_t target, const Count& count) {
  const int lane = threadIdx.x & 31;
  const int32_t share = (batch + 31) / 32;
  auto upto_lane = [&](int64_t mine) {  // inclusive sum over the lanes
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t other = __shfl_up_sync(0xffffffffu, mine, o);
      if (lane >= o) mine += other;
    }
    return mine;
  };
  int64_t mine = 0;
#pragma unroll 4
  for (int32_t i = 0; i < share; ++i)
    if (lane * share + i < batch) mine += count(lane * share + i);
  int64_t upto = upto_lane(mine);
  const unsigned past = __ballot_sync(0xffffffffu, upto > target);
  if (!past) return Piece{-1, target - __shfl_sync(0xffffffffu, upto, 31)};
  int32_t first = __ffs(past) - 1;
  int64_t before = __shfl_sync(0xffffffffu, upto - mine, first);
  first *= share;
  for (int32_t base = first; share > 1; base += 32) {
    mine = base + lane < min(first + share, batch) ? count(base + lane) : 0;
    upto = before + upto_lane(mine);
    const unsigned here = __ballot_sync(0xffffffffu, upto > target);
    if (here) {
      first = base + __ffs(here) - 1;
      before = __shfl_sync(0xffffffffu, upto - mine, __ffs(here) - 1);
      break;
    }
    before = __shfl_sync(0xffffffffu, upto, 31);
  }
  return Piece{first, target - before};
}

// Rows [begin, begin + count) of sequence b in a packed tensor of `total` rows. Offsets that
// decrease or reach outside the tensor leave the sequence empty and raise a status bit.
struct Rows {
  int64_t begin, count;
};
__device__ __forceinline__ Rows rows_of(const int32_t* offsets, int32_t b, int64_t total, int32_t* status) {
  const int64_t begin = offsets[b], end = offsets[b + 1];
  if (begin < 0 || end < begin || end > total) {
    if (status) atomicOr(status, kErrOffsets);
    return Rows{0, 0};
  }
  return Rows{begin, end - begin};
}
// The rows behind the last sequence, which the operators fill with zeros.
__device__ __forceinline__ Rows rows_behind(const int32_t* offsets, int32_t batch, int64_t total) {
  const int64_t end = offsets[batch];
  return end < 0 || end > total ? Rows{0, 0} : Rows{end, total - end};
}

}  // namespace
}  // namespace b200
