// What the kernels over a paged KV cache share (paged.hip, paged_tree.hip):
// checks of device-held indices and the runs that a ragged batch is cut into.
#pragma once

#include <cfloat>

#include "cascade_device.h"
#include "cascade_internal.h"

namespace cascade {

__device__ __forceinline__ void flag_range(int32_t *error) {
  if (error != nullptr)
    __hip_atomic_fetch_or(error, CASCADE_PAGED_ERANGE, __ATOMIC_RELAXED,
                          __HIP_MEMORY_SCOPE_AGENT);
}

struct PagedAttnArgs {
  const uint16_t *q;  // batch row b, head h at b * q_token + h * q_head
  int64_t q_token, q_head;
  const uint16_t *k_pages, *v_pages;
  int64_t page_stride, head_stride;
  int32_t num_pages;
  int32_t page_shift;
  const int32_t *table;
  int64_t table_stride;
  int64_t sequences;
  const int32_t *lengths;
  const int32_t *rows;  // nullable: batch row b reads table row b
  int32_t batch;
  int32_t max_length;
  int32_t kv_heads;
  int32_t group;  // query heads a KV head, at most 16
  float scale_log2;
  uint16_t *out;  // [batch, q_heads, dim]
  int64_t out_token, out_head;
  int32_t *error;
  // split runs (SPLIT kernels): see "Runs"
  double per_round, per_two;  // 1 / runs wanted, in one round and in two
  int32_t *plan;    // [batch][2]: first run of a batch row, and how many
  // [run][q_heads][2]: maximum (of scores as they are summed for trees, in powers
  // of two for single tokens), sum; of trees [run][node][q_heads], part_acc too
  float *part_ml;
  float *part_acc;  // [run][q_heads][D]
  int32_t runs;     // that the workspace holds
};

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kPagedWaves = 4;   // of a workgroup that takes a run
constexpr int kWholeBlocks = 16;  // rows of at most this many blocks are not split
constexpr int kPagedBlock = 32;  // positions a wave step
constexpr int kPagedGroup = 16;  // MFMA columns
constexpr int kPagedMinRun = 4;  // blocks
constexpr double kPagedLongRun = 100.0;  // blocks
constexpr size_t kPagedAlign = 256;

__device__ __forceinline__ float paged_exp2(float x) {
  return __builtin_amdgcn_exp2f(x);
}

// Table row and length of batch row b.  row < 0: nothing to do.
struct PagedRow {
  int64_t row;
  int32_t len;
};

// Runs.  The lengths are on the device, so the launch is sized for any of
// them and each workgroup finds its own piece of work: the blocks of 32
// positions of all batch rows are cut into runs of `size` blocks,
//   size = max(kPagedMinRun, floor(blocks of all rows / wanted) + 1),
// rounded up to the workgroup's waves, and row b gets max(1, ceil(blocks_b /
// size)) runs, numbered through the batch.  There are at most wanted + batch
// runs whatever the lengths, all but a row's last of one size, so a ragged
// batch and a single long sequence both fill the device.  Every wave works
// this out for itself from the lengths (64 rows at a time), with no barrier.
// Wanted is one round of workgroups where rows get three runs or more; two
// rounds otherwise, and where one makes runs of more than 100 blocks: uneven
// ends then cost more than a second start (8 KV heads of 128: 3 sequences of
// up to 20000 positions 22.4 us in one round and 25.8 in two, 16 of 4096 27.8
// and 30.0, 64 of 2000 52.9 and 49.7, 64 of 16384 327 and 320).
struct PagedRun {
  int b;      // batch row; -1: no such run
  int64_t row;
  int len;
  int first;  // blocks [first, end) of the row
  int end;
  int count;  // runs of the row
};

__device__ __forceinline__ int blocks_of(int len) {
  return (len + kPagedBlock - 1) / kPagedBlock;
}

// The run's place; `first` (one wave of the launch) also flags what is out of
// range and writes the plan for the launch that joins the runs.
// row_of(b, flag): batch row b.
template <typename RowOf>
__device__ __forceinline__ PagedRun find_run(const PagedAttnArgs &a, int run, int lane,
                                             bool first, RowOf row_of) {
  // the first 64 rows stay in registers
  const PagedRow head = row_of(lane, first);
  unsigned long long blocks = static_cast<uint32_t>(blocks_of(head.len));
  for (int base = kWave; base < a.batch; base += kWave)
    blocks += static_cast<uint32_t>(blocks_of(row_of(base + lane, first).len));
  blocks = lane_u64(wave_prefix(blocks), kWave - 1);
  // more than blocks / target, in fp64 (no row has more than 2^26 blocks)
  double per_run = static_cast<double>(blocks) * a.per_round;
  if (per_run > kPagedLongRun) per_run = static_cast<double>(blocks) * a.per_two;
  const int want = static_cast<int>(fmin(per_run, 67108864.0 - kPagedWaves)) + 1;
  const int size = max((want + kPagedWaves - 1) / kPagedWaves * kPagedWaves, kPagedMinRun);
  PagedRun out{-1, -1, 0, 0, 0, 0};
  int before = 0;
  for (int base = 0; base < a.batch; base += kWave) {
    const PagedRow r = base == 0 ? head : row_of(base + lane, false);
    const int mine = r.row < 0 ? 0 : max(1, (blocks_of(r.len) + size - 1) / size);
    const int upto = before + wave_prefix(mine);
    if (first && base + lane < a.batch) {
      a.plan[2 * (base + lane)] = upto - mine;
      a.plan[2 * (base + lane) + 1] = mine;
    }
    const uint64_t past = __ballot(upto > run);
    if (out.b < 0 && past != 0) {
      const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
      out.b = base + at;
      out.row = __builtin_amdgcn_readlane(static_cast<int>(r.row), at);
      out.len = __builtin_amdgcn_readlane(r.len, at);
      out.count = __builtin_amdgcn_readlane(mine, at);
      const int place = run - (__builtin_amdgcn_readlane(upto, at) - out.count);
      out.first = place * size;
      out.end = min(out.first + size, blocks_of(out.len));
      if (!first) return out;
    }
    before = __builtin_amdgcn_readlane(upto, kWave - 1);
  }
  return out;
}

// Threads that one launch can have.
constexpr int64_t kMaxThreads = 0xffffffff;

inline bool page_shift_of(int64_t page_size, int32_t *shift) {
  if (page_size < 8 || page_size > 1024 || (page_size & (page_size - 1))) return false;
  *shift = __builtin_ctzll(static_cast<unsigned long long>(page_size));
  return true;
}

inline bool stride_ok(int64_t stride) { return stride >= 0 && (stride & 7) == 0; }

}  // namespace cascade
