// Drafted trees over a KV cache kept in pages (gfx950): attention of every
// node over the past and its own ancestors, and the acceptance of the nodes
// that the drawn tokens follow, with the move of their K and V rows.
//
// Tree b holds n <= 64 nodes, rows starts[b] .. of the step, and sits at the
// last n of the lengths[row] positions of its sequence: "past" below is what
// lies before it.  As everywhere over pages, device-held indices are checked
// before they form an address.
#include <cmath>

#include "paged_device.h"

namespace cascade {

constexpr int kTreeNodes = 64;  // one mask word, one node a lane

struct TreeArgs : PagedAttnArgs {
  const int32_t *starts;
  const int64_t *masks;
  int64_t tokens;
  int32_t max_tree;
  int32_t col_groups;      // workgroups that share a run of a KV head
  uint32_t sign;           // flips the signs of q: scale_log2 is not negative
  float slack;             // in raw scores, see the running maximum
  uint32_t group_inverse;  // column / group = column * group_inverse >> 16
};

struct Tree {
  int64_t row;  // < 0: nothing to do
  int32_t first;  // of its q rows
  int32_t nodes;
};

// Tree b's place among the step's rows, if it has any.
__device__ __forceinline__ Tree tree_of(const int32_t *starts, const int32_t *rows,
                                        int64_t tokens, int max_tree, int64_t b,
                                        int32_t *error) {
  Tree t{-1, 0, 0};
  const int64_t first = starts[b], end = starts[b + 1];
  const int64_t row = rows != nullptr ? rows[b] : b;
  if (row < 0) return t;
  if (first < 0 || end < first || end > tokens || end - first > max_tree) {
    flag_range(error);
    return t;
  }
  t.row = row;
  t.first = static_cast<int32_t>(first);
  t.nodes = static_cast<int32_t>(end - first);
  return t;
}

// ------------------------------------------------------------- attention
// A tree and the length of its sequence, if both are in range.
struct TreeRow {
  PagedRow place{-1, 0};
  int32_t first = 0, nodes = 0;
};

__device__ __forceinline__ TreeRow tree_row(const TreeArgs &a, int b, bool flag) {
  TreeRow r;
  if (b >= a.batch) return r;
  int32_t *error = flag ? a.error : nullptr;
  // (the loads side by side: the length's does not wait for the checks)
  const int64_t row = a.rows != nullptr ? a.rows[b] : b;
  const int32_t len = row >= 0 && row < a.sequences ? a.lengths[row] : -1;
  const Tree t = tree_of(a.starts, a.rows, a.tokens, a.max_tree, b, error);
  if (t.row < 0 || t.nodes == 0) return r;
  if (len < t.nodes || len > a.max_length) {
    flag_range(error);
    return r;
  }
  r.place = {t.row, len};
  r.first = t.first;
  r.nodes = t.nodes;
  return r;
}

// Lane l's 16 bytes at base + voff land at LDS byte lds + 16 l (dma_lds16 for
// a base of 64 bits).
__device__ __forceinline__ void dma_lds16_from(uint64_t base, uint32_t voff, uint32_t lds,
                                               bool once) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(base));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(base >> 32));
  const uint64_t at = (static_cast<uint64_t>(hi) << 32) | lo;
  if (once)
    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2 nt"
                 :: "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(at)
                 : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :: "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(at)
                 : "memory", "m0");
}

template <int DIM, int CT_, int WC_, int WP_>
struct TreeShape {
  static constexpr int D = DIM, CT = CT_, WC = WC_, WP = WP_;
  static constexpr int WAVES = WC * WP;
  static constexpr int COLS = 16 * CT * WC;  // of a workgroup
  // Rows that no other workgroup reads need no place in a cache: 64 trees of 8
  // nodes over up to 4096 positions 131 -> 118 us, one of 16 over 32768 45.9 ->
  // 45.2 (heads of 64 27.3 -> 28.6).  Of 16 tiles the workgroups may share rows.
  static constexpr bool ONCE = CT * WC < 16;
  static constexpr int KC = D / 32;          // 32-dim chunks
  static constexpr int DV = D / 16;          // tiles of 16 dims
  static constexpr int ROW = 2 * D;          // bytes
  static constexpr int TILE = kPagedBlock * ROW;
  static constexpr int SLOT = 2 * TILE;      // K and V of a block
  static constexpr int LOADS = SLOT / 1024 / WC;  // of a wave
  // Workgroups a CU, in whose share of the LDS the slots have to fit: two that
  // wait at barriers of their own are worth more than one with twice the waves
  // and slots (19 sequences of up to 2048 positions, 14 heads of 64, 9 nodes:
  // 26.7 -> 19.8 us; 64 of up to 4096, 8 nodes: 128 -> 118).  Sixteen tiles take
  // all registers, four groups of 128 dims all of the LDS.
  static constexpr int PAIR = CT * WC <= 8 && 4 * WP * SLOT <= 160 * 1024 - 32 ? 2 : 1;
  static constexpr int FIT = (160 * 1024 / PAIR - 16) / (WP * SLOT);
  static constexpr int COUNT = 63 / LOADS + 2, FEW = FIT < COUNT ? FIT : COUNT;
  static constexpr int DEPTH = FEW < 5 ? FEW : 5;  // slots
  static constexpr int PITCH = D + 4;  // floats of a column where the groups join
  static constexpr int SUMS = WAVES * 16 * (PITCH * 4 + 8);
  static constexpr int LDS = DEPTH * WP * SLOT > SUMS ? DEPTH * WP * SLOT : SUMS;
  static_assert(DEPTH >= 2 && LDS <= 160 * 1024 && LOADS >= 1, "shape");
};

// The columns of 16 query rows in a wave.
template <int DV>
struct TreeColumns {
  float m, l;
  f32x4 o[DV];
};

// The halves of a pair of bf16 values that are infinities or NaN, as a mask.
__device__ __forceinline__ uint32_t special_of(uint32_t pair) {
  return ((pair & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) |
         ((pair & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
}

// Sixteen lanes read 4 rows of 16 values, eight bytes each, and get a column
// each, four values.
__device__ __forceinline__ u32x2 read_turned(const unsigned char *from) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(
      u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                 (__attribute__((address_space(3))) s16x4 *)(from)));
}

// Two weights as sums of three bf16 values each, cut off one after the other:
// 8 bits each of the 24 that fp32 has, so nothing is rounded.
struct WeightParts {
  uint32_t upper, middle, lower;
};

__device__ __forceinline__ WeightParts tree_weights(float a, float b) {
  auto cut = [&] {
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
  };
  WeightParts w;
  w.upper = cut();
  a -= lo_bf16(w.upper);
  b -= hi_bf16(w.upper);
  w.middle = cut();
  a -= lo_bf16(w.middle);
  b -= hi_bf16(w.middle);
  w.lower = cut();
  return w;
}

// One workgroup takes the columns (node, query head of the KV head) of a tree
// and a run of its sequence's blocks of 32 positions, which find_run cuts out of
// all trees' blocks.  WP groups of waves take turns at the blocks; a group's K
// and V rows come into LDS once, by loads that go there directly into a ring of
// slots, and its WC waves multiply them with 16 CT columns each:
//   S^T = K q^T, running maximum m and sum l a column, O^T += V^T P^T,
// all on the matrix cores, S, m, l and O in fp32, and P as three bf16 parts, which
// are all of its bits.  Two parts are 2^-16 off: enough to turn the rounding of
// one result in 500 (rows 1.3e-4 from those of exact weights in the mean, 0.5e-4
// with three, which is what the order of fp32 sums does), for 15% of the time
// of wide trees (24 of up to 63 nodes 332 us and 390) and 2 to 8% of others'.
// K and V rows lie swizzled in LDS, K for plain reads of its operands, V for
// reads that turn 4 x 16 values.  The reference of the exponents follows the
// maximum only where it is passed by 2^8, so O is rarely scaled, and the next
// block's K operands are read beside this block's product with V.
//
// What bounds it: to 64 columns or so the loads, 64 trees of 8 nodes over up to
// 4096 positions (606 MB) 117 us, 5.2 TB/s, one of 16 over 32768 (135 MB) 39 us
// with the join of its runs (the start, page lookups and the join are 14 of it);
// above, vector and matrix instructions, which two waves of a SIMD hardly overlap:
// a wave's block of 32 columns is 64 MFMAs (1024 cycles) and 200 vector
// instructions (900, a sixth of them exponentials), a block of 256 columns 2.0 us;
// 24 trees of up to 63 nodes over up to 16384 positions (885 MB) 390 us. With two
// parts of P, lookups of sixteen blocks' pages at a time, lane by lane, and
// operands read ahead took that from 570 us to 355, V's turned reads in place of
// 32 permutations a block to 326.
template <typename T, bool SPLIT>
__global__ __launch_bounds__(T::WAVES * kWave) void tree_attention_kernel(TreeArgs a) {
  constexpr int D = T::D, CT = T::CT, WC = T::WC, WP = T::WP;
  constexpr int KC = T::KC, DV = T::DV, ROW = T::ROW;
  __shared__ __attribute__((aligned(16))) unsigned char s_mem[T::LDS];
  __shared__ int s_special;  // the first block whose infinities and NaN were left out
  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int wc = wave % WC, wp = wave / WC;
  const int c16 = lane & 15, g4 = lane >> 4;
  const int kv = static_cast<int>(blockIdx.x) % a.kv_heads;
  const int rest = static_cast<int>(blockIdx.x) / a.kv_heads;
  const int cg = rest % a.col_groups, run = rest / a.col_groups;
  int b = run, len, first = 0, end, count = 1, token0, nodes;
  int64_t row;
  {
    const bool flags = blockIdx.x == 0 && wave == 0;
    if constexpr (SPLIT) {
      TreeRow head;  // of the first 64 trees, a lane each
      auto row_of = [&](int i, bool flag) {
        const TreeRow r = tree_row(a, i, flag);
        if (i == lane) head = r;
        return r.place;
      };
      const PagedRun r = find_run(a, run, lane, flags, row_of);
      if (r.b < 0) return;
      b = r.b;
      row = r.row;
      len = r.len;
      first = r.first;
      end = r.end;
      count = r.count;
      if (b < kWave) {
        token0 = __builtin_amdgcn_readlane(head.first, b);
        nodes = __builtin_amdgcn_readlane(head.nodes, b);
      } else {
        token0 = a.starts[b];
        nodes = a.starts[b + 1] - token0;
      }
    } else {
      const TreeRow r = tree_row(a, b, kv == 0 && cg == 0 && tid == 0);
      if (r.place.row < 0) return;
      row = r.place.row;
      len = r.place.len;
      end = blocks_of(len);
      token0 = r.first;
      nodes = r.nodes;
    }
  }
  row = __builtin_amdgcn_readfirstlane(static_cast<int>(row));
  len = __builtin_amdgcn_readfirstlane(len);
  b = __builtin_amdgcn_readfirstlane(b);
  first = __builtin_amdgcn_readfirstlane(first);
  end = __builtin_amdgcn_readfirstlane(end);
  token0 = __builtin_amdgcn_readfirstlane(token0);
  nodes = __builtin_amdgcn_readfirstlane(nodes);
  const int cols = nodes * a.group;
  const int col0 = cg * T::COLS;
  if (col0 >= cols) return;
  const int mine = col0 + 16 * CT * wc;  // the wave's first column
  const int past = len - nodes, last = len - 1;
  const uint64_t kb = reinterpret_cast<uint64_t>(a.k_pages + kv * a.head_stride);
  const uint64_t vb = reinterpret_cast<uint64_t>(a.v_pages + kv * a.head_stride);
  const int page_mask = (1 << a.page_shift) - 1;
  const uint32_t lds = lds_address(s_mem);
  const uint32_t ring = wp * T::DEPTH * T::SLOT;

  // A lane's place in a load of 1 KiB: its row, and its 16 bytes of it.  Row r
  // of a block keeps its chunk ch at ch ^ key(r), where the keys of the 16 rows
  // of an operand differ (of the eight of one parity, for 64 dims: two rows
  // share the banks).
  constexpr int CH = D / 8;
  const int lrow = lane / CH, lch = lane % CH;
  // The pages of sixteen of the wave's blocks, a lane a group of eight positions:
  // what the group's rows lie behind the pools' start, and a bit a bad page.
  const int steps = (end - first + WP - 1) / WP;  // of the workgroup
  // (past the run's end its last block again, which takes no part)
  auto block_of = [&](int step) { return min(first + step * WP + wp, end - 1); };
  const int32_t *table = a.table + row * a.table_stride;
  auto entry_of = [&](int step) {  // of the lane, in the sixteen steps from `step` on
    return table[min(block_of(step + (lane >> 2)) * kPagedBlock + 8 * (lane & 3), last) >>
                 a.page_shift];
  };
  struct Pages {
    uint32_t lo, hi;
    uint64_t bad;
  };
  auto pages_of = [&](int step, int page) {
    Pages p;
    const bool good = page >= 0 && page < a.num_pages;
    const int slot = (block_of(step + (lane >> 2)) * kPagedBlock + 8 * (lane & 3)) & page_mask;
    const uint64_t at = static_cast<uint64_t>(good ? page : 0) *
                            static_cast<uint64_t>(2 * a.page_stride) +
                        static_cast<uint64_t>(slot * ROW);
    p.lo = static_cast<uint32_t>(at);
    p.hi = static_cast<uint32_t>(at >> 32);
    p.bad = __ballot(!good);
    return p;
  };
  // A wave's loads: K's and V's of all groups, or one of them, or that of some.
  constexpr int kGroups = WC <= 2 ? 4 : 8 / WC;  // that a wave loads
  constexpr int kHalves = D / 64;                // loads of a group
  const int group0 = (wc >> 1) * kGroups;
  auto v_off = [&](int grp, int h) {
    const uint32_t key = D == 128 ? 2 * lrow + 8 * (grp & 1) : (lrow & 2) + 4 * (grp & 1);
    return h * 1024 + lrow * ROW + ((lch ^ key) << 4);
  };
  uint32_t k_off[kGroups][kHalves];
#pragma unroll
  for (int g = 0; g < kGroups; ++g)
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      const int grp = group0 + g;
      const uint32_t key = D == 128 ? 4 * grp + lrow : 2 * grp + ((lrow >> 1) & 1);
      k_off[g][h] = h * 1024 + lrow * ROW + ((lch ^ key) << 4);
      if (WC > 1 && (wc & 1)) k_off[g][h] = v_off(grp, h);  // this wave loads V
    }
  Pages pages = pages_of(0, entry_of(0));
  int entry = entry_of(16);
  uint32_t all_bad = 0;
  // Starts the loads of step `step` (they are asked for in order) into a slot.
  auto issue = [&](int step, int slot) __attribute__((always_inline)) {
    const int at = (step & 15) * 4;
    if (at == 0 && step != 0) {
      pages = pages_of(step, entry);
      entry = entry_of(step + 16);
    }
    const uint32_t to = lds + ring + slot * T::SLOT;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const int grp = group0 + g;
      const uint64_t behind =
          (static_cast<uint64_t>(__builtin_amdgcn_readlane(pages.hi, at + grp)) << 32) |
          static_cast<uint32_t>(__builtin_amdgcn_readlane(pages.lo, at + grp));
#pragma unroll
      for (int kvs = 0; kvs < (WC == 1 ? 2 : 1); ++kvs) {
        const bool is_v = WC == 1 ? kvs : wc & 1;
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
          dma_lds16_from((is_v ? vb : kb) + behind,
                         WC == 1 && kvs ? v_off(grp, h) : k_off[g][h],
                         to + (is_v ? T::TILE : 0) + (grp * kHalves + h) * 1024, T::ONCE);
      }
    }
    return static_cast<uint32_t>(pages.bad >> at) & 0xfu;
  };
  uint32_t bads = 0;  // bad pages of the blocks under way, four bits a step
  for (int d = 0; d < T::DEPTH; ++d) bads |= issue(d, d) << (4 * d);

  // the q operands, zeros past the tree's columns
  u32x4 q[CT][KC];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int col = mine + 16 * ct + c16;
    const int node = static_cast<int>((static_cast<uint32_t>(col) * a.group_inverse) >> 16);
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const int64_t at = (token0 + min(node, nodes - 1)) * a.q_token +
                         (static_cast<int64_t>(kv) * a.group +
                          (col < cols ? col - node * a.group : 0)) * a.q_head;
      u32x4 x = *reinterpret_cast<const u32x4 *>(a.q + at + 32 * c + 8 * g4);
      x ^= a.sign;
      q[ct][c] = col < cols ? x : u32x4{0u, 0u, 0u, 0u};
    }
  }

  if (tid == 0) s_special = end;
  TreeColumns<DV> state[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    state[ct].m = -FLT_MAX;
    state[ct].l = 0.0f;
#pragma unroll
    for (int e = 0; e < DV; ++e) state[ct].o[e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const int krow = 8 * (c16 >> 2) + (c16 & 3);
  const int kkey = D == 128 ? c16 : 2 * (c16 >> 2) + ((c16 >> 1) & 1);
  // of the 16 lanes of a turned read of 4 rows and 16 dims: row 8 g4 + c16 / 4,
  // four dims from 4 (c16 % 4) on
  const int vkey = D == 128 ? 2 * (c16 >> 2) + 8 * (g4 & 1) : ((c16 >> 2) & 2) + 4 * (g4 & 1);
  const int v_at = (8 * g4 + (c16 >> 2)) * ROW + ((((c16 >> 1) & 1) ^ vkey) << 4) + 8 * (c16 & 1);

  u32x4 k0[KC], k1[KC];  // the next block's K operands
  auto read_k = [&](int slot) __attribute__((always_inline)) {
    const unsigned char *at = s_mem + ring + slot * T::SLOT;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const unsigned char *kp = at + krow * ROW + (((4 * c + g4) ^ kkey) << 4);
      k0[c] = *reinterpret_cast<const u32x4 *>(kp);
      k1[c] = *reinterpret_cast<const u32x4 *>(kp + 4 * ROW);
    }
  };
  // The next step's loads are here, and everyone has read this step's slot (its
  // reads have ended, not only begun: lgkmcnt), which
  // takes the loads of the step that is DEPTH behind it (no fence: it would
  // wait for all loads).
  auto turn = [&](int i, int slot) __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(waitcnt_imm((T::DEPTH - 2) * T::LOADS, 0));
    if constexpr (WC > 1) __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    bads = (bads >> 4) | (issue(i + T::DEPTH, slot) << (4 * (T::DEPTH - 1)));
    __builtin_amdgcn_sched_barrier(0);
  };
  auto step = [&](int i, int slot) __attribute__((always_inline)) {
    const int blk = first + i * WP + wp;
    const bool gone = blk >= end;  // (a group's last turn, where others have one)
    const uint32_t bad = gone ? 0xfu : bads & 0xfu;
    all_bad |= gone ? 0u : bad;
    // a block with positions of the tree or past the end, or with a bad page
    const bool tail = bad || (blk + 1) * kPagedBlock > past;
    const unsigned char *at = s_mem + ring + slot * T::SLOT;
    const int r0 = blk * kPagedBlock;
    // V's operands, dim 16 e + c16 of eight positions, as the reads turn them
    u32x4 vop[DV];
#pragma unroll
    for (int e = 0; e < DV; ++e) {
      const unsigned char *vp = at + T::TILE + (v_at ^ (32 * e));
      const u32x2 lo = read_turned(vp), hi = read_turned(vp + 4 * ROW);
      vop[e] = u32x4{lo[0], lo[1], hi[0], hi[1]};
    }
    f32x4 score[CT][2];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
      score[ct][0] = score[ct][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        score[ct][0] = mfma_16x16x32_bf16(k0[c], q[ct][c], score[ct][0]);
        score[ct][1] = mfma_16x16x32_bf16(k1[c], q[ct][c], score[ct][1]);
      }
    const bool mine_bad = (bad >> g4) & 1;
    float s[CT][8];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int j = 0; j < 8; ++j) s[ct][j] = score[ct][j >> 2][j & 3];
    if (tail) {
      // Rows past the end, or of a page outside the pool, take no part
      // whatever they hold.  An infinity or a NaN of a row that a column does not see must not
      // reach it, and 0 times one is a NaN: they are left out here, and
      // added where the columns are joined, to those that see them.
      uint32_t any = 0;
#pragma unroll
      for (int e = 0; e < DV; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at_row = r0 + 8 * g4 + 2 * i;
          const uint32_t in = mine_bad ? 0u : (at_row < len ? 0xffffu : 0u) |
                                                  (at_row + 1 < len ? 0xffff0000u : 0u);
          const uint32_t pair = vop[e][i] & in, bits = special_of(pair);
          any |= bits;
          vop[e][i] = pair & ~bits;
        }
      if (any != 0) atomicMin(&s_special, blk);
    }
    if (tail) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const int col = mine + 16 * ct + c16;
        const int node =
            static_cast<int>((static_cast<uint32_t>(col) * a.group_inverse) >> 16);
        uint64_t mask = col < cols ? static_cast<uint64_t>(a.masks[token0 + node]) : 0;
        if (nodes < kTreeNodes) mask &= (uint64_t{1} << nodes) - 1;
        // bit j: the column sees position r0 + 8 g4 + j
        const int rel = r0 + 8 * g4 - past;
        uint64_t bits = 0xffu;
        if (rel >= kTreeNodes)
          bits = 0;
        else if (rel >= 0)
          bits = mask >> rel;
        else if (rel > -8)
          bits = (mask << -rel) | ((1u << -rel) - 1);
        const uint32_t sees = mine_bad ? 0u : static_cast<uint32_t>(bits);
#pragma unroll
        for (int j = 0; j < 8; ++j) s[ct][j] = (sees >> j) & 1 ? s[ct][j] : -INFINITY;
      }
      // (nothing is left under way that a wait behind this would be for)
      __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 15));
    }
    // The reference of the exponents follows the maximum where it is passed by
    // more than 2^8: until then weights stay in fp32's range, and the columns
    // keep their scale.
    float bmax[CT];
    bool passed = false;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      bmax[ct] = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j) bmax[ct] = fmaxf(bmax[ct], s[ct][j]);
      bmax[ct] = xor32_max(xor16_max(bmax[ct]));
      passed |= bmax[ct] > state[ct].m + a.slack;
    }
    if (__any(passed)) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        TreeColumns<DV> &x = state[ct];
        const float m = bmax[ct] > x.m ? bmax[ct] : x.m;
        const float alpha = paged_exp2((x.m - m) * a.scale_log2);
        x.m = m;
        x.l *= alpha;
#pragma unroll
        for (int e = 0; e < DV; ++e) x.o[e] *= alpha;
      }
    }
    u32x4 upper[CT], middle[CT], lower[CT];
    auto weights = [&](int ct) __attribute__((always_inline)) {
      TreeColumns<DV> &x = state[ct];
      // (a masked score's -inf stays so)
      const float base = fminf(-x.m * a.scale_log2, FLT_MAX);
      float p[8], psum = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = paged_exp2(fmaf(s[ct][j], a.scale_log2, base));
#pragma unroll
      for (int j = 0; j < 8; ++j) psum += p[j];
      x.l += psum;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const WeightParts w = tree_weights(p[2 * n], p[2 * n + 1]);
        upper[ct][n] = w.upper;
        middle[ct][n] = w.middle;
        lower[ct][n] = w.lower;
      }
    };
    weights(0);
    turn(i, slot);
    read_k(slot == T::DEPTH - 1 ? 0 : slot + 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      TreeColumns<DV> &x = state[ct];
#pragma unroll
      for (int e = 0; e < DV; ++e) {
        x.o[e] = mfma_16x16x32_bf16(vop[e], lower[ct], x.o[e]);
        x.o[e] = mfma_16x16x32_bf16(vop[e], middle[ct], x.o[e]);
        x.o[e] = mfma_16x16x32_bf16(vop[e], upper[ct], x.o[e]);
      }
      if (ct + 1 < CT) weights(ct + 1);
    }
    if constexpr (CT > 1) {
      // a tile's product with V beside the next one's weights
#pragma unroll
      for (int n = 0; n < 3 * DV * (CT - 1); ++n) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x8, 3 * DV, 0);
    }
  };

  // (the q rows are here: no wait for them inside the loop)
  __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
  __builtin_amdgcn_s_barrier();
  auto next_slot = [](int slot) { return slot == T::DEPTH - 1 ? 0 : slot + 1; };
  if (mine < cols) {
    read_k(0);
    for (int i = 0, slot = 0; i < steps; ++i, slot = next_slot(slot)) step(i, slot);
  } else {
    // (columns that this tree has not: the wave's loads alone)
    for (int i = 0, slot = 0; i < steps; ++i, slot = next_slot(slot)) {
      all_bad |= first + i * WP + wp < end ? bads & 0xfu : 0u;
      turn(i, slot);
    }
  }
  __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
  __syncthreads();
  if (all_bad && lane == 0) flag_range(a.error);

  // Writes eight dims of a column from their sums and the weights' sum, or,
  // where the tree has more runs, what these are joined from.
  auto put = [&](int col, int d, float m, float den, f32x4 (&sum)[2]) __attribute__((always_inline)) {
    const int node = static_cast<int>((static_cast<uint32_t>(col) * a.group_inverse) >> 16);
    const int head = kv * a.group + col - node * a.group;
    // Infinities and NaN of V: the blocks with the tree or a bad page left theirs
    // out, and in the others a part of a weight that is zero may have made an
    // infinity a NaN.
    int from = s_special;
    if (den < INFINITY)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (!(fabsf(sum[i / 4][i % 4]) < INFINITY)) from = first;
    if (from < end) {
      const uint64_t mask = static_cast<uint64_t>(a.masks[token0 + node]);
      const int to = min(end * kPagedBlock, len);
      f32x4 special[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
      for (int p = from * kPagedBlock; p < to; ++p) {
        const int page = table[p >> a.page_shift];
        if (page < 0 || page >= a.num_pages) continue;
        if (p >= past && !((mask >> (p - past)) & 1)) continue;
        const uint16_t *v = a.v_pages + page * a.page_stride + kv * a.head_stride +
                            static_cast<int64_t>(p & page_mask) * D + d;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float value = bf16_to_f32(v[i]);
          if (!(fabsf(value) < INFINITY)) special[i / 4][i % 4] += value;
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float value = special[i / 4][i % 4];
        if (!(fabsf(value) < INFINITY)) sum[i / 4][i % 4] = value;
      }
    }
    if (!SPLIT || count == 1) {
      const float by = den == 0.0f ? 0.0f : 1.0f / den;
      u32x4 x;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x[i] = den == 0.0f ? 0u
                           : pack_bf16x2(sum[i / 2][2 * i % 4] * by, sum[i / 2][2 * i % 4 + 1] * by);
      *reinterpret_cast<u32x4 *>(a.out + (token0 + node) * a.out_token + head * a.out_head + d) = x;
    } else {
      const int64_t at =
          (static_cast<int64_t>(run) * a.max_tree + node) * (a.kv_heads * a.group) + head;
      f32x4 *to = reinterpret_cast<f32x4 *>(a.part_acc + at * D + d);
      to[0] = sum[0];
      to[1] = sum[1];
      if (d == 0) {
        a.part_ml[2 * at] = m;
        a.part_ml[2 * at + 1] = den;
      }
    }
  };
  float sums[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) sums[ct] = xor32_sum(xor16_sum(state[ct].l));
  // The groups' columns join in LDS, one tile of them after the other.  o[e][r]
  // is O[dim 16 e + 4 g4 + r][column c16]; columns are 16 bytes further apart
  // than their dims are long, so that a lane's column has banks of its own.
  constexpr int kPitch = T::PITCH;
  float *s_acc = reinterpret_cast<float *>(s_mem);  // [wave][column][dim]
  float *s_ml = s_acc + T::WAVES * 16 * kPitch;     // [wave][column][2]
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    if (ct) __syncthreads();
#pragma unroll
    for (int e = 0; e < DV; ++e)
      *reinterpret_cast<f32x4 *>(s_acc + (wave * 16 + c16) * kPitch + 16 * e + 4 * g4) =
          state[ct].o[e];
    if (g4 == 0) {
      s_ml[(wave * 16 + c16) * 2] = state[ct].m;
      s_ml[(wave * 16 + c16) * 2 + 1] = sums[ct];
    }
    __syncthreads();
    for (int i = tid; i < WC * 2 * D; i += T::WAVES * kWave) {
      const int w = i / (2 * D), c = i / (D / 8) % 16, d = 8 * (i % (D / 8));
      const int col = col0 + 16 * (CT * w + ct) + c;
      if (col >= cols) continue;
      float mm = -FLT_MAX;
#pragma unroll
      for (int k = 0; k < WP; ++k) mm = fmaxf(mm, s_ml[((k * WC + w) * 16 + c) * 2]);
      float den = 0.0f;
      f32x4 sum[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
      for (int k = 0; k < WP; ++k) {
        const int from = (k * WC + w) * 16 + c;
        const float wt = paged_exp2((s_ml[from * 2] - mm) * a.scale_log2);
        den = fmaf(wt, s_ml[from * 2 + 1], den);
        const f32x4 *x = reinterpret_cast<const f32x4 *>(s_acc + from * kPitch + d);
        const f32x4 x0 = x[0], x1 = x[1];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          sum[0][n] = fmaf(wt, x0[n], sum[0][n]);
          sum[1][n] = fmaf(wt, x1[n], sum[1][n]);
        }
      }
      put(col, d, mm, den, sum);
    }
  }
}

// Joins the runs of a node: out = sum_r 2^(m_r - M) acc_r / sum_r 2^(m_r - M) l_r.
// D / 4 threads (four dims each) are a slice, SLICES slices a head, and each
// takes every SLICES-th run with a running maximum of its own: eight where a
// tree has more than eight runs, whose loads would follow each other, two
// otherwise.  Bound by its three dependent loads (4.6 us for one tree of 32
// runs), for large batches by the partial results (24 trees of 63 nodes: 19 us
// for 79 MB).
constexpr int kTreeMergeThreads = 256;

// A run's factor for one of its sums: an infinite one keeps its value, which a
// factor of zero would make a NaN.
__device__ __forceinline__ float run_factor(float w, float sum) {
  return fabsf(sum) < INFINITY ? w : 1.0f;
}

template <int D, int SLICES>
__global__ __launch_bounds__(kTreeMergeThreads) void tree_merge_kernel(TreeArgs a) {
  constexpr int kHeads = kTreeMergeThreads / (SLICES * D / 4);
  __shared__ f32x4 s_acc[kHeads][SLICES][D / 4];
  __shared__ float s_ml[kHeads][SLICES][2];
  const int heads = a.kv_heads * a.group;
  const int parts = (heads + kHeads - 1) / kHeads;
  const int64_t id = blockIdx.x;
  const int part = static_cast<int>(id % parts);
  const int node = static_cast<int>(id / parts % a.max_tree);
  const int b = static_cast<int>(id / parts / a.max_tree);
  const int index = a.plan[2 * b], count = a.plan[2 * b + 1];
  const int token0 = a.starts[b], past = a.starts[b + 1];
  // left out, or written already (or, past the workspace, a plan that another
  // call has overwritten)
  if (count <= 1 || index < 0 || count > a.runs - index) return;
  if (node >= past - token0) return;
  const int d = threadIdx.x % (D / 4);
  const int slice = threadIdx.x / (D / 4) % SLICES;
  const int h = threadIdx.x / (D / 4) / SLICES;
  const int head = part * kHeads + h;
  float m = -FLT_MAX, den = 0.0f;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  if (head < heads) {
    const int64_t step = static_cast<int64_t>(a.max_tree) * heads;
    const int64_t base = (static_cast<int64_t>(index) * a.max_tree + node) * heads + head;
#pragma unroll 4
    for (int r = slice; r < count; r += SLICES) {
      const int64_t at = base + r * step;
      const float2 ml = *reinterpret_cast<const float2 *>(a.part_ml + 2 * at);
      const f32x4 v = *reinterpret_cast<const f32x4 *>(a.part_acc + at * D + 4 * d);
      const float mnew = fmaxf(m, ml.x);
      const float keep = paged_exp2((m - mnew) * a.scale_log2);
      const float w = paged_exp2((ml.x - mnew) * a.scale_log2);
      m = mnew;
      den = fmaf(w, ml.y, den * keep);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        acc[i] = fmaf(run_factor(w, v[i]), v[i], acc[i] * run_factor(keep, acc[i]));
    }
  }
  s_acc[h][slice][d] = acc;
  if (d == 0) {
    s_ml[h][slice][0] = m;
    s_ml[h][slice][1] = den;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kHeads * D; i += kTreeMergeThreads) {
    const int hh = i / D, dim = i % D;
    if (part * kHeads + hh >= heads) return;
    float mm = -FLT_MAX;
#pragma unroll
    for (int k = 0; k < SLICES; ++k) mm = fmaxf(mm, s_ml[hh][k][0]);
    float sum = 0.0f, r = 0.0f;
#pragma unroll
    for (int k = 0; k < SLICES; ++k) {
      const float w = paged_exp2((s_ml[hh][k][0] - mm) * a.scale_log2);
      const float part = s_acc[hh][k][dim / 4][dim % 4];
      sum = fmaf(w, s_ml[hh][k][1], sum);
      r = fmaf(run_factor(w, part), part, r);
    }
    a.out[(token0 + node) * a.out_token + (part * kHeads + hh) * a.out_head + dim] =
        f32_to_bf16(sum == 0.0f ? 0.0f : r / sum);
  }
}

// Which shape a call takes, whether it splits, and its sizes (times in us).
// - Tiles of 16 columns: the least power of two that takes a tree of max_tree
//   nodes, to 16; more columns take workgroups of their own.
// - Split over runs up to 256 trees, which fill the device, and from so many
//   blocks on that whole trees would leave it unbalanced: 17, where the launch has
//   128 workgroups or less, to 65 at 512, in proportion (below, one workgroup is a
//   whole tree and no second launch is needed).  64 trees of 8 nodes, 8 KV heads,
//   over up to 1000 positions: 32.5 whole, 36.6 split, up to 2000 56.6 and 61.0;
//   40 trees of 4 up to 1000 26.0 and 26.3, of 60 80.7 and 94.4, of 4 up to 2000
//   49.2 and 42.4.  So of up to 256 trees none of more than 2048 positions waits
//   for one workgroup; of more trees the longest does.
// - Runs: one workgroup a CU for few trees (one over 32768 positions: of 32 nodes
//   54.7, two a CU 55.4; of 16 39.3 and 37.6; heads of 64, 4 nodes: 20.9 and
//   20.6), two where there are more trees than a third of that (16 trees of 8
//   nodes, heads of 64, over up to 4096: 22.9, one a CU 26.2, four 29.2; 19 of 9
//   over up to 2048: 19.3, one 25.5), and four where a run would pass 100 blocks
//   (24 of 63 over up to 16384: 383, two 424, one 529; 64 of 8 368, 402 and 402;
//   8 of 16 over up to 30000 123, 110 and 130).
struct TreePlan {
  int shape;  // tiles of 16 columns a workgroup: 1, 2, 4, 8, 16
  int col_groups;
  bool split;
  int64_t round, two;  // runs wanted, in one round and in two
  int64_t runs;        // at most
  size_t plan_bytes, ml_bytes, acc_bytes;

  size_t bytes() const { return kPagedAlign + plan_bytes + ml_bytes + acc_bytes; }
};

// Workgroups of a round, one a CU; up to 128 columns a CU holds two (PAIR).
constexpr int64_t kTreeSlots = 256;
constexpr int64_t kTreeMaxBatch = 256;   // of a split launch
constexpr int64_t kTreeColumns = 256;    // that a workgroup takes at most

static TreePlan tree_plan(int64_t trees, int64_t max_tree, int64_t q_heads, int64_t kv_heads,
                          int64_t dim, int64_t max_length) {
  TreePlan p{};
  const int64_t cols = max_tree * (q_heads / kv_heads);
  p.shape = cols <= 16 ? 1 : cols <= 32 ? 2 : cols <= 64 ? 4 : cols <= 128 ? 8 : 16;
  p.col_groups = static_cast<int>((cols + 16 * p.shape - 1) / (16 * p.shape));
  const int64_t blocks = (max_length + kPagedBlock - 1) / kPagedBlock;
  const int64_t each = kv_heads * p.col_groups;
  int64_t whole = kWholeBlocks * trees * each / (kTreeSlots / 2);
  whole = whole < kWholeBlocks ? kWholeBlocks : whole > 4 * kWholeBlocks ? 4 * kWholeBlocks : whole;
  p.split = blocks > whole && trees <= kTreeMaxBatch;
  if (blocks <= kWholeBlocks || trees > kTreeMaxBatch) return p;
  // (sizes for fewer trees, which are split, too)
  const int64_t slots = (kTreeSlots + each - 1) / each;
  auto wanted = [trees](int64_t runs) {
    return runs - trees / 2 > runs / 2 ? runs - trees / 2 : (runs + 1) / 2;
  };
  p.two = wanted(4 * slots);
  p.round = wanted(slots);
  if (3 * trees > p.round) p.round = wanted(2 * slots);
  p.runs = p.two + trees;
  const int64_t most = trees * ((blocks + kPagedMinRun - 1) / kPagedMinRun);
  if (p.runs > most) p.runs = most;
  auto rounded = [](int64_t bytes) {
    return (static_cast<size_t>(bytes) + kPagedAlign - 1) / kPagedAlign * kPagedAlign;
  };
  p.plan_bytes = rounded(trees * 8);
  p.ml_bytes = rounded(p.runs * max_tree * q_heads * 8);
  p.acc_bytes = rounded(p.runs * max_tree * q_heads * dim * 4);
  return p;
}

// WIDE: twice the groups of waves, for launches that leave CUs with one workgroup
// or none, which are whole trees of up to 512 positions: one tree of 16 nodes
// 14.3 us, 18.3 with fewer waves; 64 of them 34.1 and 27.9.
template <int D, bool SPLIT, bool WIDE>
static hipError_t launch_tree(const TreeArgs &a, int shape, int64_t blocks, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(blocks));
  // Groups of waves: as many as leave each two slots.  (64 dims, 64 columns: two
  // groups and one 28.6 / 33.4 us for one tree over 32768 positions; 128 dims,
  // 8 nodes of 4 heads: two groups and one 117.9 / 121.9 for 64 trees.)
  constexpr int kNarrow = WIDE || D == 64 ? 4 : 2;
#define CASCADE_TREE(CT, WC, WP)                                                     \
  {                                                                                  \
    using T = TreeShape<D, CT, WC, WP>;                                              \
    return launch_kernel(tree_attention_kernel<T, SPLIT>, grid, dim3(T::WAVES * kWave), 0, s, a); \
  }
  switch (shape) {
    case 1: CASCADE_TREE(1, 1, kNarrow)
    case 2: CASCADE_TREE(1, 2, 2)
    case 4: CASCADE_TREE(1, 4, kNarrow / 2)
    case 8: CASCADE_TREE(2, 4, WIDE ? 2 : 1)
    default: CASCADE_TREE(2, 8, 1)
  }
#undef CASCADE_TREE
}

template <int D>
static hipError_t launch_tree_merge(const TreeArgs &a, int64_t runs_a_tree, hipStream_t s) {
  const int64_t heads = static_cast<int64_t>(a.kv_heads) * a.group;
  auto grid = [&](int64_t per) {
    return dim3(static_cast<unsigned>(a.batch * static_cast<int64_t>(a.max_tree) *
                                      ((heads + per - 1) / per)));
  };
  const dim3 block(kTreeMergeThreads);
  if (runs_a_tree > 8)
    return launch_kernel(tree_merge_kernel<D, 8>, grid(128 / D), block, 0, s, a);
  return launch_kernel(tree_merge_kernel<D, 2>, grid(512 / D), block, 0, s, a);
}

// ------------------------------------------------------------ acceptance
struct AcceptArgs {
  const int32_t *starts;
  const int64_t *ids;
  const int32_t *parents;
  const int64_t *targets;
  int64_t tokens;
  int32_t max_tree;
  int32_t *path, *counts;
  int64_t *next_ids;
  unsigned char *pages;  // null: no rows to move
  int64_t plane_bytes, page_bytes, row_bytes;
  int32_t num_pages;
  int32_t page_shift;
  const int32_t *table;
  int64_t table_stride;
  int64_t sequences;
  int64_t max_length;
  const int32_t *lengths;
  const int32_t *rows;
  int64_t vectors;  // 16-byte pieces that a position has in all planes
  int32_t row_vectors, head_vectors;  // of one row, of a position in one plane
  int32_t *error;
};

constexpr int kAcceptThreads = 256;

// Workgroup (tree, piece of the planes).  Every wave follows the path for
// itself, a node a lane: the children that fit are one ballot, and since a
// child lies behind its parent the path is an ascending set of bits and the
// walk ends.  A thread owns one 16-byte column of the rows and moves it for
// all nodes of the path, in order: the j-th goes to slot j, which lies before
// its own and before those of all later ones.
__global__ __launch_bounds__(kAcceptThreads) void tree_accept_kernel(AcceptArgs a) {
  const int64_t b = blockIdx.x;
  const int lane = threadIdx.x & (kWave - 1);
  const bool writes = blockIdx.y == 0 && threadIdx.x < kWave;
  const Tree t = tree_of(a.starts, a.rows, a.tokens, a.max_tree, b,
                         writes && lane == 0 ? a.error : nullptr);
  const int n = t.row < 0 ? 0 : t.nodes;
  int64_t id = 0, target = -1;
  int parent = -1;
  if (lane < n) {
    id = a.ids[t.first + lane];
    parent = a.parents[t.first + lane];
    target = a.targets[t.first + lane];
  }
  uint64_t on = n > 0 ? 1 : 0;
  int64_t next = -1;
  for (int cur = 0; n > 0;) {
    next = static_cast<int64_t>(lane_u64(static_cast<uint64_t>(target), cur));
    const uint64_t fits = __ballot(lane > cur && lane < n && parent == cur && id == next);
    if (next < 0 || fits == 0) break;
    cur = __ffsll(static_cast<unsigned long long>(fits)) - 1;
    on |= uint64_t{1} << cur;
  }
  const int count = __popcll(on);
  if (writes) {
    const int place = __popcll(on & ((uint64_t{1} << lane) - 1));
    if ((on >> lane) & 1) a.path[b * a.max_tree + place] = lane;
    if (lane >= count && lane < a.max_tree) a.path[b * a.max_tree + lane] = -1;
    if (lane == 0) {
      a.counts[b] = count;
      a.next_ids[b] = next;
    }
  }
  if (a.pages == nullptr || n == 0) return;
  if (t.row >= a.sequences) {
    if (writes && lane == 0) flag_range(a.error);
    return;
  }
  const int64_t len = a.lengths[t.row];
  if (len < n || len > a.max_length) {
    if (writes && lane == 0) flag_range(a.error);
    return;
  }
  const int64_t v = static_cast<int64_t>(blockIdx.y) * kAcceptThreads + threadIdx.x;
  const int64_t plane = v / a.head_vectors;
  const int in_plane = static_cast<int>(v % a.head_vectors);
  const int64_t head = in_plane / a.row_vectors;
  const int64_t page_size = int64_t{1} << a.page_shift;
  unsigned char *base = a.pages + plane * a.plane_bytes + head * page_size * a.row_bytes +
                        (in_plane % a.row_vectors) * 16;
  const int32_t *table = a.table + t.row * a.table_stride;
  int j = 0;
  for (uint64_t left = on; left != 0; left &= left - 1, ++j) {
    const int node = __ffsll(static_cast<unsigned long long>(left)) - 1;
    if (node == j) continue;
    const int64_t from = len - n + node, to = len - n + j;
    const int from_page = table[from >> a.page_shift], to_page = table[to >> a.page_shift];
    if (from_page < 0 || from_page >= a.num_pages || to_page < 0 || to_page >= a.num_pages) {
      if (writes && lane == 0) flag_range(a.error);
      continue;
    }
    if (v >= a.vectors) continue;
    *reinterpret_cast<u32x4 *>(base + to_page * a.page_bytes + (to & (page_size - 1)) * a.row_bytes) =
        *reinterpret_cast<const u32x4 *>(base + from_page * a.page_bytes +
                                         (from & (page_size - 1)) * a.row_bytes);
  }
}

static bool tree_shape_ok(int64_t trees, int64_t max_tree, int64_t n_q_heads,
                          int64_t n_kv_heads, int64_t head_dim, int64_t max_length) {
  return trees > 0 && trees <= 0xffff && max_tree > 0 && max_tree <= kTreeNodes &&
         n_kv_heads > 0 && n_q_heads > 0 && n_q_heads % n_kv_heads == 0 &&
         n_q_heads / n_kv_heads <= kPagedGroup && n_q_heads <= 0xffff &&
         (head_dim == 64 || head_dim == 128) && max_length > 0 &&
         max_length <= 0x7fffffff - 64;
}

static bool int32_ok(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }
static bool int64_ok(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 7) == 0; }

}  // namespace cascade

using namespace cascade;

extern "C" size_t cascade_paged_tree_attention_workspace_bytes(
    int64_t trees, int64_t max_tree, int64_t n_q_heads, int64_t n_kv_heads,
    int64_t head_dim, int64_t max_length) {
  if (!tree_shape_ok(trees, max_tree, n_q_heads, n_kv_heads, head_dim, max_length)) return 0;
  // Enough for fewer trees, nodes and positions too: a launch of more than
  // kTreeMaxBatch trees needs none, and more trees or positions have as many
  // runs or more.  Fewer nodes may take fewer workgroups a run, and so more runs:
  // the largest trees of each number of workgroups are looked at.
  const int64_t group = n_q_heads / n_kv_heads;
  const int64_t n = trees < kTreeMaxBatch ? trees : kTreeMaxBatch;
  size_t most = 0;
  for (int64_t nodes = max_tree; nodes > 0;) {
    const TreePlan p = tree_plan(n, nodes, n_q_heads, n_kv_heads, head_dim, max_length);
    most = p.bytes() > most ? p.bytes() : most;
    nodes = p.col_groups > 1 ? kTreeColumns * (p.col_groups - 1) / group : 0;
  }
  return most;
}

extern "C" int cascade_paged_tree_attention_bf16(
    const void *q, int64_t q_token_stride, int64_t q_head_stride, int64_t tokens,
    const int32_t *starts, const int64_t *masks, int64_t trees, int64_t max_tree,
    const void *k_pages, const void *v_pages, int64_t page_stride,
    int64_t page_head_stride, int64_t num_pages, int64_t page_size,
    const int32_t *page_table, int64_t table_stride, int64_t sequences,
    const int32_t *lengths, const int32_t *rows, int64_t max_length,
    int64_t n_q_heads, int64_t n_kv_heads, int64_t head_dim, float scale,
    void *out, int64_t out_token_stride, int64_t out_head_stride, void *workspace,
    size_t workspace_bytes, int32_t *error_flag, void *stream) {
  if (q == nullptr || starts == nullptr || masks == nullptr || k_pages == nullptr ||
      v_pages == nullptr || page_table == nullptr || lengths == nullptr || out == nullptr ||
      workspace == nullptr)
    return CASCADE_EINVAL;
  if (tokens <= 0 || tokens > 0x7fffffff || trees <= 0 || max_tree <= 0 || n_kv_heads <= 0 ||
      sequences <= 0 || num_pages <= 0 || num_pages > 0x7fffffff || max_length <= 0)
    return CASCADE_EINVAL;
  TreeArgs a{};
  if (!tree_shape_ok(trees, max_tree, n_q_heads, n_kv_heads, head_dim, max_length) ||
      !page_shift_of(page_size, &a.page_shift))
    return CASCADE_ESHAPE;
  if (table_stride < (max_length + page_size - 1) / page_size ||
      page_head_stride < page_size * head_dim ||
      page_stride < (n_kv_heads - 1) * page_head_stride + page_size * head_dim)
    return CASCADE_EINVAL;
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(out) ||
      !aligned16(workspace) || !int32_ok(starts) || !int64_ok(masks) ||
      !int32_ok(page_table) || !int32_ok(lengths) || !int32_ok(rows) ||
      !int32_ok(error_flag))
    return CASCADE_EALIGN;
  const int64_t strides[] = {q_token_stride, q_head_stride, page_stride,
                             page_head_stride, out_token_stride, out_head_stride};
  for (int64_t s : strides)
    if (!stride_ok(s)) return CASCADE_EALIGN;
  const TreePlan p = tree_plan(trees, max_tree, n_q_heads, n_kv_heads, head_dim, max_length);
  if (workspace_bytes < (p.split ? p.bytes() : kPagedAlign)) return CASCADE_EWORKSPACE;
  a.q = static_cast<const uint16_t *>(q);
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.k_pages = static_cast<const uint16_t *>(k_pages);
  a.v_pages = static_cast<const uint16_t *>(v_pages);
  a.page_stride = page_stride;
  a.head_stride = page_head_stride;
  a.num_pages = static_cast<int32_t>(num_pages);
  a.table = page_table;
  a.table_stride = table_stride;
  a.sequences = sequences;
  a.lengths = lengths;
  a.rows = rows;
  a.max_length = static_cast<int32_t>(max_length);
  a.group = static_cast<int32_t>(n_q_heads / n_kv_heads);
  a.scale_log2 = fabsf(scale) * 1.4426950408889634f;
  a.sign = scale < 0.0f ? 0x80008000u : 0u;
  // (a scale of zero would make a masked score's infinity a NaN: finite scores do
  // not show one as small as this)
  if (a.scale_log2 < 1e-37f) a.scale_log2 = 1e-37f;
  a.slack = 8.0f / a.scale_log2;
  a.out = static_cast<uint16_t *>(out);
  a.out_token = out_token_stride;
  a.out_head = out_head_stride;
  a.error = error_flag;
  a.batch = static_cast<int32_t>(trees);
  a.kv_heads = static_cast<int32_t>(n_kv_heads);
  a.starts = starts;
  a.masks = masks;
  a.tokens = tokens;
  a.max_tree = static_cast<int32_t>(max_tree);
  a.col_groups = p.col_groups;
  a.group_inverse = (65536u + a.group - 1) / a.group;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t each = n_kv_heads * p.col_groups;
  if (!p.split) {
    if (trees * each > kMaxThreads / 512) return CASCADE_ESHAPE;
    const bool wide = trees * each <= kTreeSlots;
    if (head_dim == 128)
      return wide ? launch_tree<128, false, true>(a, p.shape, trees * each, s)
                  : launch_tree<128, false, false>(a, p.shape, trees * each, s);
    return wide ? launch_tree<64, false, true>(a, p.shape, trees * each, s)
                : launch_tree<64, false, false>(a, p.shape, trees * each, s);
  }
  if (p.runs * each > kMaxThreads / 512 ||
      trees * max_tree > kMaxThreads / kTreeMergeThreads / n_q_heads)
    return CASCADE_ESHAPE;
  unsigned char *ws = static_cast<unsigned char *>(workspace);
  a.runs = static_cast<int32_t>(p.runs);
  a.per_round = 1.0 / static_cast<double>(p.round);
  a.per_two = 1.0 / static_cast<double>(p.two);
  a.plan = reinterpret_cast<int32_t *>(ws);
  a.part_ml = reinterpret_cast<float *>(ws + p.plan_bytes);
  a.part_acc = reinterpret_cast<float *>(ws + p.plan_bytes + p.ml_bytes);
  const int64_t runs_a_tree = p.runs / trees;
  if (head_dim == 128) {
    const hipError_t e = launch_tree<128, true, false>(a, p.shape, p.runs * each, s);
    return e != hipSuccess ? e : launch_tree_merge<128>(a, runs_a_tree, s);
  }
  const hipError_t e = launch_tree<64, true, false>(a, p.shape, p.runs * each, s);
  return e != hipSuccess ? e : launch_tree_merge<64>(a, runs_a_tree, s);
}

extern "C" int cascade_paged_tree_accept(
    const int32_t *starts, const int64_t *ids, const int32_t *parents,
    const int64_t *targets, int64_t tokens, int64_t trees, int64_t max_tree,
    int32_t *path, int32_t *counts, int64_t *next_ids, void *pages,
    int64_t planes, int64_t plane_bytes, int64_t num_pages, int64_t n_kv_heads,
    int64_t page_size, int64_t row_bytes, const int32_t *page_table,
    int64_t table_stride, int64_t sequences, int64_t max_pages,
    const int32_t *lengths, const int32_t *rows, int32_t *error_flag,
    void *stream) {
  if (starts == nullptr || ids == nullptr || parents == nullptr || targets == nullptr ||
      path == nullptr || counts == nullptr || next_ids == nullptr)
    return CASCADE_EINVAL;
  if (tokens <= 0 || tokens > 0x7fffffff || trees <= 0 || max_tree <= 0)
    return CASCADE_EINVAL;
  if (max_tree > kTreeNodes || trees > kMaxThreads / kAcceptThreads) return CASCADE_ESHAPE;
  if (!int32_ok(starts) || !int64_ok(ids) || !int32_ok(parents) || !int64_ok(targets) ||
      !int32_ok(path) || !int32_ok(counts) || !int64_ok(next_ids) || !int32_ok(rows) ||
      !int32_ok(error_flag))
    return CASCADE_EALIGN;
  AcceptArgs a{};
  a.starts = starts;
  a.ids = ids;
  a.parents = parents;
  a.targets = targets;
  a.tokens = tokens;
  a.max_tree = static_cast<int32_t>(max_tree);
  a.path = path;
  a.counts = counts;
  a.next_ids = next_ids;
  a.rows = rows;
  a.error = error_flag;
  int64_t pieces = 1;
  if (pages != nullptr) {
    if (page_table == nullptr || lengths == nullptr || planes <= 0 || num_pages <= 0 ||
        num_pages > 0x7fffffff || n_kv_heads <= 0 || row_bytes <= 0 || sequences <= 0 ||
        max_pages <= 0 || table_stride < max_pages || plane_bytes < 0)
      return CASCADE_EINVAL;
    if (n_kv_heads > 1024 || row_bytes > 2048 || planes > 0xffff ||
        !page_shift_of(page_size, &a.page_shift) || max_pages > 0x7fffffff / page_size)
      return CASCADE_ESHAPE;
    if (!aligned16(pages) || (plane_bytes & 15) || (row_bytes & 15) || !int32_ok(page_table) ||
        !int32_ok(lengths))
      return CASCADE_EALIGN;
    a.page_bytes = n_kv_heads * page_size * row_bytes;
    if (planes > 1 && plane_bytes / num_pages < a.page_bytes) return CASCADE_EINVAL;
    a.pages = static_cast<unsigned char *>(pages);
    a.plane_bytes = plane_bytes;
    a.row_bytes = row_bytes;
    a.num_pages = static_cast<int32_t>(num_pages);
    a.table = page_table;
    a.table_stride = table_stride;
    a.sequences = sequences;
    a.max_length = max_pages * page_size;
    a.lengths = lengths;
    a.row_vectors = static_cast<int32_t>(row_bytes / 16);
    a.head_vectors = static_cast<int32_t>(n_kv_heads) * a.row_vectors;
    a.vectors = planes * a.head_vectors;
    pieces = (a.vectors + kAcceptThreads - 1) / kAcceptThreads;
    if (pieces > 0xffff) return CASCADE_ESHAPE;
  }
  const dim3 grid(static_cast<unsigned>(trees), static_cast<unsigned>(pieces));
  return launch_kernel(tree_accept_kernel, grid, dim3(kAcceptThreads), 0,
                       static_cast<hipStream_t>(stream), a);
}
