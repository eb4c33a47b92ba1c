// The operators of a KV cache kept in pages (gfx950): rotary positions with
// the write of K and V rows into pages, attention of one new token a
// sequence over its pages, and copies of pages.
//
// A page holds page_size consecutive positions of a sequence for every KV
// head, head-major: rows of one head are contiguous, so that a wave's loads
// cover whole runs of page_size x head_dim x 2 bytes.  Page p of a layer's K
// (or V) pool starts p * page_stride elements behind the pool's start, head
// g of it g * head_stride further.  A page table row lists the pages of one
// sequence in order.  page_size is a power of two of at least 8: the eight
// consecutive rows that a lane group handles then share a page, and a page
// lookup is a shift.
//
// Device-held indices (rows, positions, lengths, page numbers) are checked
// in the kernels before they form an address: what they reject is left out
// and CASCADE_PAGED_ERANGE is or-ed into the caller's error word.
#include "paged_device.h"

namespace cascade {

// ---------------------------------------------------------------- append
struct AppendArgs {
  const uint16_t *q, *k, *v;  // token t, head h at t * token + h * head
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;
  const int32_t *positions;
  const int32_t *turns;  // nullable: the rope tables' row, where not the position
  const int32_t *rows;   // nullable: token t belongs to table row t
  const int32_t *table;
  int64_t table_stride;
  int64_t sequences;
  int32_t max_pages;
  const uint16_t *cos, *sin;  // [rope_positions, rope_dim / 2], nullable
  int64_t rope_positions;
  int32_t rope_dim;
  int32_t interleaved;
  uint16_t *q_out;
  int64_t qo_token, qo_head;
  uint16_t *k_pages, *v_pages;
  int64_t page_stride, head_stride;
  int32_t num_pages;
  int32_t page_shift;
  int32_t q_heads, kv_heads, dim;
  int32_t *error;
};

constexpr int kAppendThreads = 512;  // at most

// One workgroup a token.  A thread's unit is 16 dims of one head as two
// 16-byte vectors: for rotated dims the two vectors whose elements form
// pairs (half layout: 8 dims and the 8 dims rope_dim / 2 behind them;
// interleaved: 16 neighbouring dims), so that both read one vector of cos
// and one of sin; other dims are copied.  Products and sums in fp32 and one
// rounding.  Bound by HBM for prompts: 8002 tokens of 48 heads of 128 take
// 34.5 us (5.7 TB/s read and written); one token 2.7 us, three trips to
// memory one behind the other (position, page, and the write), 61 tokens 3.7.
__global__ __launch_bounds__(kAppendThreads) void paged_append_kernel(AppendArgs a) {
  const int64_t t = blockIdx.x;
  const int64_t pos = a.positions[t];
  const int64_t row = a.rows != nullptr ? a.rows[t] : t;
  if (pos < 0 || row < 0) return;  // a padding token
  const int64_t turn_row = a.turns != nullptr ? a.turns[t] : pos;
  const int64_t slot_page = pos >> a.page_shift;
  bool ok = row < a.sequences && slot_page < a.max_pages &&
            (a.rope_dim == 0 || (turn_row >= 0 && turn_row < a.rope_positions));
  const int64_t page = ok ? a.table[row * a.table_stride + slot_page] : -1;
  ok = page >= 0 && page < a.num_pages;
  if (!ok) {
    if (threadIdx.x == 0) flag_range(a.error);
    return;
  }
  const int64_t slot = pos & ((int64_t{1} << a.page_shift) - 1);
  const int64_t base = page * a.page_stride + slot * a.dim;
  const int per_head = a.dim / 16;
  const int rotated = a.rope_dim / 16;
  const int half = a.rope_dim / 2;
  const int units = (a.q_heads + 2 * a.kv_heads) * per_head;
  for (int u = threadIdx.x; u < units; u += static_cast<int>(blockDim.x)) {
    int head = u / per_head;
    const int part = u % per_head;
    const uint16_t *src;
    uint16_t *dst;
    bool turn = part < rotated;
    if (head < a.q_heads) {
      src = a.q + t * a.q_token + head * a.q_head;
      dst = a.q_out + t * a.qo_token + head * a.qo_head;
    } else if ((head -= a.q_heads) < a.kv_heads) {
      src = a.k + t * a.k_token + head * a.k_head;
      dst = a.k_pages + base + head * a.head_stride;
    } else {
      head -= a.kv_heads;
      src = a.v + t * a.v_token + head * a.v_head;
      dst = a.v_pages + base + head * a.head_stride;
      turn = false;
    }
    const bool split = turn && !a.interleaved;
    const int d0 = split ? 8 * part : 16 * part;
    const int d1 = split ? half + 8 * part : 16 * part + 8;
    u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(src + d0));
    u32x4 y = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(src + d1));
    if (turn) {
      const u32x4 c = *reinterpret_cast<const u32x4 *>(a.cos + turn_row * half + 8 * part);
      const u32x4 s = *reinterpret_cast<const u32x4 *>(a.sin + turn_row * half + 8 * part);
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t xi = x[i], yi = y[i], ci = c[i >> 1], si = s[i >> 1];
          const uint32_t cj = c[2 + (i >> 1)], sj = s[2 + (i >> 1)];
          const float cx = i & 1 ? hi_bf16(ci) : lo_bf16(ci);
          const float sx = i & 1 ? hi_bf16(si) : lo_bf16(si);
          const float cy = i & 1 ? hi_bf16(cj) : lo_bf16(cj);
          const float sy = i & 1 ? hi_bf16(sj) : lo_bf16(sj);
          x[i] = pack_bf16x2(lo_bf16(xi) * cx - hi_bf16(xi) * sx,
                             hi_bf16(xi) * cx + lo_bf16(xi) * sx);
          y[i] = pack_bf16x2(lo_bf16(yi) * cy - hi_bf16(yi) * sy,
                             hi_bf16(yi) * cy + lo_bf16(yi) * sy);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t xi = x[i], yi = y[i], ci = c[i], si = s[i];
          x[i] = pack_bf16x2(lo_bf16(xi) * lo_bf16(ci) - lo_bf16(yi) * lo_bf16(si),
                             hi_bf16(xi) * hi_bf16(ci) - hi_bf16(yi) * hi_bf16(si));
          y[i] = pack_bf16x2(lo_bf16(yi) * lo_bf16(ci) + lo_bf16(xi) * lo_bf16(si),
                             hi_bf16(yi) * hi_bf16(ci) + hi_bf16(xi) * hi_bf16(si));
        }
      }
    }
    *reinterpret_cast<u32x4 *>(dst + d0) = x;
    *reinterpret_cast<u32x4 *>(dst + d1) = y;
  }
}

// ------------------------------------------------------------- attention
constexpr int kWholeWaves = 8;   // of one that takes a whole row
constexpr int kPagedMaxBatch = 1024;  // of a split launch
// Workgroups that the device holds at a time (256 CUs with four and with six).
constexpr int64_t kPagedSlots128 = 1024, kPagedSlots64 = 1536;

// Two weights as sums of two bf16 values each, for the product with V: one
// value alone, 2^-8 off, shows next to the rounding of the result where V's
// rows cancel.  The upper parts are cut off just below the weights (a factor
// of 1 - 2^-24 leaves no normal fp32 number as it is), so that the lower ones,
// which fp32 holds exactly, are positive: a zero or a negative one would turn
// an infinite value of V into a NaN.  Of a weight in [2^e, 2^(e+1)) the lower
// part is at most 2^(e-7), and its rounding, half a step, 2^(e-16).  The second
// product hides behind the loads (64 ragged sequences of up to 16384 positions
// 318 us, 317 with one; 32769 positions 28.8 and 28.6).
struct SplitWeights {
  uint32_t upper, lower;
};

__device__ __forceinline__ SplitWeights split_weights(float a, float b) {
  constexpr float kBelow = 1.0f - 0x1p-24f;
  const uint32_t upper = __builtin_amdgcn_perm(__float_as_uint(b * kBelow),
                                               __float_as_uint(a * kBelow), 0x07060302u);
  return {upper, pack_bf16x2(a - lo_bf16(upper), b - hi_bf16(upper))};
}

__device__ __forceinline__ PagedRow paged_row(const PagedAttnArgs &a, int b, bool flag) {
  PagedRow r{-1, 0};
  if (b >= a.batch) return r;
  r.row = a.rows != nullptr ? a.rows[b] : b;
  if (r.row >= a.sequences) {
    if (flag) flag_range(a.error);
    r.row = -1;
  }
  if (r.row < 0) return r;
  r.len = a.lengths[r.row];
  if (r.len < 0 || r.len > a.max_length) {
    if (flag) flag_range(a.error);
    r.len = min(max(r.len, 0), a.max_length);
  }
  return r;
}

// Workgroup (run, KV head), or (batch row, KV head) without SPLIT; each wave
// runs an online softmax over every WAVES-th block of 32 positions and the
// waves merge in LDS.  The products are v_mfma_f32_16x16x32_bf16 with the
// query heads of the KV head as columns (zeros past group):
//   S = K_blk q^T    two 16-row tiles x D / 32 chunks
//   O += V_blk^T P   D / 16 tiles, K = the 32 positions, for either part of P
// Lane (c, g4) = (l % 16, l / 16) owns the scores of head c at rows
// 8 g4 .. 8 g4 + 7 (the row order inside a K tile is chosen for that), which
// is its piece of the P operand.  K rows are transposed through LDS, V rows
// (16 lanes a row, dims DV c .. DV c + DV - 1 with DV = D / 16) in registers.
// Scores carry scale * log2(e).  The running maximum starts at -FLT_MAX, so
// a block whose rows are all left out keeps it and adds nothing; a sequence
// with no row at all ends with a zero sum and writes zeros.
// Bound by HBM: 64 ragged sequences of up to 16384 positions (8 KV heads of
// 128) 316 us at 6.2 TB/s, where a plain read of those bytes takes 285; one of
// 32769 positions 25.1 us (21.1), the lookups before the first rows and the
// join behind the last ones showing.  Four waves on a SIMD (at most 128
// registers, hence the q operands in LDS) hide the loads better than a second
// register set of rows with two waves does (351 against 347 us for the first,
// 32.2 against 33.5 for the second, when both were built).
template <int D, bool SPLIT>
__global__ __launch_bounds__((SPLIT ? kPagedWaves : kWholeWaves) * kWave, 4) void
paged_attention_kernel(PagedAttnArgs a) {
  constexpr int WAVES = SPLIT ? kPagedWaves : kWholeWaves;
  constexpr int DV = D / 16;  // dims a lane holds of a V row
  constexpr int KC = D / 32;  // 32-dim chunks
  constexpr int CH = D / 8;   // 16-byte chunks of a row
  __shared__ float s_ml[WAVES][kPagedGroup][2];
  // a wave's K block, and in the end its output (both 64 D bytes)
  __shared__ union {
    u32x4 k[kPagedBlock * CH];
    float acc[kPagedGroup][D];
  } s_wave[WAVES];
  __shared__ u32x4 s_q[KC][kWave];
  static_assert(KC <= WAVES, "a chunk of q a wave");
  const int g = static_cast<int>(blockIdx.x) % a.kv_heads;
  const int run = static_cast<int>(blockIdx.x) / a.kv_heads;
  const int G = a.group;
  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int wave = tid / kWave;
  const int c16 = lane & 15;
  const int g4 = lane >> 4;
  int b, len, first, end, count = 1;
  int64_t row;
  if constexpr (SPLIT) {
    const PagedRun r = find_run(a, run, lane, blockIdx.x == 0 && wave == 0,
                                [&](int i, bool flag) { return paged_row(a, i, flag); });
    if (r.b < 0) return;
    b = r.b;
    row = r.row;
    len = r.len;
    first = r.first;
    end = r.end;
    count = r.count;
  } else {
    b = run;
    const PagedRow r = paged_row(a, b, g == 0 && tid == 0);
    if (r.row < 0) return;
    row = r.row;
    len = r.len;
    first = 0;
    end = (len + kPagedBlock - 1) / kPagedBlock;
  }
  const int last = len - 1;
  const int32_t *table = a.table + row * a.table_stride;
  const uint16_t *kb = a.k_pages + g * a.head_stride;
  const uint16_t *vb = a.v_pages + g * a.head_stride;
  const int page_mask = (1 << a.page_shift) - 1;

  // the q operands, a chunk a wave, kept in LDS: 16 registers less are what
  // lets four waves share a SIMD
  if (wave < KC)
    s_q[wave][lane] = c16 < G ? *reinterpret_cast<const u32x4 *>(
                                    a.q + b * a.q_token + (g * G + c16) * a.q_head +
                                    32 * wave + 8 * g4)
                              : u32x4{0u, 0u, 0u, 0u};
  __syncthreads();
  const uint32_t head_mask = c16 < G ? 0xffffffffu : 0u;

  float m = -FLT_MAX, l = 0.0f;
  f32x4 o[DV];
#pragma unroll
  for (int e = 0; e < DV; ++e) o[e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  // Rows come in whole, 16 lanes a row (8 for K rows of 64 dims), so that a
  // load covers runs of 128 bytes or more.  A lane's V rows are group g4 of
  // eight of a block, which lies in one page; groups past the end take the
  // last row's page: its rows are memory of the pool whatever they hold.
  auto page_of = [&](int blk) {
    return table[min(blk * kPagedBlock + 8 * g4, last) >> a.page_shift];
  };
  // One block's rows in registers: V of rows 8 g4 + j, dims DV c16 ..; K as
  // laid out by k_slot.
  struct Rows {
    u32x4 k[D / 16];
    uint32_t v[8][DV / 2];
    bool bad;  // the group's page is none of the pool's
  };
  // K rows go through LDS to become MFMA operands.  Row r keeps its chunk ch at
  // slot CH r + (ch ^ key(r)), where the keys of the 16 rows of an operand
  // (of the eight of one parity, for 64 dims: two rows share the banks)
  // differ: neither the writes nor the reads meet in a bank.
  auto k_slot = [](int r, int ch) {
    const int key = D == 128 ? 4 * (r >> 3) + (r & 3) : 2 * (r >> 3) + ((r >> 1) & 1);
    return CH * r + (ch ^ key);
  };
  auto load = [&](int blk, int page, Rows &x) __attribute__((always_inline)) {
    x.bad = page < 0 || page >= a.num_pages;
    if (x.bad) {
      page = 0;
      flag_range(a.error);
    }
    const int64_t at = page * a.page_stride + ((blk * kPagedBlock + 8 * g4) & page_mask) * D;
    if constexpr (D == 128) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        x.k[j] = __builtin_nontemporal_load(
            reinterpret_cast<const u32x4 *>(kb + at + j * D + 8 * c16));
    } else {
      // group i of eight rows, eight lanes a row
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(at), 16 * i);
        const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(at >> 32), 16 * i);
        const int64_t group = static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
        x.k[i] = __builtin_nontemporal_load(
            reinterpret_cast<const u32x4 *>(kb + group + 8 * lane));
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint16_t *vp = vb + at + j * D + DV * c16;
      if constexpr (DV == 8) {
        const u32x4 w = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(vp));
#pragma unroll
        for (int i = 0; i < 4; ++i) x.v[j][i] = w[i];
      } else {
        const u32x2 w = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(vp));
        x.v[j][0] = w[0];
        x.v[j][1] = w[1];
      }
    }
  };
  auto step = [&](int blk, Rows &x) __attribute__((always_inline)) {
    const int r0 = blk * kPagedBlock;
    u32x4 *sk = s_wave[wave].k;
    // the slots are worked out again in each step, and s_q is read again:
    // kept in registers they would cost the fourth wave of a SIMD
    int ln = lane;
    asm volatile("" : "+v"(ln)::"memory");
    const int lc = ln & 15, lg = ln >> 4;
    if constexpr (D == 128) {
#pragma unroll
      for (int j = 0; j < 8; ++j) sk[k_slot(8 * lg + j, lc)] = x.k[j];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) sk[k_slot(8 * i + (ln >> 3), ln & 7)] = x.k[i];
    }
    asm volatile("" ::: "memory");
    // K tile row i is block row 8 (i / 4) + i % 4 + 4 hf
    const int krow = 8 * (lc >> 2) + (lc & 3);
    f32x4 s0 = {0.0f, 0.0f, 0.0f, 0.0f}, s1 = s0;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const u32x4 qop = s_q[c][ln];
      s0 = mfma_16x16x32_bf16(sk[k_slot(krow, 4 * c + lg)], qop, s0);
      s1 = mfma_16x16x32_bf16(sk[k_slot(krow + 4, 4 * c + lg)], qop, s1);
    }
    float s[8] = {s0[0], s0[1], s0[2], s0[3], s1[0], s1[1], s1[2], s1[3]};
    float bmax = -INFINITY;
    const bool cut = r0 + kPagedBlock > len || __any(x.bad);  // uniform
    if (cut) {
      // rows past the end, or of a page outside the pool, take no part
      // whatever they hold: 0 times a NaN of theirs would be one
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool out = x.bad || r0 + 8 * g4 + j >= len;
        s[j] = out ? -INFINITY : s[j] * a.scale_log2;
#pragma unroll
        for (int i = 0; i < DV / 2; ++i) x.v[j][i] = out ? 0u : x.v[j][i];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] *= a.scale_log2;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) bmax = fmaxf(bmax, s[j]);
    bmax = xor32_max(xor16_max(bmax));
    const float mnew = fmaxf(m, bmax);
    const float alpha = paged_exp2(m - mnew);
    m = mnew;
    float p[8], psum = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      p[j] = paged_exp2(s[j] - mnew);
      psum += p[j];
    }
    l = fmaf(l, alpha, psum);
    u32x4 pop, rest;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const SplitWeights w = split_weights(p[2 * i], p[2 * i + 1]);
      pop[i] = w.upper & head_mask;
      rest[i] = w.lower & head_mask;
    }
    if (alpha != 1.0f) {
#pragma unroll
      for (int e = 0; e < DV; ++e) o[e] *= alpha;
    }
#pragma unroll
    for (int e = 0; e < DV; ++e) {
      const uint32_t sel = (e & 1) ? 0x07060302u : 0x05040100u;
      u32x4 vop;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        vop[i] = __builtin_amdgcn_perm(x.v[2 * i + 1][e >> 1], x.v[2 * i][e >> 1], sel);
      o[e] = mfma_16x16x32_bf16(vop, rest, o[e]);
      o[e] = mfma_16x16x32_bf16(vop, pop, o[e]);
    }
  };
  int page = first + wave < end ? page_of(first + wave) : 0;
  for (int blk = first + wave; blk < end; blk += WAVES) {
    Rows x;
    load(blk, page, x);
    // the next block's pages, while this one's rows are on their way
    if (blk + WAVES < end) page = page_of(blk + WAVES);
    step(blk, x);
  }

  l = xor32_sum(xor16_sum(l));
  if (c16 < G) {
    // o[e][r] = O[dim DV (4 g4 + r) + e][head c16]
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int e = 0; e < DV; ++e) s_wave[wave].acc[c16][DV * (4 * g4 + r) + e] = o[e][r];
    if (g4 == 0) {
      s_ml[wave][c16][0] = m;
      s_ml[wave][c16][1] = l;
    }
  }
  __syncthreads();
  for (int i = tid; i < G * D; i += WAVES * kWave) {
    const int h = i / D;
    const int d = i % D;
    float mm = -FLT_MAX;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) mm = fmaxf(mm, s_ml[w][h][0]);
    float den = 0.0f, r = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float wt = paged_exp2(s_ml[w][h][0] - mm);
      den = fmaf(wt, s_ml[w][h][1], den);
      r = fmaf(wt, s_wave[w].acc[h][d], r);
    }
    if (!SPLIT || count == 1) {
      a.out[b * a.out_token + (g * G + h) * a.out_head + d] =
          f32_to_bf16(den == 0.0f ? 0.0f : r / den);
    } else {
      const int64_t slot = static_cast<int64_t>(run) * (a.kv_heads * G) + g * G + h;
      a.part_acc[slot * D + d] = r;
      if (d == 0) {
        a.part_ml[2 * slot] = mm;
        a.part_ml[2 * slot + 1] = den;
      }
    }
  }
}

// Joins the runs of one (batch row, query head):
//   out = sum_r 2^(m_r - M) acc_r / sum_r 2^(m_r - M) l_r,  M = max_r m_r.
// A slice of D / 4 threads (four dims each) takes every kSlices-th run with a
// running maximum of its own, so that no load waits for another, and the
// slices join in LDS in a fixed order.  Rows of one run were written already.
// Bound by latency, the plan and then the partials: 4.5 us for the 86 runs of
// one row of 32 heads, 4.6 for 64 rows.
constexpr int kPagedMergeThreads = 256;

template <int D>
__global__ __launch_bounds__(kPagedMergeThreads) void paged_merge_kernel(PagedAttnArgs a) {
  constexpr int kSlices = kPagedMergeThreads * 4 / D;
  __shared__ f32x4 s_acc[kSlices][D / 4];
  __shared__ float s_ml[kSlices][2];
  const int heads = a.kv_heads * a.group;
  const int b = static_cast<int>(blockIdx.x) / heads;
  const int h = static_cast<int>(blockIdx.x) % heads;
  const int slice = threadIdx.x / (D / 4);
  const int d = threadIdx.x % (D / 4);
  const int index = a.plan[2 * b], count = a.plan[2 * b + 1];
  // a padding row, or written already (or, past the workspace, a plan that
  // another call has overwritten)
  if (count <= 1 || index < 0 || count > a.runs - index) return;
  const int64_t base = static_cast<int64_t>(index) * heads + h;
  float m = -FLT_MAX, den = 0.0f;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int r = slice; r < count; r += kSlices) {
    const int64_t slot = base + static_cast<int64_t>(r) * heads;
    const float2 ml = *reinterpret_cast<const float2 *>(a.part_ml + 2 * slot);
    const f32x4 v = *reinterpret_cast<const f32x4 *>(a.part_acc + slot * D + 4 * d);
    const float mnew = fmaxf(m, ml.x);
    const float keep = paged_exp2(m - mnew), w = paged_exp2(ml.x - mnew);
    m = mnew;
    den = fmaf(w, ml.y, den * keep);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = fmaf(w, v[i], acc[i] * keep);
  }
  s_acc[slice][d] = acc;
  if (d == 0) {
    s_ml[slice][0] = m;
    s_ml[slice][1] = den;
  }
  __syncthreads();
  if (threadIdx.x >= D) return;
  const int dim = threadIdx.x;
  float mm = -FLT_MAX;
#pragma unroll
  for (int k = 0; k < kSlices; ++k) mm = fmaxf(mm, s_ml[k][0]);
  float sum = 0.0f, r = 0.0f;
#pragma unroll
  for (int k = 0; k < kSlices; ++k) {
    const float w = paged_exp2(s_ml[k][0] - mm);
    sum = fmaf(w, s_ml[k][1], sum);
    r = fmaf(w, s_acc[k][dim / 4][dim % 4], r);
  }
  a.out[b * a.out_token + h * a.out_head + dim] = f32_to_bf16(sum == 0.0f ? 0.0f : r / sum);
}

// Whether a launch splits, and its sizes.  Rows of at most kWholeBlocks blocks
// take one workgroup of eight waves each, which costs less than a second
// launch (512 positions, 8 KV heads: 1 row 6.8 us against 7.6 split, 64 rows
// 16.4 against 20.3; at 1000 positions 12.5 against 7.7 and 28.9 against
// 30.1).  Past kPagedMaxBatch rows every wave's walk over the lengths would
// cost more than the balance is worth, and the rows fill the device.
struct PagedPlan {
  bool split;
  int64_t round, two;  // runs wanted, in one round and in two
  int64_t runs;        // at most
  size_t plan_bytes, ml_bytes, acc_bytes;
};

static PagedPlan paged_plan(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim,
                            int64_t max_length) {
  PagedPlan p{};
  const int64_t blocks = (max_length + kPagedBlock - 1) / kPagedBlock;
  p.split = blocks > kWholeBlocks && batch <= kPagedMaxBatch;
  if (!p.split) return p;
  const int64_t slots =
      ((dim == 128 ? kPagedSlots128 : kPagedSlots64) + kv_heads - 1) / kv_heads;
  // (half a run a row is lost to the last runs)
  auto wanted = [batch](int64_t runs) {
    return runs - batch / 2 > runs / 2 ? runs - batch / 2 : (runs + 1) / 2;
  };
  p.two = wanted(2 * slots);
  p.round = wanted(slots);
  if (3 * batch > p.round) p.round = p.two;
  p.runs = p.two + batch;
  const int64_t most = batch * ((blocks + kPagedMinRun - 1) / kPagedMinRun);
  if (p.runs > most) p.runs = most;
  auto rounded = [](int64_t bytes) {
    return (static_cast<size_t>(bytes) + kPagedAlign - 1) / kPagedAlign * kPagedAlign;
  };
  p.plan_bytes = rounded(batch * 8);
  p.ml_bytes = rounded(p.runs * q_heads * 8);
  p.acc_bytes = rounded(p.runs * q_heads * dim * 4);
  return p;
}

// ----------------------------------------------------------------- copies
struct CopyPagesArgs {
  unsigned char *base;  // page p of plane i at i * plane_bytes + p * page_bytes
  int64_t plane_bytes;
  int64_t page_bytes;
  int32_t num_pages;
  int32_t planes;
  const int32_t *pairs;  // [count][2]: source, destination
  int64_t pieces;        // pieces a page
  int64_t total;         // count * planes * pieces
  int32_t *error;
};

constexpr int kCopyThreads = 256;
constexpr int64_t kCopyPiece = int64_t{kCopyThreads} * 16;  // a 16-byte vector a thread

// One workgroup copies a piece of 4 KiB of one page of one plane.  Bound by
// HBM: 257 pages of 128 KiB in 8 planes take 92 us (5.8 TB/s read and
// written; a 1 GiB device copy reaches 5.1), 99 in pieces of 8 KiB, 109 of 16 KiB with
// neither side's nontemporal hint.
__global__ __launch_bounds__(kCopyThreads) void copy_pages_kernel(CopyPagesArgs a) {
  for (int64_t w = blockIdx.x; w < a.total; w += gridDim.x) {
    const int64_t piece = w % a.pieces;
    const int64_t rest = w / a.pieces;
    const int64_t plane = rest % a.planes;
    const int64_t pair = rest / a.planes;
    const int32_t src = a.pairs[2 * pair];
    const int32_t dst = a.pairs[2 * pair + 1];
    if (src < 0 || dst < 0) continue;  // a padding pair
    if (src >= a.num_pages || dst >= a.num_pages) {
      if (threadIdx.x == 0) flag_range(a.error);
      continue;
    }
    unsigned char *plane_base = a.base + plane * a.plane_bytes;
    const unsigned char *from = plane_base + src * a.page_bytes;
    unsigned char *to = plane_base + dst * a.page_bytes;
    const int64_t at = piece * kCopyPiece + threadIdx.x * 16;
    if (at < a.page_bytes)
      __builtin_nontemporal_store(
          __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(from + at)),
          reinterpret_cast<u32x4 *>(to + at));
  }
}

}  // namespace cascade

using namespace cascade;

extern "C" int cascade_paged_append_turned_bf16(
    const void *q, int64_t q_token_stride, int64_t q_head_stride, const void *k,
    int64_t k_token_stride, int64_t k_head_stride, const void *v,
    int64_t v_token_stride, int64_t v_head_stride, int64_t tokens,
    int64_t n_q_heads, int64_t n_kv_heads, int64_t head_dim,
    const int32_t *positions, const int32_t *turns, const int32_t *rows,
    const int32_t *page_table,
    int64_t table_stride, int64_t sequences, int64_t max_pages,
    const void *rope_cos, const void *rope_sin, int64_t rope_positions,
    int64_t rope_dim, int interleaved, void *q_out, int64_t q_out_token_stride,
    int64_t q_out_head_stride, void *k_pages, void *v_pages, int64_t page_stride,
    int64_t page_head_stride, int64_t num_pages, int64_t page_size,
    int32_t *error_flag, void *stream) {
  if (k == nullptr || v == nullptr || positions == nullptr || page_table == nullptr ||
      k_pages == nullptr || v_pages == nullptr)
    return CASCADE_EINVAL;
  if (n_q_heads < 0 || (n_q_heads > 0 && (q == nullptr || q_out == nullptr)))
    return CASCADE_EINVAL;
  if (tokens <= 0 || tokens > 0x7fffffff || n_kv_heads <= 0 || sequences <= 0 ||
      max_pages <= 0 || table_stride < max_pages || num_pages <= 0 ||
      num_pages > 0x7fffffff)
    return CASCADE_EINVAL;
  AppendArgs a{};
  if (head_dim < 16 || head_dim > 1024 || (head_dim & 15) || n_q_heads > 1024 ||
      n_kv_heads > 1024 || !page_shift_of(page_size, &a.page_shift) ||
      max_pages > 0x7fffffff / page_size)
    return CASCADE_ESHAPE;
  const int64_t units = (n_q_heads + 2 * n_kv_heads) * (head_dim / 16);
  int64_t threads = (units + kWave - 1) / kWave * kWave;
  if (threads > kAppendThreads) threads = kAppendThreads;
  if (tokens > kMaxThreads / threads) return CASCADE_ESHAPE;
  if (rope_dim < 0 || rope_dim > head_dim || (rope_dim & 15)) return CASCADE_ESHAPE;
  if (rope_dim > 0 &&
      (rope_cos == nullptr || rope_sin == nullptr || rope_positions <= 0))
    return CASCADE_EINVAL;
  if (page_head_stride < page_size * head_dim ||
      page_stride < (n_kv_heads - 1) * page_head_stride + page_size * head_dim)
    return CASCADE_EINVAL;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(rope_cos) ||
      !aligned16(rope_sin) || !aligned16(q_out) || !aligned16(k_pages) ||
      !aligned16(v_pages) || (reinterpret_cast<uintptr_t>(positions) & 3) ||
      (reinterpret_cast<uintptr_t>(turns) & 3) ||
      (reinterpret_cast<uintptr_t>(rows) & 3) ||
      (reinterpret_cast<uintptr_t>(page_table) & 3) ||
      (reinterpret_cast<uintptr_t>(error_flag) & 3))
    return CASCADE_EALIGN;
  const int64_t strides[] = {q_token_stride, q_head_stride, k_token_stride,
                             k_head_stride,  v_token_stride, v_head_stride,
                             q_out_token_stride, q_out_head_stride, page_stride,
                             page_head_stride};
  for (int64_t s : strides)
    if (!stride_ok(s)) return CASCADE_EALIGN;
  a.q = static_cast<const uint16_t *>(q);
  a.k = static_cast<const uint16_t *>(k);
  a.v = static_cast<const uint16_t *>(v);
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.k_token = k_token_stride;
  a.k_head = k_head_stride;
  a.v_token = v_token_stride;
  a.v_head = v_head_stride;
  a.positions = positions;
  a.turns = turns;
  a.rows = rows;
  a.table = page_table;
  a.table_stride = table_stride;
  a.sequences = sequences;
  a.max_pages = static_cast<int32_t>(max_pages);
  a.cos = static_cast<const uint16_t *>(rope_cos);
  a.sin = static_cast<const uint16_t *>(rope_sin);
  a.rope_positions = rope_positions;
  a.rope_dim = static_cast<int32_t>(rope_dim);
  a.interleaved = interleaved;
  a.q_out = static_cast<uint16_t *>(q_out);
  a.qo_token = q_out_token_stride;
  a.qo_head = q_out_head_stride;
  a.k_pages = static_cast<uint16_t *>(k_pages);
  a.v_pages = static_cast<uint16_t *>(v_pages);
  a.page_stride = page_stride;
  a.head_stride = page_head_stride;
  a.num_pages = static_cast<int32_t>(num_pages);
  a.q_heads = static_cast<int32_t>(n_q_heads);
  a.kv_heads = static_cast<int32_t>(n_kv_heads);
  a.dim = static_cast<int32_t>(head_dim);
  a.error = error_flag;
  return launch_kernel(paged_append_kernel, dim3(static_cast<unsigned>(tokens)),
                       dim3(static_cast<unsigned>(threads)),
                       0, static_cast<hipStream_t>(stream), a);
}

extern "C" int cascade_paged_append_bf16(
    const void *q, int64_t q_token_stride, int64_t q_head_stride, const void *k,
    int64_t k_token_stride, int64_t k_head_stride, const void *v,
    int64_t v_token_stride, int64_t v_head_stride, int64_t tokens,
    int64_t n_q_heads, int64_t n_kv_heads, int64_t head_dim,
    const int32_t *positions, const int32_t *rows, const int32_t *page_table,
    int64_t table_stride, int64_t sequences, int64_t max_pages,
    const void *rope_cos, const void *rope_sin, int64_t rope_positions,
    int64_t rope_dim, int interleaved, void *q_out, int64_t q_out_token_stride,
    int64_t q_out_head_stride, void *k_pages, void *v_pages, int64_t page_stride,
    int64_t page_head_stride, int64_t num_pages, int64_t page_size,
    int32_t *error_flag, void *stream) {
  return cascade_paged_append_turned_bf16(
      q, q_token_stride, q_head_stride, k, k_token_stride, k_head_stride, v,
      v_token_stride, v_head_stride, tokens, n_q_heads, n_kv_heads, head_dim, positions,
      nullptr, rows, page_table, table_stride, sequences, max_pages, rope_cos, rope_sin,
      rope_positions, rope_dim, interleaved, q_out, q_out_token_stride, q_out_head_stride,
      k_pages, v_pages, page_stride, page_head_stride, num_pages, page_size, error_flag,
      stream);
}

extern "C" size_t cascade_paged_attention_workspace_bytes(int64_t batch,
                                                          int64_t n_q_heads,
                                                          int64_t n_kv_heads,
                                                          int64_t head_dim,
                                                          int64_t max_length) {
  if (batch <= 0 || n_kv_heads <= 0 || n_q_heads <= 0 || n_q_heads % n_kv_heads ||
      n_q_heads / n_kv_heads > kPagedGroup || (head_dim != 64 && head_dim != 128) ||
      max_length <= 0 || max_length > 0x7fffffff - 64)
    return 0;
  // enough for fewer rows too: a launch of more than kPagedMaxBatch needs none
  const PagedPlan p = paged_plan(batch < kPagedMaxBatch ? batch : kPagedMaxBatch, n_q_heads,
                                 n_kv_heads, head_dim, max_length);
  return kPagedAlign + p.plan_bytes + p.ml_bytes + p.acc_bytes;
}

extern "C" int cascade_paged_decode_attention_bf16(
    const void *q, int64_t q_token_stride, int64_t q_head_stride,
    const void *k_pages, const void *v_pages, int64_t page_stride,
    int64_t page_head_stride, int64_t num_pages, int64_t page_size,
    const int32_t *page_table, int64_t table_stride, int64_t sequences,
    const int32_t *lengths, const int32_t *rows, int64_t batch, int64_t max_length,
    int64_t n_q_heads, int64_t n_kv_heads, int64_t head_dim, float scale,
    void *out, int64_t out_token_stride, int64_t out_head_stride, void *workspace,
    size_t workspace_bytes, int32_t *error_flag, void *stream) {
  if (q == nullptr || k_pages == nullptr || v_pages == nullptr ||
      page_table == nullptr || lengths == nullptr || out == nullptr ||
      workspace == nullptr)
    return CASCADE_EINVAL;
  if (batch <= 0 || batch > 0x7fffffff || n_kv_heads <= 0 || sequences <= 0 ||
      num_pages <= 0 || num_pages > 0x7fffffff || max_length <= 0)
    return CASCADE_EINVAL;
  PagedAttnArgs a{};
  if ((head_dim != 64 && head_dim != 128) || n_q_heads <= 0 || n_q_heads % n_kv_heads ||
      n_q_heads / n_kv_heads > kPagedGroup || n_kv_heads > 0xffff ||
      batch > kMaxThreads / (kWholeWaves * kWave) / n_kv_heads ||
      !page_shift_of(page_size, &a.page_shift) || max_length > 0x7fffffff - 64)
    return CASCADE_ESHAPE;
  if (table_stride < (max_length + page_size - 1) / page_size ||
      page_head_stride < page_size * head_dim ||
      page_stride < (n_kv_heads - 1) * page_head_stride + page_size * head_dim)
    return CASCADE_EINVAL;
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(out) ||
      !aligned16(workspace) || (reinterpret_cast<uintptr_t>(page_table) & 3) ||
      (reinterpret_cast<uintptr_t>(lengths) & 3) ||
      (reinterpret_cast<uintptr_t>(rows) & 3) ||
      (reinterpret_cast<uintptr_t>(error_flag) & 3))
    return CASCADE_EALIGN;
  const int64_t strides[] = {q_token_stride, q_head_stride, page_stride,
                             page_head_stride, out_token_stride, out_head_stride};
  for (int64_t s : strides)
    if (!stride_ok(s)) return CASCADE_EALIGN;
  const PagedPlan p = paged_plan(batch, n_q_heads, n_kv_heads, head_dim, max_length);
  if (p.split && batch > kMaxThreads / kPagedMergeThreads / n_q_heads) return CASCADE_ESHAPE;
  if (workspace_bytes < kPagedAlign + p.plan_bytes + p.ml_bytes + p.acc_bytes)
    return CASCADE_EWORKSPACE;
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
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = static_cast<uint16_t *>(out);
  a.out_token = out_token_stride;
  a.out_head = out_head_stride;
  a.error = error_flag;
  a.batch = static_cast<int32_t>(batch);
  a.kv_heads = static_cast<int32_t>(n_kv_heads);
  const dim3 block((p.split ? kPagedWaves : kWholeWaves) * kWave);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (!p.split) {
    const dim3 grid(static_cast<unsigned>(batch * n_kv_heads));
    return head_dim == 128
               ? launch_kernel(paged_attention_kernel<128, false>, grid, block, 0, s, a)
               : launch_kernel(paged_attention_kernel<64, false>, grid, block, 0, s, a);
  }
  unsigned char *ws = static_cast<unsigned char *>(workspace);
  a.runs = static_cast<int32_t>(p.runs);
  a.per_round = 1.0 / static_cast<double>(p.round);
  a.per_two = 1.0 / static_cast<double>(p.two);
  a.plan = reinterpret_cast<int32_t *>(ws);
  a.part_ml = reinterpret_cast<float *>(ws + p.plan_bytes);
  a.part_acc = reinterpret_cast<float *>(ws + p.plan_bytes + p.ml_bytes);
  const dim3 grid(static_cast<unsigned>(p.runs * n_kv_heads));
  const dim3 merge(static_cast<unsigned>(batch * n_q_heads));
  const dim3 merge_block(kPagedMergeThreads);
  if (head_dim == 128) {
    const hipError_t e =
        launch_kernel(paged_attention_kernel<128, true>, grid, block, 0, s, a);
    if (e != hipSuccess) return e;
    return launch_kernel(paged_merge_kernel<128>, merge, merge_block, 0, s, a);
  }
  const hipError_t e = launch_kernel(paged_attention_kernel<64, true>, grid, block, 0, s, a);
  if (e != hipSuccess) return e;
  return launch_kernel(paged_merge_kernel<64>, merge, merge_block, 0, s, a);
}

extern "C" int cascade_copy_pages(void *pages, int64_t planes, int64_t plane_bytes,
                                  int64_t num_pages, int64_t page_bytes,
                                  const int32_t *pairs, int64_t count,
                                  int32_t *error_flag, void *stream) {
  if (pages == nullptr || pairs == nullptr) return CASCADE_EINVAL;
  if (planes <= 0 || planes > 0x7fffffff || num_pages <= 0 || num_pages > 0x7fffffff ||
      page_bytes <= 0 || count <= 0 || count > 0x7fffffff ||
      page_bytes > (int64_t{1} << 40) || plane_bytes < 0 ||
      (planes > 1 && plane_bytes / num_pages < page_bytes))
    return CASCADE_EINVAL;
  if ((page_bytes & 15) || (plane_bytes & 15) || !aligned16(pages) ||
      (reinterpret_cast<uintptr_t>(pairs) & 3) ||
      (reinterpret_cast<uintptr_t>(error_flag) & 3))
    return CASCADE_EALIGN;
  CopyPagesArgs a{};
  a.base = static_cast<unsigned char *>(pages);
  a.plane_bytes = plane_bytes;
  a.page_bytes = page_bytes;
  a.num_pages = static_cast<int32_t>(num_pages);
  a.planes = static_cast<int32_t>(planes);
  a.pairs = pairs;
  a.pieces = (page_bytes + kCopyPiece - 1) / kCopyPiece;
  if (a.pieces > INT64_MAX / planes / count) return CASCADE_EINVAL;
  a.total = a.pieces * planes * count;
  a.error = error_flag;
  const int64_t blocks = a.total < (1 << 22) ? a.total : (1 << 22);
  return launch_kernel(copy_pages_kernel, dim3(static_cast<unsigned>(blocks)),
                       dim3(kCopyThreads), 0, static_cast<hipStream_t>(stream), a);
}
