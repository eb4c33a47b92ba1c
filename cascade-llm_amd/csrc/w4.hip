// Products of rows with matrices of 4-bit weights (gfx950).
//
// The layout (include/cascade_hip.h) is that of a wave's load: a tile of 16
// matrix rows and 128 columns is 1 KiB, of which lane l takes the 16 bytes at
// 16 l: row l % 16, and of each 32 columns the eight from 8 (l / 16) on, which
// is its piece of an MFMA operand.
#include "cascade_device.h"
#include "cascade_internal.h"

namespace cascade {

struct W4Matrix {
  const u32x4 *packed;
  const uint16_t *scales;
  const uint8_t *zeros;  // nullable: 8
};

struct W4Args {
  const uint16_t *x;
  int64_t x_stride;
  W4Matrix w[2];  // gate and up for SwiGLU
  int32_t m, n, k;
  int32_t tiles;   // of 128 columns
  int32_t groups;  // of a row
  int32_t group_shift;
  const uint16_t *residual;
  int64_t residual_stride;
  void *y;
  int64_t y_stride;
  int32_t f32;  // y's type
  int32_t once;  // the matrix is read past the caches
  int32_t wide;  // four columns of y and residual are one access
  int32_t splits;  // of K over workgroups
  float *partial;  // [splits][m][16 ceil(n / 16)] of these
};

enum W4Out { kW4Bf16, kW4F32, kW4Swiglu };

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// Eight 4-bit values of a packed word as 16 + q in bf16, an MFMA operand: the
// value lands in the upper mantissa bits of 16.0, so one rotation and one
// and-or give two of them.
__device__ __forceinline__ u32x4 w4_operand(uint32_t word) {
  uint32_t mask = 0x00780078u, base = 0x41804180u;
  asm("" : "+s"(mask));  // (registers: an and-or takes no constant)
  asm("" : "+v"(base));
  u32x4 r;
  r[0] = (word & mask) | base;
  r[1] = ((word >> 4) & mask) | base;
  r[2] = ((word >> 8) & mask) | base;
  r[3] = (__builtin_amdgcn_alignbit(word, word, 12) & mask) | base;
  return r;
}

// The same as 48 + q - zero, from 0x42404240 - 0x00040004 zero: 33 .. 63, where
// the mantissas of bf16 are linear and the sums of the halves carry nothing.
__device__ __forceinline__ u32x4 w4_operand_from(uint32_t word, uint32_t base) {
  constexpr uint32_t kMask = 0x003c003cu;
  u32x4 r;
  r[0] = ((word >> 1) & kMask) + base;
  r[1] = ((word >> 5) & kMask) + base;
  r[2] = ((word >> 9) & kMask) + base;
  r[3] = (__builtin_amdgcn_alignbit(word, word, 13) & kMask) + base;
  return r;
}

// Buffer descriptors: what lies past the end reads as zeros.  The bounds hold
// for voffset alone, so all of an offset that may lie there goes into it.
typedef __amdgpu_buffer_rsrc_t Rsrc;

__device__ __forceinline__ Rsrc w4_rsrc(const void *base, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), 0,
                                           static_cast<int>(bytes), 0x00020000);
}

constexpr int64_t kW4Rows = 0xffff * 64;  // of x: a grid's second dimension
constexpr int kNontemporal = 2;
// Matrices of which the memory-side cache (256 MB) holds little at the next
// pass go past it: 5 rows by 128256 x 4096 (263 MB) 51.9 -> 49.3 us.  Smaller
// ones lose: gate and up 14336 x 4096 (59 MB), one row, 12.4 -> 13.4.
constexpr int64_t kW4OnceBytes = 128 << 20;
constexpr int64_t kW4AgainBytes = 60 << 20;  // see w4_plan
constexpr int kOutside = 0x7f000000;  // past every descriptor's end, with room for 2^24 more

// The output of four matrix rows for one row of x.
__device__ __forceinline__ void w4_store(const W4Args &a, f32x4 v, int row, int col) {
  const int64_t y = row * a.y_stride + col;
  if (a.wide && col + 4 <= a.n) {
    if (a.f32) {
      *reinterpret_cast<f32x4 *>(static_cast<float *>(a.y) + y) = v;
      return;
    }
    if (a.residual != nullptr) {
      const u32x2 add =
          *reinterpret_cast<const u32x2 *>(a.residual + row * a.residual_stride + col);
      v[0] += lo_bf16(add[0]);
      v[1] += hi_bf16(add[0]);
      v[2] += lo_bf16(add[1]);
      v[3] += hi_bf16(add[1]);
    }
    *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(a.y) + y) =
        u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    return;
  }
  for (int r = 0; r < 4 && col + r < a.n; ++r) {
    float out = v[0];
    if (a.f32) {
      static_cast<float *>(a.y)[y + r] = out;
    } else {
      if (a.residual != nullptr)
        out += bf16_to_f32(a.residual[row * a.residual_stride + col + r]);
      static_cast<uint16_t *>(a.y)[y + r] = f32_to_bf16(out);
    }
    v = f32x4{v[1], v[2], v[3], 0.0f};  // (no indexing of registers)
  }
}

// Loads to LDS that the compiler does not see (dma_lds16): 4 bytes a lane, and
// with a scalar part of the offset, which the bounds do not see: for what is
// known to lie inside.
__device__ __forceinline__ void dma_lds4(const u32x4 &rsrc, int voff, uint32_t lds) {
  u32x4 r;
  r.x = __builtin_amdgcn_readfirstlane(rsrc.x);
  r.y = __builtin_amdgcn_readfirstlane(rsrc.y);
  r.z = __builtin_amdgcn_readfirstlane(rsrc.z);
  r.w = __builtin_amdgcn_readfirstlane(rsrc.w);
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :: "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(r)
               : "memory", "m0");
}

__device__ __forceinline__ void dma_lds16_inside(const u32x4 &rsrc, int voff, int soff,
                                                 uint32_t lds) {
  u32x4 r;
  r.x = __builtin_amdgcn_readfirstlane(rsrc.x);
  r.y = __builtin_amdgcn_readfirstlane(rsrc.y);
  r.z = __builtin_amdgcn_readfirstlane(rsrc.z);
  r.w = __builtin_amdgcn_readfirstlane(rsrc.w);
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :: "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(r),
                  "s"(__builtin_amdgcn_readfirstlane(soff))
               : "memory", "m0");
}
__device__ __forceinline__ void dma_lds4_inside(const u32x4 &rsrc, int voff, int soff,
                                                uint32_t lds) {
  u32x4 r;
  r.x = __builtin_amdgcn_readfirstlane(rsrc.x);
  r.y = __builtin_amdgcn_readfirstlane(rsrc.y);
  r.z = __builtin_amdgcn_readfirstlane(rsrc.z);
  r.w = __builtin_amdgcn_readfirstlane(rsrc.w);
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dword %1, %2, %3 offen lds"
               :: "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(r),
                  "s"(__builtin_amdgcn_readfirstlane(soff))
               : "memory", "m0");
}

// y[r, i] = sum over K of x[r, k] scale[i, k/group] (q[i, k] - zero[i, k/group]).
//
// A wave holds NT tiles of 16 matrix rows (A) by MT of 16 rows of x (B) and goes
// through K in steps of 128 columns; WN waves share a step's x, WK waves take
// turns at the steps and are joined at the end, and a long K is split over
// a.splits workgroups, joined by a second launch.
//
// The weights become MFMA operands without a float conversion: 4 bits in the
// mantissa of 16 (or 32 .. 63) are 16 + q, and the product's sum begins with
// -24 (or, with zero points in the operand, -48) times the sum of x, which is
// an MFMA of its own for all NT tiles.  Both are exact in bf16, and sums are
// fp32; the sum over a group is scaled in fp32, so that no weight is rounded.
// The start costs what cancels: a group's fp32 sum has terms of 24 |x| (48 |x|
// with zero points) and rounds as they do, not as (q - zero) x would.  Of rows
// whose x has no common sign little is seen (4096 columns 0.9e-7 to 1.6e-7 off,
// plain fp32 sums 3.4e-7), of x all positive 1.2e-7 to 9.7e-7 (3.1e-7).  A large
// x under weights of zero leaves that rounding of itself behind, and a matrix row
// of zeros gives as little, not exactly 0.
//
// x, scales and zero points go to LDS without passing registers, the weights,
// which one wave needs once, to registers, both a step ahead: what a step waits
// for at its start was sent for a whole step before.
//
// What bounds it: vector instructions, of which a SIMD starts one in 4.5 cycles
// (shifts and masks of several waves in 2.5), but one wave alone one in 7.4,
// whatever it is; so tiles are kept small enough for four waves a SIMD (128
// registers).  Gate and up of 61 rows by 14336 x 4096, group 64 with zeros: 32 us,
// where tiles of 4 x 4 took 35 to 49; a step of 2 x 4 tiles, 48 MFMAs beside 200
// vector instructions (64 the scaling, 96 the operands) and 16 reads of x from
// LDS, takes two waves of a SIMD 1.7 us, 0.7 of it the MFMAs.  Few rows: one by
// 14336 x 4096 twice, group 128, 12.0 us, 5.1 TB/s; 5 by 128256 x 4096 44.8 us,
// 6.1 TB/s.
template <bool SWIGLU, bool ZEROS, int GP, int NT, int MT, int WN, int WK>
struct W4Tile {
  static constexpr int WAVES = WN * WK;
  static constexpr int PARTS = SWIGLU ? 2 : 1;
  static constexpr int RT = NT / PARTS;                  // tiles of one matrix a wave
  static constexpr int SCALES = (RT * GP * 8 + 63) / 64;  // loads of 64 dwords
  static constexpr int META = PARTS * 256 * (SCALES + (ZEROS ? 1 : 0));
  static constexpr int X = MT * 4096;                    // bytes of a K group's slot
  static constexpr int SLOT = WK * X + WAVES * META;
  static constexpr int SUM = WAVES * NT * MT * 1024;
  static constexpr int XLOADS = MT * 4 / WN;
  static constexpr int LDS = 2 * SLOT > SUM ? 2 * SLOT : SUM;
  static_assert(RT * GP * 4 <= 64 && MT * 4 % WN == 0 && LDS <= 160 * 1024, "shape");
};

template <bool SWIGLU, bool ZEROS, int GP, int NT, int MT, int WN, int WK>
__global__ __launch_bounds__(WN * WK * kWave) void w4_tile_kernel(W4Args a) {
  using R = W4Tile<SWIGLU, ZEROS, GP, NT, MT, WN, WK>;
  constexpr int RT = R::RT, J = 4 / GP;
  __shared__ __attribute__((aligned(16))) unsigned char s_tile[R::LDS];
  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int wn = wave % WN, kg = wave / WN;
  const int c16 = lane & 15, g4 = lane >> 4;
  const int first = (static_cast<int>(blockIdx.x) * WN + wn) * RT;  // row tile
  const int m0 = static_cast<int>(blockIdx.y) * 16 * MT;
  const int last_tile = (a.n + 15) / 16 - 1;
  const int64_t base_tile = min(first, last_tile);
  // of the wave's tiles, the offset of tile i from the first (past the last
  // one: the last one again)
  auto behind = [&](int i) { return static_cast<int>(min(first + i, last_tile) - base_tile); };

  Rsrc wr[R::PARTS];
  u32x4 sr[R::PARTS], zr[R::PARTS];
#pragma unroll
  for (int p = 0; p < R::PARTS; ++p) {
    const W4Matrix &w = a.w[p];
    wr[p] = w4_rsrc(w.packed + base_tile * a.tiles * kWave,
                    static_cast<int64_t>(a.tiles) * 1024 * RT);
    sr[p] = buffer_rsrc_words(w.scales + base_tile * a.groups * 16,
                              static_cast<int64_t>(a.groups) * 32 * RT);
    if constexpr (ZEROS)
      zr[p] = buffer_rsrc_words(w.zeros + base_tile * a.groups * 16,
                                static_cast<int64_t>(a.groups) * 16 * RT);
  }
  const int rows = min(16 * MT, a.m - m0);
  const int pitch = static_cast<int>(a.x_stride) * 2;
  const u32x4 xr = buffer_rsrc_words(a.x + m0 * a.x_stride,
                                     static_cast<int64_t>(rows - 1) * pitch + 2 * a.k);
  int xoff[R::XLOADS];
#pragma unroll
  for (int i = 0; i < R::XLOADS; ++i) {
    const int block = wn + WN * i, row = 16 * (block / 4) + c16;
    xoff[i] = row < rows ? row * pitch + 64 * (block % 4) + 16 * g4 : kOutside;
  }
  // a lane's dword of the scales (of the zero points): tile and dword in it
  int soff[R::SCALES], sgroup[R::SCALES];
#pragma unroll
  for (int i = 0; i < R::SCALES; ++i) {
    const int at = i * kWave + lane, tile = at / (8 * GP), word = at % (8 * GP);
    sgroup[i] = word / 8;
    soff[i] = tile < RT ? behind(tile) * a.groups * 32 + word * 4 : kOutside;
  }
  const int ztile = lane / (4 * GP), zword = lane % (4 * GP);
  const int zoff = ztile < RT ? behind(ztile) * a.groups * 16 + zword * 4 : kOutside;
  const uint32_t lds = lds_address(s_tile);
  const uint32_t x_at = kg * R::X, meta_at = WK * R::X + wave * R::META;

  const int steps = (a.tiles + WK * a.splits - 1) / (WK * a.splits);
  const int t0 = static_cast<int>(blockIdx.z) * steps * WK + kg;
  const int tend = min(a.tiles, (static_cast<int>(blockIdx.z) + 1) * steps * WK);
  auto issue = [&](int t, uint32_t at, u32x4 (&w)[NT]) __attribute__((always_inline)) {
    if (t >= tend) return;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int from = (behind(i % RT) * a.tiles + t) * 1024;
      w[i] = a.once ? __builtin_amdgcn_raw_buffer_load_b128(wr[i / RT], lane * 16, from,
                                                            kNontemporal)
                    : __builtin_amdgcn_raw_buffer_load_b128(wr[i / RT], lane * 16, from, 0);
    }
    const uint32_t meta = at + meta_at;
    constexpr int PITCH = 256 * (R::SCALES + (ZEROS ? 1 : 0));
    if (128 * (t + 1) <= a.k) {
#pragma unroll
      for (int p = 0; p < R::PARTS; ++p) {
#pragma unroll
        for (int i = 0; i < R::SCALES; ++i)
          dma_lds4_inside(sr[p], soff[i], t * GP * 32, meta + p * PITCH + i * 256);
        if constexpr (ZEROS)
          dma_lds4_inside(zr[p], zoff, t * GP * 16, meta + p * PITCH + R::SCALES * 256);
      }
#pragma unroll
      for (int i = 0; i < R::XLOADS; ++i)
        dma_lds16_inside(xr, xoff[i], t * 256, at + x_at + (wn + WN * i) * 1024);
    } else {
#pragma unroll
      for (int p = 0; p < R::PARTS; ++p) {
#pragma unroll
        for (int i = 0; i < R::SCALES; ++i)
          dma_lds4(sr[p], t * GP + sgroup[i] < a.groups ? soff[i] + t * GP * 32 : kOutside,
                   meta + p * PITCH + i * 256);
        if constexpr (ZEROS)
          dma_lds4(zr[p], t * GP + zword / 4 < a.groups ? zoff + t * GP * 16 : kOutside,
                   meta + p * PITCH + R::SCALES * 256);
      }
#pragma unroll
      for (int i = 0; i < R::XLOADS; ++i) {
        const bool in = 128 * t + 32 * ((wn + WN * i) % 4) + 8 * g4 < a.k;
        dma_lds16(xr, in ? xoff[i] + t * 256 : kOutside, at + x_at + (wn + WN * i) * 1024);
      }
    }
  };
  f32x4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[i][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  // the sum's start: -24 x = -(16 + 8) x, or -48 x
  constexpr uint32_t kFirst = ZEROS ? 0xc240c240u : 0xc1c0c1c0u;
  const u32x4 first_op = {kFirst, kFirst, kFirst, kFirst};
  auto step = [&](uint32_t slot, const u32x4 (&w)[NT]) __attribute__((always_inline)) {
    const unsigned char *at = s_tile + slot;
    const u32x4 *xs_at = reinterpret_cast<const u32x4 *>(at + x_at) + lane;
#pragma unroll
    for (int g = 0; g < GP; ++g) {
      u32x4 op[NT][J];
      float scale[NT][4];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const unsigned char *meta =
            at + meta_at + (i / RT) * 256 * (R::SCALES + (ZEROS ? 1 : 0));
        const u32x2 two =
            *reinterpret_cast<const u32x2 *>(meta + ((i % RT) * GP + g) * 32 + 8 * g4);
        scale[i][0] = lo_bf16(two[0]);
        scale[i][1] = hi_bf16(two[0]);
        scale[i][2] = lo_bf16(two[1]);
        scale[i][3] = hi_bf16(two[1]);
        uint32_t zero = 0;
        if constexpr (ZEROS)
          zero = 0x42404240u -
                 __umul24(meta[R::SCALES * 256 + ((i % RT) * GP + g) * 16 + c16], 0x00040004u);
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const uint32_t word = w[i][J * g + j];
          op[i][j] = ZEROS ? w4_operand_from(word, zero) : w4_operand(word);
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        u32x4 x[J];
        f32x4 start = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < J; ++j) {
          x[j] = xs_at[(4 * m + J * g + j) * kWave];
          start = mfma_16x16x32_bf16(first_op, x[j], start);
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          f32x4 part = start;
#pragma unroll
          for (int j = 0; j < J; ++j) part = mfma_16x16x32_bf16(op[i][j], x[j], part);
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][m][r] = fmaf(scale[i][r], part[r], acc[i][m][r]);
        }
      }
    }
  };
  auto turn = [&](int t, uint32_t slot, u32x4 (&w)[NT], u32x4 (&next)[NT])
      __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
    if constexpr (WN > 1) __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    issue(t + WK, lds + (R::SLOT - slot), next);
    __builtin_amdgcn_sched_barrier(0);
    if (t < tend) step(slot, w);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  u32x4 even[NT], odd[NT];
  issue(t0, lds, even);
  for (int s = 0, t = t0; s < steps; s += 2, t += 2 * WK) {
    turn(t, 0, even, odd);
    if (s + 1 < steps) turn(t + WK, R::SLOT, odd, even);
  }
  __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
  __syncthreads();
  // The waves' sums, four matrix rows of one row of x a place.  Places are
  // turned so that both a wave's tile and a row's neighbours (which leave
  // together) lie in different banks.
  constexpr int T = WN * RT, Q = 4 * T, ROUND = T < 4 ? 4 / T : 1;
  f32x4 *s_sum = reinterpret_cast<f32x4 *>(s_tile);
  auto place = [&](int tile, int m, int row, int quad) {
    return (tile * MT + m) * kWave + 16 * (quad & 3) + ((row + ROUND * quad) & 15);
  };
  constexpr int kAll = R::PARTS * T * MT * kWave;  // places of a K group
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int m = 0; m < MT; ++m)
      s_sum[kg * kAll + place((i / RT) * T + wn * RT + i % RT, m, c16,
                              4 * (wn * RT + i % RT) + g4)] = acc[i][m];
  __syncthreads();
  for (int item = tid; item < Q * MT * 16; item += R::WAVES * kWave) {
    const int quad = item % Q, r16 = item / Q % 16, m = item / (Q * 16);
    auto joined = [&](int part) {
      const int from = place(part * T + quad / 4, m, r16, quad);
      f32x4 v = s_sum[from];
#pragma unroll
      for (int k = 1; k < WK; ++k) {
        const f32x4 u = s_sum[k * kAll + from];
        v += u;
      }
      return v;
    };
    f32x4 v = joined(0);
    if constexpr (SWIGLU) {
      const f32x4 u = joined(1);
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = v[r] / (1.0f + __expf(-v[r])) * u[r];
    }
    const int row = m0 + 16 * m + r16;
    const int col = 16 * T * static_cast<int>(blockIdx.x) + 4 * quad;
    if (row >= a.m || col > 16 * last_tile + 15) continue;
    if (a.splits > 1)
      *reinterpret_cast<f32x4 *>(
          a.partial + (static_cast<int64_t>(blockIdx.z) * a.m + row) * 16 * (last_tile + 1) +
          col) = v;
    else
      w4_store(a, v, row, col);
  }
}

// Sums over K that several workgroups took parts of.
__global__ __launch_bounds__(256) void w4_join_kernel(W4Args a) {
  const int quads = (a.n + 15) / 16 * 4;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = item / quads;
  const int col = 4 * static_cast<int>(item - row * quads);
  if (row >= a.m || col >= a.n) return;
  const f32x4 *from = reinterpret_cast<const f32x4 *>(a.partial) + item;
  f32x4 v = *from;
  for (int z = 1; z < a.splits; ++z) {
    const f32x4 u = from[static_cast<int64_t>(z) * a.m * quads];
    v += u;
  }
  w4_store(a, v, static_cast<int>(row), col);
}

template <bool SWIGLU, int NT, int MT, int WN, int WK>
static int launch_w4_tile(const W4Args &a, hipStream_t s) {
  constexpr int RT = SWIGLU ? NT / 2 : NT;
  const int64_t tiles = (a.n + 15) / 16;
  const int64_t x = (tiles + RT * WN - 1) / (RT * WN), y = (a.m + 16 * MT - 1) / (16 * MT);
  if (y > 0xffff || x > 0xffffffffll / (WN * WK * kWave)) return CASCADE_ESHAPE;
  const dim3 grid(static_cast<unsigned>(x), static_cast<unsigned>(y),
                  static_cast<unsigned>(a.splits));
  const dim3 block(WN * WK * kWave);
  const int which = (a.group_shift - 5) + (a.w[0].zeros != nullptr ? 3 : 0);
  hipError_t status;
  switch (which) {
    case 0: status = launch_kernel(w4_tile_kernel<SWIGLU, false, 4, NT, MT, WN, WK>, grid, block, 0, s, a); break;
    case 1: status = launch_kernel(w4_tile_kernel<SWIGLU, false, 2, NT, MT, WN, WK>, grid, block, 0, s, a); break;
    case 2: status = launch_kernel(w4_tile_kernel<SWIGLU, false, 1, NT, MT, WN, WK>, grid, block, 0, s, a); break;
    case 3: status = launch_kernel(w4_tile_kernel<SWIGLU, true, 4, NT, MT, WN, WK>, grid, block, 0, s, a); break;
    case 4: status = launch_kernel(w4_tile_kernel<SWIGLU, true, 2, NT, MT, WN, WK>, grid, block, 0, s, a); break;
    default: status = launch_kernel(w4_tile_kernel<SWIGLU, true, 1, NT, MT, WN, WK>, grid, block, 0, s, a);
  }
  if (status != hipSuccess || a.splits == 1) return status;
  const int64_t blocks = (tiles * 4 * a.m + 255) / 256;
  return launch_kernel(w4_join_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, a);
}

// The shape of a product's workgroups and the parts that K is split into, from
// sizes alone; times in us, group 64 with zeros.
// - 16 rows of x a workgroup, up to 16 rows and where reading the matrix again
//   for each 16 costs little, up to 60 MB in all: 2048 x 2048, 64 rows, 5.1 / 9.3;
//   1024 x 4096, 128 rows, 7.5 / 11.0; 4096 x 4096, 32 rows, 7.5 / 11.4, 65 rows
//   (42 MB) 14.0 / 14.6; 14336 x 4096, 24 rows (59 MB), 15.0 / 16.7, 64 rows (117
//   MB) 25.3 / 21.4.  Of these, 4 tiles a wave, of which 4 share K (x is read from
//   LDS once for four tiles), where the other form, 2 tiles and 8 waves, would
//   give a CU more than one workgroup: gate and up 14336 x 4096, 16 rows, 16.6 /
//   21.6, 4096 x 4096, 16 rows, 9.4 / 7.2; up to 4 rows, whose x is short, more
//   than two: 14336 x 4096, one row, 10.7 / 9.4, 16 rows 11.1 / 12.4.
// - More rows: 32 of x a workgroup; 64 where two of these a CU are left: 157
//   rows, gate and up 14336 x 4096: 74 with 64, 80 with 32; 613 rows, 4096 x
//   4096: 47 / 44.
// - Parts of K up to a workgroup a CU (two for more rows), which have tiles
//   enough to be worth the second launch.  The wide form from 28 on: 16 rows, 4096
//   x 14336 whole 25.5, in 4 parts 12.7; 4096 x 8192 10.1 in two parts, 11.0 in four
//   of 16 tiles; 6144 x 4096 7.5 whole, 9.4 in two of 16.  The other from 32 on: 16
//   rows, 2048 x 4096 6.8 whole, 6.9 in two of 16, one row 5.6 and 6.1; one row,
//   1024 x 14336 12.9 whole, 8.3 in three (where K is that long, seven of 16 take
//   7.3).  More rows from 8 on, where the limit is mostly the workgroups wanted: 61
//   rows 4096 x 14336 whole 62, 4 parts 22.3, 8 21.3, 14 26.2; 157 rows 4096 x 4096
//   20.1 in three, 21.5 in two; 613 rows 45 whole, four parts 52.  Gate and up have
//   no workspace and are not split.
enum W4Shape { kW4Rows16Wide, kW4Rows16, kW4Rows32, kW4Rows64 };

struct W4Plan {
  W4Shape shape;
  int32_t splits;
};

static W4Plan w4_plan(int64_t m, int64_t n, int64_t k, bool swiglu) {
  const int64_t row_tiles = (n + 15) / 16 * (swiglu ? 2 : 1), tiles = (k + 127) / 128;
  // parts of `least` tiles or more, so many that there are `wanted` workgroups
  auto splits = [&](int64_t groups, int64_t wanted, int64_t least) {
    if (swiglu) return int64_t{1};
    int64_t parts = wanted / groups;
    if (parts > tiles / least) parts = tiles / least;
    return parts < 1 ? int64_t{1} : parts;
  };
  auto plan = [](W4Shape shape, int64_t parts) {
    return W4Plan{shape, static_cast<int32_t>(parts)};
  };
  const int64_t blocks16 = (m + 15) / 16;
  if (m <= 16 || row_tiles * tiles * 1024 * blocks16 <= kW4AgainBytes) {
    const int64_t groups = (row_tiles + 3) / 4 * blocks16, parts = splits(groups, 256, 28);
    if (groups * parts > (m <= 4 ? 256 : 128)) return plan(kW4Rows16Wide, parts);
    return plan(kW4Rows16, splits((row_tiles + 1) / 2 * blocks16, 256, 32));
  }
  const int64_t groups = (row_tiles + 7) / 8;
  if (groups * ((m + 63) / 64) >= 512) return plan(kW4Rows64, 1);
  return plan(kW4Rows32, splits(groups * ((m + 31) / 32), 512, 8));
}

static int64_t w4_workspace_bytes(const W4Plan &plan, int64_t m, int64_t n) {
  return plan.splits == 1 ? 0 : plan.splits * m * ((n + 15) / 16 * 16) * 4;
}

template <int OUT>
static int launch_w4(W4Args a, int64_t x_stride, int64_t m, int64_t n, int64_t k,
                     int64_t group, void *workspace, size_t workspace_bytes,
                     void *stream) {
  if (m <= 0 || n <= 0 || k <= 0) return CASCADE_EINVAL;
  if (k & 7) return CASCADE_EALIGN;
  if ((group != 32 && group != 64 && group != 128) || m > kW4Rows || n > 0x7fffff ||
      k > 0x7fffff || x_stride > 0x7fffff)
    return CASCADE_ESHAPE;
  if (x_stride < 0 || (m > 1 && x_stride < k) || a.y_stride < 0 ||
      (m > 1 && a.y_stride < n) || a.residual_stride < 0)
    return CASCADE_EINVAL;
  if ((x_stride & 7) || !aligned16(a.x)) return CASCADE_EALIGN;
  for (int i = 0; i < (OUT == kW4Swiglu ? 2 : 1); ++i) {
    if (a.w[i].packed == nullptr || a.w[i].scales == nullptr) return CASCADE_EINVAL;
    if (!aligned16(a.w[i].packed) || !aligned16(a.w[i].scales) || !aligned16(a.w[i].zeros))
      return CASCADE_EALIGN;
  }
  if (a.x == nullptr || a.y == nullptr || a.x == a.y) return CASCADE_EINVAL;
  if (OUT == kW4Swiglu && (a.w[0].zeros == nullptr) != (a.w[1].zeros == nullptr))
    return CASCADE_EINVAL;
  if ((reinterpret_cast<uintptr_t>(a.y) & (OUT == kW4F32 ? 3 : 1)) ||
      (reinterpret_cast<uintptr_t>(a.residual) & 1))
    return CASCADE_EALIGN;
  a.x_stride = x_stride;
  a.m = static_cast<int32_t>(m);
  a.n = static_cast<int32_t>(n);
  a.k = static_cast<int32_t>(k);
  a.tiles = static_cast<int32_t>((k + 127) / 128);
  a.group_shift = group == 128 ? 7 : group == 64 ? 6 : 5;
  a.groups = static_cast<int32_t>((k + group - 1) / group);
  a.f32 = OUT == kW4F32;
  a.wide = (a.y_stride & 3) == 0 && (a.residual_stride & 3) == 0 &&
           (reinterpret_cast<uintptr_t>(a.y) & (OUT == kW4F32 ? 15 : 7)) == 0 &&
           (reinterpret_cast<uintptr_t>(a.residual) & 7) == 0;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  constexpr bool kSwiglu = OUT == kW4Swiglu;
  const W4Plan plan = w4_plan(m, n, k, kSwiglu);
  if (plan.splits > 1) {
    if (workspace == nullptr || static_cast<int64_t>(workspace_bytes) <
                                    w4_workspace_bytes(plan, m, n))
      return CASCADE_EWORKSPACE;
    if (!aligned16(workspace)) return CASCADE_EALIGN;
  }
  a.splits = plan.splits;
  a.partial = static_cast<float *>(workspace);
  a.once = m <= 16 && (n + 15) / 16 * a.tiles * 1024 * (kSwiglu ? 2 : 1) >= kW4OnceBytes;
  switch (plan.shape) {
    case kW4Rows16Wide: return launch_w4_tile<kSwiglu, 4, 1, 1, 4>(a, s);
    case kW4Rows16: return launch_w4_tile<kSwiglu, 2, 1, 1, 8>(a, s);
    case kW4Rows32: return launch_w4_tile<kSwiglu, 2, 2, 4, 2>(a, s);
    default: return launch_w4_tile<kSwiglu, 2, 4, 4, 2>(a, s);
  }
}

}  // namespace cascade

using namespace cascade;

extern "C" size_t cascade_linear_w4_workspace_bytes(int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || k <= 0 || m > kW4Rows || n > 0x7fffff || k > 0x7fffff) return 0;
  return static_cast<size_t>(w4_workspace_bytes(w4_plan(m, n, k, false), m, n));
}

extern "C" int cascade_linear_w4_bf16(const void *x, int64_t x_stride, const void *packed,
                                      const void *scales, const void *zeros, int64_t m,
                                      int64_t n, int64_t k, int64_t group,
                                      const void *residual, int64_t residual_stride,
                                      void *y, int64_t y_stride, void *workspace,
                                      size_t workspace_bytes, void *stream) {
  W4Args a{};
  a.x = static_cast<const uint16_t *>(x);
  a.w[0] = {static_cast<const u32x4 *>(packed), static_cast<const uint16_t *>(scales),
            static_cast<const uint8_t *>(zeros)};
  a.residual = static_cast<const uint16_t *>(residual);
  a.residual_stride = residual_stride;
  a.y = y;
  a.y_stride = y_stride;
  return launch_w4<kW4Bf16>(a, x_stride, m, n, k, group, workspace, workspace_bytes, stream);
}

extern "C" int cascade_linear_w4_f32out_bf16(const void *x, int64_t x_stride,
                                             const void *packed, const void *scales,
                                             const void *zeros, int64_t m, int64_t n,
                                             int64_t k, int64_t group, float *y,
                                             int64_t y_stride, void *workspace,
                                             size_t workspace_bytes, void *stream) {
  W4Args a{};
  a.x = static_cast<const uint16_t *>(x);
  a.w[0] = {static_cast<const u32x4 *>(packed), static_cast<const uint16_t *>(scales),
            static_cast<const uint8_t *>(zeros)};
  a.y = y;
  a.y_stride = y_stride;
  return launch_w4<kW4F32>(a, x_stride, m, n, k, group, workspace, workspace_bytes, stream);
}

extern "C" int cascade_gate_up_swiglu_w4_bf16(
    const void *x, int64_t x_stride, const void *gate_packed, const void *gate_scales,
    const void *gate_zeros, const void *up_packed, const void *up_scales,
    const void *up_zeros, int64_t m, int64_t n_half, int64_t k, int64_t group, void *y,
    int64_t y_stride, void *stream) {
  W4Args a{};
  a.x = static_cast<const uint16_t *>(x);
  a.w[0] = {static_cast<const u32x4 *>(gate_packed),
            static_cast<const uint16_t *>(gate_scales),
            static_cast<const uint8_t *>(gate_zeros)};
  a.w[1] = {static_cast<const u32x4 *>(up_packed), static_cast<const uint16_t *>(up_scales),
            static_cast<const uint8_t *>(up_zeros)};
  a.y = y;
  a.y_stride = y_stride;
  return launch_w4<kW4Swiglu>(a, x_stride, m, n_half, k, group, nullptr, 0, stream);
}
