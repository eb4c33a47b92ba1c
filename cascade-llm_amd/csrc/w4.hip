// Products of a few rows with matrices of 4-bit weights (gfx950).
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
};

enum W4Out { kW4Bf16, kW4F32, kW4Swiglu };

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kW4Ones = 0x3f803f80u;  // 1.0 twice

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

constexpr int kNontemporal = 2;
constexpr int64_t kW4FewBytes = 64 * 1024;  // of x in LDS
constexpr int kOutside = 0x7f000000;  // past every descriptor's end, with room for 2^24 more

// The output of four matrix rows for one row of x.  (One loop after the other:
// the residual's loads wait for nothing.)
__device__ __forceinline__ void w4_store(const W4Args &a, f32x4 v, int row, int col) {
  const int64_t y = row * a.y_stride + col;
  const int count = min(4, a.n - col);
  if (a.residual != nullptr) {
    const uint16_t *from = a.residual + row * a.residual_stride + col;
    uint16_t add[4] = {0, 0, 0, 0};
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < count) add[r] = from[r];
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] += bf16_to_f32(add[r]);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (r >= count) break;
    if (a.f32)
      static_cast<float *>(a.y)[y + r] = v[r];
    else
      static_cast<uint16_t *>(a.y)[y + r] = f32_to_bf16(v[r]);
  }
}

// Few rows of x, all of them in LDS: M rows as MFMA operands, tile by tile.
template <bool SWIGLU, bool ZEROS, int NT, int WAVES, int D, int GP>
__global__ __launch_bounds__(WAVES * kWave) void w4_few_kernel(W4Args a) {
  constexpr int RT = SWIGLU ? NT / 2 : NT;  // tiles of output columns
  constexpr int J = 4 / GP;                 // operands a group
  extern __shared__ u32x4 s_mem[];
  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int c16 = lane & 15, g4 = lane >> 4;
  const int t0 = static_cast<int>(blockIdx.x) * RT;
  const int last_tile = (a.n + 15) / 16 - 1;

  Rsrc wr[NT], sr[NT], zr[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const W4Matrix &w = a.w[SWIGLU ? i / RT : 0];
    const int64_t row = min(t0 + i % RT, last_tile);
    wr[i] = w4_rsrc(w.packed + row * a.tiles * kWave, static_cast<int64_t>(a.tiles) * 1024);
    sr[i] = w4_rsrc(w.scales + row * a.groups * 16, static_cast<int64_t>(a.groups) * 32);
    if constexpr (ZEROS)
      zr[i] = w4_rsrc(w.zeros + row * a.groups * 16, static_cast<int64_t>(a.groups) * 16);
  }
  const int woff = lane * 16, soff = g4 * 8, zoff = g4 * 4;
  struct Tile {
    u32x4 w[NT];
    u32x2 scale[NT][GP];
    uint32_t zero[NT][GP];
  };
  auto load = [&](int t, Tile &f) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      f.w[i] = __builtin_amdgcn_raw_buffer_load_b128(wr[i], woff + t * 1024, 0, kNontemporal);
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        f.scale[i][g] = __builtin_amdgcn_raw_buffer_load_b64(sr[i], soff + (t * GP + g) * 32, 0, 0);
        if constexpr (ZEROS)
          f.zero[i][g] =
              __builtin_amdgcn_raw_buffer_load_b32(zr[i], zoff + (t * GP + g) * 16, 0, 0);
      }
    }
  };
  Tile ring[D];
#pragma unroll
  for (int p = 0; p < D - 1; ++p) load(wave + p * WAVES, ring[p]);
  __builtin_amdgcn_sched_barrier(0);
  // unit (tile and quarter, row, eighth of the quarter)
  const int units = a.tiles * 16 * a.m;
  const Rsrc xr = w4_rsrc(a.x, (static_cast<int64_t>(a.m - 1) * a.x_stride + a.k) * 2);
  for (int u = tid; u < units; u += WAVES * kWave) {
    const int part = u / (4 * a.m), rest = u - part * (4 * a.m);
    const int k = 32 * part + 8 * (rest & 3);
    s_mem[u] = __builtin_amdgcn_raw_buffer_load_b128(
        xr, k < a.k ? ((rest >> 2) * static_cast<int>(a.x_stride) + k) * 2 : kOutside, 0, 0);
  }
  __syncthreads();
  const int xrow = min(c16, a.m - 1) * 4 + g4;  // columns past the last repeat it
  f32x4 acc[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  constexpr uint32_t kFirst = ZEROS ? kW4Ones : 0xc1c0c1c0u;
  const u32x4 ones = {kFirst, kFirst, kFirst, kFirst};
  auto step = [&](int t, const Tile &f) __attribute__((always_inline)) {
    u32x4 x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = s_mem[(4 * t + j) * (4 * a.m) + xrow];
#pragma unroll
    for (int g = 0; g < GP; ++g) {
      f32x4 xs = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < J; ++j) xs = mfma_16x16x32_bf16(ones, x[J * g + j], xs);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const uint32_t s01 = f.scale[i][g][0], s23 = f.scale[i][g][1];
        const float scale[4] = {lo_bf16(s01), hi_bf16(s01), lo_bf16(s23), hi_bf16(s23)};
        f32x4 part = xs;
        if constexpr (ZEROS) {
          const uint32_t z = f.zero[i][g];
          const float x16 = -16.0f * xs[0];  // (a column's sums are all alike)
          part[0] = fmaf(static_cast<float>(z & 255u), -xs[0], x16);
          part[1] = fmaf(static_cast<float>((z >> 8) & 255u), -xs[0], x16);
          part[2] = fmaf(static_cast<float>((z >> 16) & 255u), -xs[0], x16);
          part[3] = fmaf(static_cast<float>(z >> 24), -xs[0], x16);
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const uint32_t word = f.w[i][J * g + j];
          part = mfma_16x16x32_bf16(w4_operand(word), x[J * g + j], part);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][r] = fmaf(scale[r], part[r], acc[i][r]);
      }
    }
  };
  for (int t = wave; t < a.tiles;) {
#pragma unroll
    for (int p = 0; p < D; ++p) {
      load(t + (D - 1) * WAVES, ring[(p + D - 1) % D]);
      __builtin_amdgcn_sched_barrier(0);
      if (t < a.tiles) step(t, ring[p]);
      __builtin_amdgcn_sched_barrier(0);
      t += WAVES;
    }
  }
  __syncthreads();
  f32x4 *s_sum = reinterpret_cast<f32x4 *>(s_mem);
#pragma unroll
  for (int i = 0; i < NT; ++i) s_sum[(wave * NT + i) * kWave + lane] = acc[i];
  __syncthreads();
  for (int item = tid; item < RT * kWave; item += WAVES * kWave) {
    auto joined = [&](int at) {
      f32x4 v = s_sum[at];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) {
        const f32x4 u = s_sum[w * NT * kWave + at];
        v += u;
      }
      return v;
    };
    f32x4 v = joined(item);
    if constexpr (SWIGLU) {
      const f32x4 u = joined(item + RT * kWave);
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = v[r] / (1.0f + __expf(-v[r])) * u[r];
    }
    const int at = item % kWave, row = at & 15;
    if (row < a.m) w4_store(a, v, row, 16 * (t0 + item / kWave) + 4 * (at >> 4));
  }
}

template <bool SWIGLU, int NT, int WAVES, int D>
static int launch_w4_few(const W4Args &a, hipStream_t s) {
  constexpr int RT = SWIGLU ? NT / 2 : NT;
  const int64_t tiles = (a.n + 15) / 16;
  const int64_t x = (tiles + RT - 1) / RT;
  if (x > 0xffffffffll / (WAVES * kWave)) return CASCADE_ESHAPE;
  size_t lds = static_cast<size_t>(a.tiles) * 256 * a.m;
  if (lds < size_t{WAVES} * NT * 1024) lds = size_t{WAVES} * NT * 1024;
  const dim3 grid(static_cast<unsigned>(x));
  const dim3 block(WAVES * kWave);
  const int which = (a.group_shift - 5) + (a.w[0].zeros != nullptr ? 3 : 0);
  switch (which) {
    case 0: return launch_kernel(w4_few_kernel<SWIGLU, false, NT, WAVES, D, 4>, grid, block, lds, s, a);
    case 1: return launch_kernel(w4_few_kernel<SWIGLU, false, NT, WAVES, D, 2>, grid, block, lds, s, a);
    case 2: return launch_kernel(w4_few_kernel<SWIGLU, false, NT, WAVES, D, 1>, grid, block, lds, s, a);
    case 3: return launch_kernel(w4_few_kernel<SWIGLU, true, NT, WAVES, D, 4>, grid, block, lds, s, a);
    case 4: return launch_kernel(w4_few_kernel<SWIGLU, true, NT, WAVES, D, 2>, grid, block, lds, s, a);
    default: return launch_kernel(w4_few_kernel<SWIGLU, true, NT, WAVES, D, 1>, grid, block, lds, s, a);
  }
}

// Rows of x through LDS: see "Rings".
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

template <bool SWIGLU, bool ZEROS, int GP, int NT, int MT, int WN, int WK, int D>
struct W4Ring {
  static constexpr int WAVES = WN * WK;
  static constexpr int PARTS = SWIGLU ? 2 : 1;
  static constexpr int RT = NT / PARTS;        // tiles of one matrix a wave
  static constexpr int X = MT * 4096;          // bytes of a group's slot
  static constexpr int META = PARTS * 256 * (ZEROS ? 2 : 1);
  static constexpr int OWN = NT * 1024 + META;  // bytes of a wave's slot
  static constexpr int GROUP = X + WN * OWN;
  static constexpr int SLOT = WK * GROUP;
  static constexpr int SUM = WAVES * NT * MT * 1024;
  static constexpr int XLOADS = MT * 4 / WN;
  static constexpr int LOADS = XLOADS + NT + PARTS * (ZEROS ? 2 : 1);
  static constexpr int FIT = 160 * 1024 / SLOT, COUNT = 63 / LOADS + 1;
  static constexpr int FEW = FIT < COUNT ? FIT : COUNT;
  static constexpr int DEPTH = D < FEW ? D : FEW;  // slots
  static constexpr int LDS = DEPTH * SLOT > SUM ? DEPTH * SLOT : SUM;
  static_assert(RT * GP * 8 <= 64 && MT * 4 % WN == 0 && LDS <= 160 * 1024, "shape");
  static_assert(DEPTH >= 2, "a slot in use, a slot to come");
};

template <bool SWIGLU, bool ZEROS, int GP, int NT, int MT, int WN, int WK, int D>
__global__ __launch_bounds__(WN * WK * kWave) void w4_ring_kernel(W4Args a) {
  using R = W4Ring<SWIGLU, ZEROS, GP, NT, MT, WN, WK, D>;
  constexpr int RT = R::RT, J = 4 / GP, DEPTH = R::DEPTH;
  __shared__ __attribute__((aligned(16))) unsigned char s_ring[R::LDS];
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

  u32x4 wr[R::PARTS], sr[R::PARTS], zr[R::PARTS];
#pragma unroll
  for (int p = 0; p < R::PARTS; ++p) {
    const W4Matrix &w = a.w[p];
    wr[p] = buffer_rsrc_words(w.packed + base_tile * a.tiles * kWave,
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
  // a lane's dword of the scales (of the zero points) of tile lane / (8 GP)
  const int stile = lane / (8 * GP), sword = lane % (8 * GP);
  const int soff = stile < RT ? behind(stile) * a.groups * 32 + sword * 4 : kOutside;
  const int ztile = lane / (4 * GP), zword = lane % (4 * GP);
  const int zoff = ztile < RT ? behind(ztile) * a.groups * 16 + zword * 4 : kOutside;
  const uint32_t lds = lds_address(s_ring);
  const uint32_t x_at = kg * R::GROUP, own_at = x_at + R::X + wn * R::OWN;

  const int steps = (a.tiles + WK - 1) / WK;
  auto issue = [&](int s, int slot) __attribute__((always_inline)) {
    const int t = s * WK + kg;
    const uint32_t at = lds + slot * R::SLOT;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int tile = behind(i % RT) * a.tiles;
      // (past the end of K: past the end of the last tile)
      const int off = t >= a.tiles ? kOutside : lane * 16 + (tile + t) * 1024;
      dma_lds16(wr[i / RT], off, at + own_at + i * 1024);
    }
#pragma unroll
    for (int p = 0; p < R::PARTS; ++p) {
      const uint32_t meta = at + own_at + NT * 1024 + p * 256 * (ZEROS ? 2 : 1);
      dma_lds4(sr[p], t * GP + sword / 8 < a.groups ? soff + t * GP * 32 : kOutside, meta);
      if constexpr (ZEROS)
        dma_lds4(zr[p], t * GP + zword / 4 < a.groups ? zoff + t * GP * 16 : kOutside, meta + 256);
    }
    const bool whole = 128 * (t + 1) <= a.k;
#pragma unroll
    for (int i = 0; i < R::XLOADS; ++i) {
      const int block = wn + WN * i;
      const bool in = whole || 128 * t + 32 * (block % 4) + 8 * g4 < a.k;
      dma_lds16(xr, in ? xoff[i] + t * 256 : kOutside, at + x_at + block * 1024);
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
  auto step = [&](int slot) __attribute__((always_inline)) {
    const unsigned char *at = s_ring + slot * R::SLOT;
    const u32x4 *xs_at = reinterpret_cast<const u32x4 *>(at + x_at) + lane;
    const unsigned char *own = at + own_at;
    u32x4 w[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
      w[i] = reinterpret_cast<const u32x4 *>(own + i * 1024)[lane];
#pragma unroll
    for (int g = 0; g < GP; ++g) {
      u32x4 x[MT][J];
      f32x4 start[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        start[m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < J; ++j) {
          x[m][j] = xs_at[(4 * m + J * g + j) * kWave];
          start[m] = mfma_16x16x32_bf16(first_op, x[m][j], start[m]);
        }
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const unsigned char *meta = own + NT * 1024 + (i / RT) * 256 * (ZEROS ? 2 : 1);
        const u32x2 sc = *reinterpret_cast<const u32x2 *>(
            meta + ((i % RT) * GP + g) * 32 + 8 * g4);
        const uint32_t s01 = sc[0], s23 = sc[1];
        const float scale[4] = {lo_bf16(s01), hi_bf16(s01), lo_bf16(s23), hi_bf16(s23)};
        uint32_t zero = 0;
        if constexpr (ZEROS)
          zero = 0x42404240u -
                 __umul24(meta[256 + ((i % RT) * GP + g) * 16 + c16], 0x00040004u);
        u32x4 op[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const uint32_t word = w[i][J * g + j];
          op[j] = ZEROS ? w4_operand_from(word, zero) : w4_operand(word);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          f32x4 part = start[m];
#pragma unroll
          for (int j = 0; j < J; ++j) part = mfma_16x16x32_bf16(op[j], x[m][j], part);
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][m][r] = fmaf(scale[r], part[r], acc[i][m][r]);
        }
      }
    }
  };
#pragma unroll
  for (int d = 0; d < DEPTH - 1; ++d) issue(d, d);
  int slot = 0;
  for (int s = 0; s < steps; ++s) {
    __builtin_amdgcn_s_waitcnt(waitcnt_imm((DEPTH - 2) * R::LOADS, 15));
    if constexpr (WN > 1) __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    issue(s + DEPTH - 1, slot == 0 ? DEPTH - 1 : slot - 1);
    __builtin_amdgcn_sched_barrier(0);
    step(slot);
    __builtin_amdgcn_sched_barrier(0);
    slot = slot == DEPTH - 1 ? 0 : slot + 1;
  }
  __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
  __syncthreads();
  f32x4 *s_sum = reinterpret_cast<f32x4 *>(s_ring);
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int m = 0; m < MT; ++m) s_sum[((wave * NT + i) * MT + m) * kWave + lane] = acc[i][m];
  __syncthreads();
  // an item: four matrix rows of one row of x
  for (int item = tid; item < WN * RT * MT * kWave; item += R::WAVES * kWave) {
    const int at = item % kWave, part = item / kWave;
    const int m = part % MT, i = part / MT % RT, n = part / MT / RT;
    auto joined = [&](int tile) {
      const int from = ((n * NT + tile) * MT + m) * kWave + at;
      f32x4 v = s_sum[from];
#pragma unroll
      for (int k = 1; k < WK; ++k) {
        const f32x4 u = s_sum[k * WN * NT * MT * kWave + from];
        v += u;
      }
      return v;
    };
    f32x4 v = joined(i);
    if constexpr (SWIGLU) {
      const f32x4 u = joined(i + RT);
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = v[r] / (1.0f + __expf(-v[r])) * u[r];
    }
    const int row = m0 + 16 * m + (at & 15);
    const int tile = (static_cast<int>(blockIdx.x) * WN + n) * RT + i;
    if (row < a.m && tile <= last_tile) w4_store(a, v, row, 16 * tile + 4 * (at >> 4));
  }
}

template <bool SWIGLU, int NT, int MT, int WN, int WK, int D>
static int launch_w4_ring(const W4Args &a, hipStream_t s) {
  constexpr int RT = SWIGLU ? NT / 2 : NT;
  const int64_t tiles = (a.n + 15) / 16;
  const int64_t x = (tiles + RT * WN - 1) / (RT * WN), y = (a.m + 16 * MT - 1) / (16 * MT);
  if (y > 0xffff || x > 0xffffffffll / (WN * WK * kWave)) return CASCADE_ESHAPE;
  const dim3 grid(static_cast<unsigned>(x), static_cast<unsigned>(y));
  const dim3 block(WN * WK * kWave);
  const int which = (a.group_shift - 5) + (a.w[0].zeros != nullptr ? 3 : 0);
  switch (which) {
    case 0: return launch_kernel(w4_ring_kernel<SWIGLU, false, 4, NT, MT, WN, WK, D>, grid, block, 0, s, a);
    case 1: return launch_kernel(w4_ring_kernel<SWIGLU, false, 2, NT, MT, WN, WK, D>, grid, block, 0, s, a);
    case 2: return launch_kernel(w4_ring_kernel<SWIGLU, false, 1, NT, MT, WN, WK, D>, grid, block, 0, s, a);
    case 3: return launch_kernel(w4_ring_kernel<SWIGLU, true, 4, NT, MT, WN, WK, D>, grid, block, 0, s, a);
    case 4: return launch_kernel(w4_ring_kernel<SWIGLU, true, 2, NT, MT, WN, WK, D>, grid, block, 0, s, a);
    default: return launch_kernel(w4_ring_kernel<SWIGLU, true, 1, NT, MT, WN, WK, D>, grid, block, 0, s, a);
  }
}

template <int OUT>
static int launch_w4(W4Args a, int64_t x_stride, int64_t m, int64_t n, int64_t k,
                     int64_t group, void *stream) {
  if (m <= 0 || n <= 0 || k <= 0) return CASCADE_EINVAL;
  if (k & 7) return CASCADE_EALIGN;
  if ((group != 32 && group != 64 && group != 128) || m > 0x7fffff || n > 0x7fffff ||
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
  const hipStream_t s = static_cast<hipStream_t>(stream);
  constexpr bool kSwiglu = OUT == kW4Swiglu;
  const int64_t row_tiles = (n + 15) / 16 * (kSwiglu ? 2 : 1);
  constexpr int kOne = kSwiglu ? 2 : 1;
  if (m <= 16 && a.tiles * 256 * m <= kW4FewBytes) {
    // workgroups of more row tiles where these still fill the device
    if (row_tiles >= 1536) return launch_w4_few<kSwiglu, 4, 4, 2>(a, s);
    if (kSwiglu || row_tiles >= 512) return launch_w4_few<kSwiglu, 2, 8, 2>(a, s);
    return launch_w4_few<kSwiglu, kOne, 8, 2>(a, s);
  }
  // the most row tiles a workgroup that leave every CU one
  const int64_t blocks = (m + 63) / 64;
  if (m <= 16)
    return row_tiles >= 1280 ? launch_w4_ring<kSwiglu, 2, 1, 4, 2, 4>(a, s)
                             : launch_w4_ring<kSwiglu, kOne, 1, 1, 8, 2>(a, s);
  if (m <= 32)
    return row_tiles >= 1280 ? launch_w4_ring<kSwiglu, 2, 2, 4, 2, 3>(a, s)
                             : launch_w4_ring<kSwiglu, 2, 2, 1, 4, 3>(a, s);
  if (row_tiles * blocks >= 8 * 160) return launch_w4_ring<kSwiglu, 2, 4, 4, 2, 2>(a, s);
  if (row_tiles * blocks >= 4 * 160) return launch_w4_ring<kSwiglu, 2, 4, 2, 2, 3>(a, s);
  return launch_w4_ring<kSwiglu, kOne, 4, 1, 4, 2>(a, s);
}

}  // namespace cascade

using namespace cascade;

extern "C" size_t cascade_linear_w4_workspace_bytes(int64_t, int64_t, int64_t) { return 0; }

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
  return launch_w4<kW4Bf16>(a, x_stride, m, n, k, group, stream);
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
  return launch_w4<kW4F32>(a, x_stride, m, n, k, group, stream);
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
  return launch_w4<kW4Swiglu>(a, x_stride, m, n_half, k, group, stream);
}
