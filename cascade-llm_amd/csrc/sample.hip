// Sampling a token a row from fp32 logits (gfx950): temperature, top-k,
// top-p and min-p, drawn by inversion with a given uniform number.
//
//   w_i = exp((x_i - max x) / T)
//   K   = the top_k largest x (of equal ones the lowest indices)
//   P   = the shortest run of K, largest first, whose mass is >= top_p mass(K)
//   S   = the i of P with w_i >= min_p
//   token = the first i of S, by index, where the mass of S up to i exceeds
//           uniform * mass(S);  logprob = log(w_token / mass(S))
//
// Borders decide which token comes out, so masses are exact sums: w_i is
// computed in fp64 and rounded once to a multiple of 2^-44 (a 64-bit integer;
// the 2^19 logits a row may hold sum to less than 2^64), and integer sums do
// not depend on their order, so neither does the token on how the row was
// cut up.  A token below 2^-45 of the likeliest one is never drawn.
//
// Rows of up to kShortVocab logits take one launch, a workgroup a row
// (sample_short_kernel).  For longer ones four launches cut a row into chunks,
// so that a few rows fill the device:
//   1. sample_max_kernel     a chunk's largest logit
//   2. sample_weigh_kernel   2048 bins of (x_i - max) / T, with the number
//                            and the mass of their tokens (rows with a top-k
//                            or top-p), or the masses of parts (other rows)
//   3. sample_collect_kernel the bins in which K and P end, from those sums;
//                            their tokens go to a list, the mass of the
//                            bins above is kept by parts of 2048.  A K of at most
//                            kShortK tokens is listed whole, which spares
//                            its row the masses.
//   4. sample_draw_kernel    one workgroup a row: sorts the list, finds the
//                            two ends in it, draws a part and then its token
// A row whose list would be longer than kListMax (ends in runs of equal
// logits) is instead cut by the last launch alone, which counts 11 bits of
// the ordered logits at a time over the row.
// One top-k of at most kTopK for all rows takes two launches instead:
//   1. sample_top_kernel     lists a chunk's top_k largest, by bins under the
//                            chunk's own largest
//   2. sample_top_draw_kernel  one workgroup a row: the row's top_k largest
//                            out of these lists, sorted, cut and drawn from
#include <algorithm>

#include "cascade_device.h"
#include "cascade_internal.h"

namespace cascade {

typedef unsigned long long u64;

constexpr int kSampleThreads = 1024;
constexpr int kSampleWaves = kSampleThreads / kWave;
constexpr int kSampleBins = 2048;
constexpr int kWeightBits = 44;
constexpr u64 kWeightOne = u64{1} << kWeightBits;
constexpr int64_t kSampleMaxVocab = int64_t{1} << 19;
constexpr int kListMax = 4096;
constexpr int kShortK = 1024;  // K up to this size is listed whole
constexpr int kChunkThreads = 256;
constexpr int kChunkMin = 2048;
constexpr int kPart = 2048;  // tokens of a chunk whose mass is kept: the draw walks one
constexpr int kChunkMax = 8192;
// Workgroups wanted of a launch: more of them find the row's bins and add to
// them for fewer tokens each (16 rows of 128256 with a top-p: 31.9 us with 256
// wanted, 34.6 with 512, 41.4 with 1024).
constexpr int kChunkWorkgroups = 256;
constexpr int kChunkVecs = kChunkMax / (4 * kChunkThreads);  // of four logits, a thread
constexpr int kChunkParts = kChunkMax / kPart;
// Threads of a draw whose list is short, and the K up to which it is: 512 sort
// as many keys in registers and have half the waves to wait for, more keys go
// through LDS (128256 logits, top-p 0.95, 512 against 1024 threads: K = 113 19.7
// and 21.4 us for a row, 38.3 and 40.2 for 64; K = 480 21.2 and 23.2, 40.8 and
// 42.9; K = 520 33.3 and 24.3, 53.0 and 44.2).  A K of 480 leaves room for ties.
// Rows without a top-k count as short: P ends in a bin or two (64 rows, top-p
// 0.5 45.0 and 46.6, 0.99 52.1 and 54.2), which hold more than 512 keys only
// where that many logits nearly equal each other (700 of them 56.1 and 47.4).
constexpr int kFewThreads = 512;
constexpr int64_t kFewK = 480;
constexpr int kShortVecs = 4;
constexpr int64_t kShortVocab = int64_t{4} * kSampleThreads * kShortVecs;
// One K up to this for all rows takes two launches (128256 logits, top-p 0.95,
// K = 40: 1 row 12.1 us against 18.9, 64 rows 17.5 against 36.3; K = 100: 16.5
// against 19.8 and 21.3 against 39.3).  Past it the draw holds the keys of many
// lists no longer (K = 128: 1 row 23.9 against 19.8).
constexpr int kTopK = 112;
constexpr int kTopCap = 4 * kTopK;  // keys of a chunk's list
constexpr int64_t kSliceRows = 256;  // rows of a launch (the workspace holds these)
// Log2 weights are held in steps of 1/32 (the table of fixed_weight); the bins
// hold the 45 units in which a weight is not 0.
constexpr int kTable = 32;
constexpr double kLeast = -60.0 * kTable;
constexpr double kBinsPerStep = kSampleBins / (45.0 * kTable);

// Four logits behind a pointer aligned to four bytes (rows of odd length);
// one 16-byte load all the same.
typedef float f32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));

struct SampleArgs {
  const float *logits;
  int64_t row_stride;
  int32_t vocab;
  const float *uniform;
  const float *temperature;  // per row, or null: temperature_value
  double temperature_value;
  const int32_t *top_k;
  int64_t top_k_value;
  const float *top_p;
  double top_p_value;
  const float *min_p;
  double min_p_value;
  int64_t *ids;
  float *logprobs;  // nullable
  // the row's cut into chunks, and the workspace (row r's part first)
  int32_t chunk;
  int32_t chunks;
  float *chunk_max;  // [rows][chunks]: the largest logit, NaN if there is one
  int32_t parts;    // of a row: ceil(vocab / kPart)
  u64 *part_mass;   // [rows][parts]
  u64 *bin_mass;    // [rows][kSampleBins]
  uint32_t *bin_count;
  struct RowEnds *ends;  // [rows]
  u64 *list;             // [rows][kListMax] keys, or [rows][chunks][kTopCap]
  uint32_t *list_count;  // [rows]
};

// Where K and P end in the bins (bin 0 holds the largest logits).
struct RowEnds {
  u64 above_k;   // mass of the bins above K's last one
  u64 above_p;   // and above P's first candidate
  u64 total;     // mass of the row
  uint32_t need_k;  // tokens that K takes of its last bin
  uint32_t before;  // list entries in bins above K's last one
  int32_t first;    // bins first .. last_p, and last_k, are listed
  int32_t last_p;   // -1: no top-p
  int32_t last_k;   // -1: no top-k
};

struct RowSettings {
  bool greedy;
  bool use_k;     // there is a top-k
  bool use_p;     // the bins' masses are needed: a top-p, and no short K
  double scale;   // 32 log2(e) / T
  int64_t top_k;  // <= 0: off
  double top_p;   // >= 1: off
  u64 min_w;      // smallest weight kept
  int min_bin;    // from this bin on no token has it
};

__device__ __forceinline__ RowSettings row_settings(const SampleArgs &a, int row) {
  RowSettings r;
  const double t = a.temperature != nullptr ? static_cast<double>(a.temperature[row])
                                            : a.temperature_value;
  r.greedy = !(t > 0.0);
  r.scale = fmin(kTable * 1.4426950408889634 / t, 1e300);  // 0 times it stays 0
  r.top_k = a.top_k != nullptr ? static_cast<int64_t>(a.top_k[row]) : a.top_k_value;
  r.top_p = a.top_p != nullptr ? static_cast<double>(a.top_p[row]) : a.top_p_value;
  const double p = a.min_p != nullptr ? static_cast<double>(a.min_p[row]) : a.min_p_value;
  r.min_w = p > 0.0 ? static_cast<u64>(ceil(fmin(p, 1.0) * static_cast<double>(kWeightOne)))
                    : u64{0};
  if (p > 1.0) r.top_k = 1;  // none reaches it: the likeliest alone stays
  // (a bin of margin for log2f)
  r.min_bin = p > 0.0 ? static_cast<int>(fminf(-log2f(static_cast<float>(fmin(p, 1.0))) *
                                                   static_cast<float>(kTable * kBinsPerStep) +
                                               2.0f,
                                           static_cast<float>(kSampleBins)))
                      : kSampleBins;
  r.use_k = r.top_k > 0;
  r.use_p = r.top_p < 1.0 && !(r.use_k && r.top_k <= kShortK);
  return r;
}

// A row's largest logit and the scale of the differences to it.
struct RowScale {
  double mx;
  double scale;
  const double *table;  // in LDS: 2^(44 + j / 32), j < 32
};

// An infinite logit counts as 1e300: equal to another infinite one, and all
// above the finite ones.
__device__ __forceinline__ double logit64(float x) {
  return fmin(static_cast<double>(x), 1e300);
}

__device__ __forceinline__ RowScale row_scale(float mx, const RowSettings &set,
                                              const double *table) {
  return RowScale{logit64(mx), set.scale, table};
}

// 32 times the log2 weight of logit x: 0 for the largest, never below kLeast
// (-inf, and 0 times an infinity, end there).  A larger logit gets no less.
__device__ __forceinline__ double log_weight(float x, const RowScale &r) {
  return fmax((logit64(x) - r.mx) * r.scale, kLeast);
}

// Bin of a log weight: bin 0 holds the largest, kSampleBins and above have no
// weight.
__device__ __forceinline__ int weight_bin(double t) {
  return static_cast<int>(t * -kBinsPerStep);
}

// 2^(44 + t / 32) rounded to an integer (0 from t / 32 = -45 on).  With n the
// integer next to t and f = t - n, the weight is 2^floor(n / 32) times the
// table's 2^(44 + (n mod 32) / 32) times 2^(f / 32), the Taylor polynomial of
// e^(f ln 2 / 32) to the 5th power, whose remainder is below 3e-15.  Adding
// 1.5 x 2^52 rounds t and leaves n in the low bits; adding 2^52 does so with
// the weight.
__device__ __forceinline__ u64 fixed_weight(double t, const double *table) {
  constexpr double kLn = 0.6931471805599453 / kTable;
  const double shifted = t + 6755399441055744.0;
  const int n = static_cast<int>(__double_as_longlong(shifted));
  const double f = t - (shifted - 6755399441055744.0);
  double p = kLn * kLn * kLn * kLn * kLn / 120.0;
  p = fma(p, f, kLn * kLn * kLn * kLn / 24.0);
  p = fma(p, f, kLn * kLn * kLn / 6.0);
  p = fma(p, f, kLn * kLn / 2.0);
  p = fma(p, f, kLn);
  p = fma(p, f, 1.0);
  const double v = ldexp(p * table[n & (kTable - 1)], n >> 5) + 4503599627370496.0;
  return static_cast<u64>(__double_as_longlong(v)) & 0xfffffffffffffull;
}

__device__ __forceinline__ u64 fixed_weight(float x, const RowScale &r) {
  return fixed_weight(log_weight(x, r), r.table);
}

// The table: 2^(j / 32) by the Taylor polynomial of e^(z ln 2), |z| <= 1/2, to
// the 12th power (remainder below 2e-16).  A barrier has to follow.
__device__ __forceinline__ void fill_table(double *table) {
  const int j = threadIdx.x;
  if (j >= kTable) return;
  const int whole = j > kTable / 2 ? 1 : 0;
  const double z = (static_cast<double>(j) / kTable - whole) * 0.6931471805599453;
  double p = 1.0;
#pragma unroll
  for (int k = 12; k >= 1; --k) p = fma(p * z, 1.0 / k, 1.0);
  table[j] = ldexp(p, whole + kWeightBits);
}

// Inclusive prefix sum over the workgroup in thread order, and its total.
// Two barriers; `lds` may be reused after the second.
template <int WAVES = kSampleWaves>
__device__ __forceinline__ u64 block_prefix(u64 v, u64 *lds, u64 *total) {
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = threadIdx.x / kWave;
  v = wave_prefix(v);
  if (lane == kWave - 1) lds[wave] = v;
  __syncthreads();
  u64 before = 0, all = 0;
#pragma unroll 4
  for (int w = 0; w < WAVES; ++w) {
    const u64 s = lds[w];
    if (w < wave) before += s;
    all += s;
  }
  __syncthreads();
  *total = all;
  return before + v;
}

// A cut of the row in the order "larger first, of equal ones the lower
// index first": element i with ordered bits o is kept where o > value, or
// o == value and i <= index.
struct Cut {
  uint32_t value;
  uint32_t index;
};

__device__ __forceinline__ bool keeps(const Cut &c, uint32_t o, uint32_t i) {
  return o > c.value || (o == c.value && i <= c.index);
}

struct SampleShared {
  uint32_t count[kSampleBins];
  u64 mass[kSampleBins];
  u64 scan[kSampleWaves];
  u64 found[4];
};

// The cut that keeps the fewest elements of the row, among those of `in`
// with a weight, so that their number (BY_MASS: mass) reaches `need` >= 1;
// *mass_kept is then the mass kept.  All elements together have to reach it.
template <int THREADS, bool BY_MASS>
__device__ Cut find_cut(const float *x, int n, const RowScale &r, Cut in, u64 need,
                        SampleShared &sh, u64 *mass_kept) {
  const int tid = threadIdx.x;
  uint32_t prefix = 0, known = 0;  // the value's bits found so far
  u64 above_count = 0, above_mass = 0;
  u64 equal = 0, equal_mass = 0;
#pragma unroll 1
  for (int round = 0; round < 3; ++round) {
    const int shift = round == 0 ? 21 : round == 1 ? 10 : 0;
    const uint32_t bins = round == 2 ? 1024u : 2048u;
    for (int b = tid; b < kSampleBins; b += THREADS) {
      sh.count[b] = 0;
      sh.mass[b] = 0;
    }
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < n; i += THREADS) {
      const float v = x[i];
      const uint32_t o = ordered_bits(v);
      if ((o & known) != prefix || !keeps(in, o, i)) continue;
      const u64 w = fixed_weight(v, r);
      if (w == 0) continue;
      const uint32_t b = (o >> shift) & (bins - 1);
      atomicAdd(&sh.count[b], 1u);
      atomicAdd(&sh.mass[b], w);
    }
    __syncthreads();
    // thread t scans kPer bins from 2047 - kPer t on, from the top down
    constexpr int kPer = kSampleBins / THREADS;
    const int top = kSampleBins - 1 - kPer * tid;
    u64 c_sum = 0, m_sum = 0, total;
#pragma unroll 1
    for (int j = 0; j < kPer; ++j) {
      c_sum += sh.count[top - j];
      m_sum += sh.mass[top - j];
    }
    u64 c_at = block_prefix<THREADS / kWave>(c_sum, sh.scan, &total) - c_sum + above_count;
    u64 m_at = block_prefix<THREADS / kWave>(m_sum, sh.scan, &total) - m_sum + above_mass;
#pragma unroll 1
    for (int j = 0; j < kPer; ++j) {
      const u64 c = sh.count[top - j], m = sh.mass[top - j];
      const u64 start = BY_MASS ? m_at : c_at, end = start + (BY_MASS ? m : c);
      if (start < need && need <= end) {
        sh.found[0] = top - j;
        sh.found[1] = c_at;
        sh.found[2] = m_at;
      }
      c_at += c;
      m_at += m;
    }
    __syncthreads();
    const uint32_t bin = static_cast<uint32_t>(sh.found[0]);
    above_count = sh.found[1];
    above_mass = sh.found[2];
    equal = sh.count[bin];
    equal_mass = sh.mass[bin];
    prefix |= bin << shift;
    known |= (bins - 1) << shift;
    __syncthreads();
  }
  // all `equal` elements left have the value `prefix` and one weight
  const u64 w = equal_mass / equal;
  const u64 take = BY_MASS ? (need - above_mass + w - 1) / w : need - above_count;
  *mass_kept = above_mass + take * w;
  Cut cut{prefix, prefix == in.value ? in.index : 0xffffffffu};
  if (take < equal) {
    // the index of the take-th of them (`in` leaves out later ones at most)
    u64 seen = 0;
#pragma unroll 1
    for (int base = 0; base < n; base += THREADS) {
      const int i = base + tid;
      const bool hit = i < n && ordered_bits(x[i]) == prefix;
      u64 total;
      const u64 at = seen + block_prefix<THREADS / kWave>(hit ? 1 : 0, sh.scan, &total);
      if (hit && at == take) sh.found[0] = i;
      seen += total;
      if (seen >= take) break;  // uniform
    }
    __syncthreads();
    cut.index = static_cast<uint32_t>(sh.found[0]);
    __syncthreads();
  }
  return cut;
}

// Maximum that a NaN wins.
__device__ __forceinline__ float nan_max(float a, float b) { return max_f32(a, b); }

__device__ __forceinline__ float wave_nan_max(float v) {
  v = nan_max(v, dpp_float<0xB1>(v));
  v = nan_max(v, dpp_float<0x4E>(v));
  v = nan_max(v, dpp_float<0x141>(v));
  v = nan_max(v, dpp_float<0x140>(v));
  return xor32_max(xor16_max(v));
}

// Largest logit of a row from its chunks'.  All threads return it.
__device__ __forceinline__ float row_max(const SampleArgs &a, int row) {
  float best = -INFINITY;
  for (int c = threadIdx.x & (kWave - 1); c < a.chunks; c += kWave)
    best = nan_max(best, a.chunk_max[static_cast<int64_t>(row) * a.chunks + c]);
  return wave_nan_max(best);
}

// A row with a NaN or without any number yields no token.
__device__ __forceinline__ bool no_token(float mx) { return mx != mx || mx == -INFINITY; }

// Logits begin .. end - 1 of a row in the registers of its workgroup: VECS
// vectors of four neighbours a thread, and the last three at most one by one.
// All are loaded before the first is used, ahead of whatever the kernel has
// to find out.
template <int THREADS, int VECS>
struct Chunk {
  f32x4_at4 v[VECS];
  float rest;
  int begin, whole, end;

  __device__ __forceinline__ Chunk(const float *x, int first, int last) {
    begin = first;
    end = last;
    whole = begin + (end - begin) / 4 * 4;
    if (whole > begin) {  // uniform
#pragma unroll
      for (int j = 0; j < VECS; ++j)
        if (begin + 4 * THREADS * j < whole)  // uniform
          v[j] = *reinterpret_cast<const f32x4_at4 *>(x + min(at(j), whole - 4));
    }
    rest = x[min(whole + static_cast<int>(threadIdx.x), end - 1)];
  }

  // first index of this thread's vector j
  __device__ __forceinline__ int at(int j) const {
    return begin + 4 * (THREADS * j + static_cast<int>(threadIdx.x));
  }

  // f(logits, index of the first, part) for every four neighbours, part being
  // the kPart tokens of the chunk that they belong to: f
  // does the arithmetic of all four before it branches on any, so that their
  // chains of fp64 instructions overlap.  The rest comes as one logit with
  // three -inf.
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll
    for (int j = 0; j < VECS; ++j)
      if (at(j) < whole) f(v[j], at(j), 4 * THREADS * j / kPart);
    const int i = whole + static_cast<int>(threadIdx.x);
    if (i < end) f(f32x4_at4{rest, -INFINITY, -INFINITY, -INFINITY}, i, (i - begin) / kPart);
  }
};

// Bins of four logits.
__device__ __forceinline__ void bins_of(const f32x4_at4 &v, const RowScale &r, double (&t)[4],
                                        int (&b)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    t[i] = log_weight(v[i], r);
    b[i] = weight_bin(t[i]);
  }
}

__device__ __forceinline__ Chunk<kChunkThreads, kChunkVecs> row_chunk(const SampleArgs &a,
                                                                      int row, int chunk) {
  const int begin = chunk * a.chunk;
  return Chunk<kChunkThreads, kChunkVecs>(a.logits + row * a.row_stride, begin,
                                          min(begin + a.chunk, a.vocab));
}

// A workgroup a chunk.  Bound by its reads: 64 rows of 128256 6.5 us (5.0
// TB/s), one row 2.7 us.
__global__ __launch_bounds__(kChunkThreads) void sample_max_kernel(SampleArgs a) {
  __shared__ float s_max[kChunkThreads / kWave];
  const int chunk = static_cast<int>(blockIdx.x) % a.chunks;
  const int row = static_cast<int>(blockIdx.x) / a.chunks;
  const int tid = threadIdx.x;
  const auto logits = row_chunk(a, row, chunk);
  // the bins and the list of the row start empty
  u64 *mass = a.bin_mass + static_cast<int64_t>(row) * kSampleBins;
  uint32_t *count = a.bin_count + static_cast<int64_t>(row) * kSampleBins;
  for (int i = chunk * kChunkThreads + tid; i < kSampleBins; i += a.chunks * kChunkThreads) {
    mass[i] = 0;
    count[i] = 0;
  }
  if (chunk == 0 && tid == 0) a.list_count[row] = 0;
  float best = -INFINITY;
  logits.each([&](const f32x4_at4 &v, int, int) {
    best = nan_max(nan_max(best, nan_max(v[0], v[1])), nan_max(v[2], v[3]));
  });
  best = wave_nan_max(best);
  if ((tid & (kWave - 1)) == 0) s_max[tid / kWave] = best;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < kChunkThreads / kWave; ++w) best = nan_max(best, s_max[w]);
    a.chunk_max[static_cast<int64_t>(row) * a.chunks + chunk] = best;
  }
}

// Writes the masses of the chunk's parts from its threads' shares of them.
__device__ __forceinline__ void store_parts(const SampleArgs &a, int row, int chunk,
                                            const u64 (&sum)[kChunkParts], u64 *lds) {
  constexpr int kWaves = kChunkThreads / kWave;
  const int tid = threadIdx.x;
#pragma unroll
  for (int k = 0; k < kChunkParts; ++k) {
    const u64 wave = wave_prefix(sum[k]);
    if ((tid & (kWave - 1)) == kWave - 1) lds[k * kWaves + tid / kWave] = wave;
  }
  __syncthreads();
  const int part = chunk * (a.chunk / kPart) + tid;
  if (tid < a.chunk / kPart && part < a.parts) {
    u64 total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += lds[tid * kWaves + w];
    a.part_mass[static_cast<int64_t>(row) * a.parts + part] = total;
  }
}

// Adds four logits to their bins: their number, and their mass.
__device__ __forceinline__ void add_to_bins(const f32x4_at4 &v, const RowScale &r, bool use_k,
                                            bool use_p, uint32_t *count, u64 *mass) {
  double t[4];
  int b[4];
  u64 w[4];
  bins_of(v, r, t, b);
  if (use_p) {  // uniform
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = fixed_weight(t[i], r.table);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (b[i] < kSampleBins) {
      if (use_k) atomicAdd(&count[b[i]], 1u);
      if (use_p) atomicAdd(&mass[b[i]], w[i]);
    }
}

// A workgroup a chunk, its bins in LDS; those in use are added to the row's.
// Bound by the fp64 arithmetic and the LDS atomics of a logit: 64 rows of
// 128256 of mixed settings 13.9 us; one row 4.8 us, the trip to memory for the
// maxima in front of it.
__global__ __launch_bounds__(kChunkThreads) void sample_weigh_kernel(SampleArgs a) {
  __shared__ u64 s_mass[kSampleBins];
  __shared__ uint32_t s_count[kSampleBins];
  __shared__ double s_table[kTable];
  const int chunk = static_cast<int>(blockIdx.x) % a.chunks;
  const int row = static_cast<int>(blockIdx.x) / a.chunks;
  const int tid = threadIdx.x;
  const auto logits = row_chunk(a, row, chunk);
  fill_table(s_table);
  const RowSettings set = row_settings(a, row);
  const float mx = row_max(a, row);
  if (set.greedy || no_token(mx)) return;
  const RowScale r = row_scale(mx, set, s_table);
  if (!set.use_k && !set.use_p) {
    __syncthreads();
    u64 sum[kChunkParts] = {};
    logits.each([&](const f32x4_at4 &v, int, int part) {
      double t[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = log_weight(v[i], r);
      if (set.min_w != 0 &&
          weight_bin(fmax(fmax(t[0], t[1]), fmax(t[2], t[3]))) >= set.min_bin)
        return;
      u64 four = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u64 w = fixed_weight(t[i], s_table);
        four += w >= set.min_w ? w : 0;
      }
#pragma unroll
      for (int k = 0; k < kChunkParts; ++k) sum[k] += part == k ? four : 0;
    });
    store_parts(a, row, chunk, sum, s_mass);
    return;
  }
  // top-k needs the numbers, top-p the masses
  const bool use_k = set.use_k, use_p = set.use_p;
  for (int i = tid; i < kSampleBins; i += kChunkThreads) {
    if (use_p) s_mass[i] = 0;
    if (use_k) s_count[i] = 0;
  }
  __syncthreads();
  logits.each([&](const f32x4_at4 &v, int, int) {
    add_to_bins(v, r, use_k, use_p, s_count, s_mass);
  });
  __syncthreads();
  u64 *mass = a.bin_mass + static_cast<int64_t>(row) * kSampleBins;
  uint32_t *count = a.bin_count + static_cast<int64_t>(row) * kSampleBins;
  for (int i = tid; i < kSampleBins; i += kChunkThreads) {
    if (use_k && s_count[i] != 0) atomicAdd(&count[i], s_count[i]);
    if (use_p && s_mass[i] != 0) atomicAdd(&mass[i], s_mass[i]);
  }
}

// The smallest whole mass that reaches top_p of `mass`, in [1, mass].
__device__ __forceinline__ u64 top_p_mass(double top_p, u64 mass) {
  const double need = ceil(top_p * static_cast<double>(mass));
  const u64 n = need >= 1.0 ? static_cast<u64>(need) : 1;
  return n < mass ? n : mass;
}

// A thread's share of the bins, neighbours: what the row's settings need.
template <int THREADS>
struct BinShare {
  static constexpr int kPer = kSampleBins / THREADS;
  u64 mass[kPer];
  uint32_t count[kPer];

  __device__ __forceinline__ BinShare(const u64 *bin_mass, const uint32_t *bin_count,
                                      const RowSettings &set) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      mass[i] = 0;
      count[i] = 0;
    }
    if (set.use_p) {  // uniform
#pragma unroll
      for (int i = 0; i < kPer; ++i) mass[i] = bin_mass[threadIdx.x * kPer + i];
    }
    if (set.use_k) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) count[i] = bin_count[threadIdx.x * kPer + i];
    }
  }
};

// The ends of K and P in the row's bins, by a workgroup of THREADS.  K's last
// bin is exact; P's is known up to what K takes of its last bin, so every bin
// in which P could end is listed.  A short K that a top-p follows is listed from
// bin 0 on.
template <int THREADS>
__device__ RowEnds find_ends(const BinShare<THREADS> &bins, const RowSettings &set) {
  constexpr int kPer = BinShare<THREADS>::kPer;
  constexpr int kWaves = THREADS / kWave;
  __shared__ u64 s_scan[kWaves];
  __shared__ RowEnds s_ends;
  __shared__ u64 s_most;           // the most that K can weigh
  __shared__ uint32_t s_above[2];  // tokens above the first listed bin, above K's last
  __shared__ uint32_t s_upto;      // tokens up to P's last candidate
  const int tid = threadIdx.x;
  const bool short_k = set.use_k && set.top_k <= kShortK;
  u64 msum = 0, nsum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    msum += bins.mass[i];
    nsum += bins.count[i];
  }
  u64 total = 0, live = 0, m_at = 0, n_at = 0;
  if (set.use_p) m_at = block_prefix<kWaves>(msum, s_scan, &total) - msum;
  if (set.use_k) n_at = block_prefix<kWaves>(nsum, s_scan, &live) - nsum;
  if (tid == 0) {
    s_ends = RowEnds{0, 0, total, 0, 0, 0, -1, -1};
    s_above[0] = s_above[1] = s_upto = 0;
  }
  __syncthreads();
  const bool use_k = set.use_k && (short_k || static_cast<u64>(set.top_k) < live);
  u64 k_least = total, k_most = total;
  if (use_k) {
    const u64 need = min(static_cast<u64>(set.top_k), live);
    u64 ma = m_at, na = n_at;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (na < need && need <= na + bins.count[i]) {
        s_ends.above_k = ma;
        s_ends.need_k = static_cast<uint32_t>(need - na);
        s_ends.last_k = tid * kPer + i;
        s_ends.first = tid * kPer + i;
        s_above[1] = static_cast<uint32_t>(na);
        s_most = ma + bins.mass[i];
      }
      ma += bins.mass[i];
      na += bins.count[i];
    }
    __syncthreads();
    k_most = s_most;
    // a token at least, if it has a weight
    k_least = min(s_ends.above_k + 1, k_most);
  }
  __syncthreads();
  if (set.use_p) {
    const u64 least = top_p_mass(set.top_p, k_least), most = top_p_mass(set.top_p, k_most);
    u64 ma = m_at, na = n_at;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (ma < least && least <= ma + bins.mass[i]) {
        s_ends.first = tid * kPer + i;
        s_ends.above_p = ma;
        s_above[0] = static_cast<uint32_t>(na);
      }
      if (ma < most && most <= ma + bins.mass[i]) {
        s_ends.last_p = tid * kPer + i;
        s_upto = static_cast<uint32_t>(na + bins.count[i]);
      }
      ma += bins.mass[i];
      na += bins.count[i];
    }
  }
  __syncthreads();
  RowEnds e = s_ends;
  if (short_k && set.top_p < 1.0) {
    e.first = 0;
    e.before = s_above[1];
    e.last_p = e.last_k;
  } else if (set.use_p && use_k) {
    if (e.last_p >= e.last_k) {  // one run of bins: first .. last_k
      e.before = s_above[1] - s_above[0];
      e.last_p = e.last_k;
    } else {
      e.before = s_upto - s_above[0];
    }
  }
  return e;
}

// Puts those of four logits that are in a listed bin (from `first` on) on a
// list of kListMax; *count counts them all.
__device__ __forceinline__ void list_of(const f32x4_at4 &v, int at, const int (&b)[4], int first,
                                        const RowEnds &e, u64 *list, uint32_t *count) {
  bool in[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) in[i] = b[i] >= first && (b[i] <= e.last_p || b[i] == e.last_k);
  if (!(in[0] || in[1] || in[2] || in[3])) return;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (in[i]) {
      const uint32_t n = atomicAdd(count, 1u);
      if (n < kListMax) list[n] = topk_key(v[i], static_cast<uint32_t>(at + i));
    }
}

// A workgroup a chunk; each finds the row's ends in the bins for itself, which
// costs less than a launch between.  64 rows of 128256 of mixed settings 14.6
// us, the masses above the ends as in the launch before; one row 5.5 us.
__global__ __launch_bounds__(kChunkThreads) void sample_collect_kernel(SampleArgs a) {
  __shared__ u64 s_keys[kListMax];
  __shared__ uint32_t s_count, s_at;
  __shared__ double s_table[kTable];
  __shared__ u64 s_sum[kChunkParts * (kChunkThreads / kWave)];
  const int chunk = static_cast<int>(blockIdx.x) % a.chunks;
  const int row = static_cast<int>(blockIdx.x) / a.chunks;
  const int tid = threadIdx.x;
  const auto logits = row_chunk(a, row, chunk);
  const RowSettings set = row_settings(a, row);
  if (set.greedy || (!set.use_k && !set.use_p)) return;
  const BinShare<kChunkThreads> bins(a.bin_mass + static_cast<int64_t>(row) * kSampleBins,
                                     a.bin_count + static_cast<int64_t>(row) * kSampleBins,
                                     set);
  fill_table(s_table);
  const float mx = row_max(a, row);
  if (no_token(mx)) return;
  const RowEnds e = find_ends(bins, set);
  if (chunk == 0 && tid == 0) a.ends[row] = e;
  // without a cut inside the bins (top_k of all tokens) nothing is listed
  const int first = e.last_p < 0 && e.last_k < 0 ? kSampleBins : e.first;
  const RowScale r = row_scale(mx, set, s_table);
  u64 sum[kChunkParts] = {};  // of the bins above the listed ones
  if (tid == 0) s_count = 0;
  __syncthreads();
  logits.each([&](const f32x4_at4 &v, int at, int part) {
    double t[4];
    int b[4];
    bins_of(v, r, t, b);
    const int least = min(min(b[0], b[1]), min(b[2], b[3]));
    if (least < min(first, set.min_bin)) {
      u64 w[4], four = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = fixed_weight(t[i], s_table);
#pragma unroll
      for (int i = 0; i < 4; ++i) four += b[i] < first && w[i] >= set.min_w ? w[i] : 0;
#pragma unroll
      for (int k = 0; k < kChunkParts; ++k) sum[k] += part == k ? four : 0;
    }
    list_of(v, at, b, first, e, s_keys, &s_count);
  });
  store_parts(a, row, chunk, sum, s_sum);  // (a barrier: the list is whole)
  const uint32_t mine = s_count;
  if (mine != 0) {
    // the list's order does not matter: the draw sorts it.  A row of more
    // than kListMax entries (list_count tells) gets no whole list.
    if (tid == 0) s_at = atomicAdd(&a.list_count[row], mine);
    __syncthreads();
    const uint32_t at = s_at;
    u64 *list = a.list + static_cast<int64_t>(row) * kListMax;
    if (mine <= kListMax && at <= kListMax - mine)
      for (uint32_t i = tid; i < mine; i += kChunkThreads) list[at + i] = s_keys[i];
  }
}

struct DrawShared {
  union {
    SampleShared row;         // the counted cut of a whole row, and bins
    u64 keys[kListMax];       // the list
  };
  u64 mass[kSampleThreads];   // of the chunks
  u64 scan[kSampleWaves];
  u64 found[2];
  double table[kTable];
  int first[2];
};

// Sorts keys[0..n) in descending order (n a power of two, at least 2).
template <int THREADS>
__device__ __forceinline__ void sort_keys(u64 *keys, int n) {
  for (int run = 2; run <= n; run *= 2)
    for (int gap = run / 2; gap >= 1; gap /= 2) {
      __syncthreads();
      for (int i = threadIdx.x; i < n / 2; i += THREADS) {
        const int lo = 2 * i - (i & (gap - 1));
        const int hi = lo + gap;
        const u64 x = keys[lo], y = keys[hi];
        if ((x < y) == ((lo & run) == 0)) {
          keys[lo] = y;
          keys[hi] = x;
        }
      }
    }
  __syncthreads();
}

// The same for up to THREADS keys, one a thread (v; 0 past the list): runs of 64
// are sorted and merged in a wave's registers, and only the steps over a
// longer gap go through LDS.  The sorted keys end up in keys[0..THREADS).
template <int THREADS>
__device__ __forceinline__ u64 sort_block(u64 v, int n, u64 *keys) {
  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int runs = (n + kWave - 1) / kWave;  // uniform
  if (tid / kWave < runs) {
    v = merge_run<2>(v, lane, lane & 2);
    v = merge_run<4>(v, lane, lane & 4);
    v = merge_run<8>(v, lane, lane & 8);
    v = merge_run<16>(v, lane, lane & 16);
    v = merge_run<32>(v, lane, lane & 32);
    v = merge_run<64>(v, lane, tid & 64);
  }
  int side = 1;  // the half of `keys` that the next step writes
  for (int run = 2 * kWave; run < 2 * kWave * runs; run *= 2) {
    const bool down = (tid & run) != 0;
    for (int gap = run / 2; gap >= kWave; gap /= 2) {
      u64 *half = keys + side * THREADS;
      half[tid] = v;
      __syncthreads();
      const u64 other = half[tid ^ gap];
      v = (v > other) == (((tid & gap) == 0) != down) ? v : other;
      side ^= 1;
    }
    v = merge_run<64>(v, lane, down);
  }
  __syncthreads();
  keys[tid] = v;
  __syncthreads();
  return v;
}

// The key of the last token of the row's P (or K) in its list of n keys, of
// which this thread has key tid (PER = 1).  PER: keys a thread holds.
// Positions of the sorted list (in sh.keys): K's last bin starts at e.before.
template <int THREADS, int PER>
__device__ u64 list_cut(const u64 *list, int n, u64 mine, const RowEnds &e,
                        const RowSettings &set, const RowScale &r, DrawShared &sh) {
  const int tid = threadIdx.x;
  if constexpr (PER == 1) {
    sort_block<THREADS>(mine, n, sh.keys);
  } else {
    int padded = 2;
    while (padded < n) padded *= 2;
    // (the list may be in sh.keys already)
    for (int i = tid; i < padded; i += THREADS) sh.keys[i] = i < n ? list[i] : 0;
    sort_keys<THREADS>(sh.keys, padded);
  }
  const int last_k = static_cast<int>(e.before + e.need_k) - 1;
  if (!(set.top_p < 1.0)) return sh.keys[last_k];
  // prefix sums of the weights, PER neighbours a thread
  u64 w[PER], sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = PER * tid + i;
    w[i] = at < n ? fixed_weight(key_value(sh.keys[at]), r) : 0;
    sum += w[i];
  }
  u64 total;
  const u64 start = block_prefix<THREADS / kWave>(sum, sh.scan, &total) - sum;
  u64 mass_k = e.total;
  if (e.last_k >= 0) {
    // mass of the list before K's last bin, and up to K's last token.  Where
    // the bins have masses the list may lack those between P's last candidate
    // and K's last bin, also if it starts at bin 0: what lies above K's last bin
    // is known from the bins.  Without masses (a short K) the list has all.
    u64 upto = start;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = PER * tid + i;
      if (at == static_cast<int>(e.before)) sh.found[0] = upto;
      upto += w[i];
      if (at == last_k) sh.found[1] = upto;
    }
    __syncthreads();
    mass_k = set.use_p ? e.above_k + (sh.found[1] - sh.found[0]) : sh.found[1];
    __syncthreads();
  }
  const u64 need = top_p_mass(set.top_p, mass_k);
  u64 upto = e.above_p + start;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (upto < need && need <= upto + w[i]) sh.found[0] = PER * tid + i;
    upto += w[i];
  }
  __syncthreads();
  return sh.keys[sh.found[0]];
}

// The cut of a row found over the whole row, as a key.
template <int THREADS>
__device__ u64 counted_cut(const float *x, int n, const RowScale &r, const RowSettings &set,
                           u64 mass_all, u64 live, SampleShared &sh) {
  Cut cut{0u, 0xffffffffu};
  if (set.top_k > 0 && static_cast<u64>(set.top_k) < live)
    cut = find_cut<THREADS, false>(x, n, r, cut, static_cast<u64>(set.top_k), sh, &mass_all);
  if (set.top_p < 1.0)
    cut = find_cut<THREADS, true>(x, n, r, cut, top_p_mass(set.top_p, mass_all), sh,
                         &mass_all);
  return (static_cast<u64>(cut.value) << 32) | (0xffffffffu - cut.index);
}

// The cut of a row whose list would be too long, and the masses of the row's
// parts under it in sh.mass.
template <int THREADS>
__device__ __forceinline__ u64 counted_row(const SampleArgs &a, const float *x,
                                           const RowScale &r, const RowSettings &set,
                                           DrawShared &sh) {
  const int tid = threadIdx.x;
  u64 live = 0, sum = 0;
#pragma unroll 1
  for (int i = tid; i < a.vocab; i += THREADS) {
    const u64 w = fixed_weight(x[i], r);
    live += w != 0 ? 1 : 0;
    sum += w;
  }
  u64 live_all, mass_all;
  block_prefix<THREADS / kWave>(live, sh.scan, &live_all);
  block_prefix<THREADS / kWave>(sum, sh.scan, &mass_all);
  const u64 cut = counted_cut<THREADS>(x, a.vocab, r, set, mass_all, live_all, sh.row);
  // a wave a part
#pragma unroll 1
  for (int c = tid / kWave; c < a.parts; c += (THREADS / kWave)) {
    const int end = min((c + 1) * kPart, a.vocab);
    u64 part = 0;
#pragma unroll 1
    for (int i = c * kPart + (tid & (kWave - 1)); i < end; i += kWave) {
      const u64 w = fixed_weight(x[i], r);
      if (w >= set.min_w && topk_key(x[i], static_cast<uint32_t>(i)) >= cut) part += w;
    }
    part = wave_prefix(part);
    if ((tid & (kWave - 1)) == kWave - 1) sh.mass[c] = part;
  }
  __syncthreads();
  return cut;
}

// The mass that `uniform` points at, of `total`.
__device__ __forceinline__ u64 target_of(float uniform, u64 total) {
  double u = static_cast<double>(uniform);
  u = u > 0.0 ? u : 0.0;  // NaN too
  const double t = u * static_cast<double>(total);
  const u64 target = t < static_cast<double>(total) ? static_cast<u64>(t) : total - 1;
  return target < total ? target : total - 1;
}

// Writes a row's token, of logit x.  Its log-probability is the log weight
// itself and not the logarithm of the rounded weight, of which an unlikely
// token's has few bits left; the sum's rounding is below vocab 2^-45.
__device__ __forceinline__ void store_token(const SampleArgs &a, int row, int64_t token, float x,
                                            const RowScale &r, u64 total) {
  constexpr double kLn = 0.6931471805599453;
  a.ids[row] = token;
  if (a.logprobs != nullptr)
    a.logprobs[row] = static_cast<float>(
        log_weight(x, r) * (kLn / kTable) -
        log(static_cast<double>(total) / static_cast<double>(kWeightOne)));
}

__device__ __forceinline__ void store_no_token(const SampleArgs &a, int row) {
  if (threadIdx.x != 0) return;
  a.ids[row] = -1;
  if (a.logprobs != nullptr) a.logprobs[row] = __builtin_nanf("");
}

// The first of the row's largest logits: in the first chunk that has it.
template <int THREADS>
__device__ __forceinline__ void store_largest(const SampleArgs &a, int row, const float *x,
                                              float mx, int *first) {
  const int tid = threadIdx.x;
  const bool has = tid < a.chunks &&
                   a.chunk_max[static_cast<int64_t>(row) * a.chunks + tid] == mx;
  if (tid == 0) first[0] = first[1] = 0x7fffffff;
  __syncthreads();
  if (has) atomicMin(&first[0], tid);
  __syncthreads();
  const int begin = min(first[0], a.chunks - 1) * a.chunk;
  const int end = min(begin + a.chunk, a.vocab);
  for (int i = begin + tid; i < end; i += THREADS)
    if (x[i] == mx) {
      atomicMin(&first[1], i);
      break;
    }
  __syncthreads();
  if (tid == 0) {
    a.ids[row] = first[1];
    if (a.logprobs != nullptr) a.logprobs[row] = 0.0f;
  }
}

// The draw from a row of which thread c has the mass of part c: a part, then
// a token in it.
template <int THREADS>
__device__ __forceinline__ void draw_token(const SampleArgs &a, int row, const float *x,
                                           float uniform, u64 mass, u64 cut, const RowScale &r,
                                           const RowSettings &set, DrawShared &sh) {
  const int tid = threadIdx.x;
  u64 total;
  const u64 upto = block_prefix<THREADS / kWave>(mass, sh.scan, &total);
  u64 target = target_of(uniform, total);
  if (upto - mass <= target && target < upto) {
    sh.found[0] = static_cast<u64>(tid);
    sh.found[1] = target - (upto - mass);
  }
  __syncthreads();
  const int begin = static_cast<int>(min(sh.found[0], static_cast<u64>(a.parts - 1))) * kPart;
  const int end = min(begin + kPart, a.vocab);
  target = sh.found[1];
  // neighbouring tokens to a thread, so that one prefix sum orders them all
  constexpr int kPer = kPart / THREADS;
  const int mine = begin + tid * kPer;
  float v[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const float logit = x[min(mine + j, end - 1)];
    v[j] = mine + j < end ? logit : -INFINITY;
  }
  auto weight_of = [&](float logit, int i) {
    const u64 w = fixed_weight(logit, r);
    return w >= set.min_w && topk_key(logit, static_cast<uint32_t>(i)) >= cut ? w : u64{0};
  };
  u64 sum = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) sum += weight_of(v[j], mine + j);
  u64 all;
  u64 at = block_prefix<THREADS / kWave>(sum, sh.scan, &all) - sum;
  if (at <= target && target < at + sum) {
    // this thread's: its tokens again, one by one
    for (int i = mine; i < end; ++i) {
      const u64 w = weight_of(x[i], i);
      if (target < at + w) {
        store_token(a, row, i, x[i], r, total);
        break;
      }
      at += w;
    }
  }
}

// One workgroup a row.  Bound by the barriers of its sort and sums: 12.4 us with
// lists of up to a thousand keys (64 rows), 5.4 with none.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void sample_draw_kernel(SampleArgs a) {
  __shared__ DrawShared sh;
  const int row = blockIdx.x;
  const int tid = threadIdx.x;
  const float *x = a.logits + row * a.row_stride;
  fill_table(sh.table);
  // what the earlier launches left, loaded at once (a row without cuts has
  // no ends and no list: those words are not used then)
  const u64 *part_mass = a.part_mass + static_cast<int64_t>(row) * a.parts;
  u64 mass = tid < a.parts ? part_mass[tid] : 0;
  const RowEnds e = a.ends[row];
  const uint32_t entries = a.list_count[row];
  const u64 key = a.list[static_cast<int64_t>(row) * kListMax + tid];
  const float uniform = a.uniform[row];
  const RowSettings set = row_settings(a, row);
  const float mx = row_max(a, row);
  if (no_token(mx)) return store_no_token(a, row);
  if (set.greedy) return store_largest<THREADS>(a, row, x, mx, sh.first);
  __syncthreads();  // the table
  const RowScale r = row_scale(mx, set, sh.table);
  u64 cut = 0;
  if (set.use_k || set.use_p) {
    if (entries > kListMax) {
      cut = counted_row<THREADS>(a, x, r, set, sh);
      if (tid < a.parts) mass = sh.mass[tid];
    } else if (entries > 0) {
      if (tid < a.parts) sh.mass[tid] = mass;
      const int n = static_cast<int>(entries);
      cut = n <= THREADS
                ? list_cut<THREADS, 1>(nullptr, n, tid < n ? key : 0, e, set, r, sh)
                : list_cut<THREADS, kListMax / THREADS>(
                      a.list + static_cast<int64_t>(row) * kListMax, n, 0, e, set, r, sh);
      // what the list adds to its parts
      for (int i = tid; i < static_cast<int>(entries); i += THREADS) {
        const u64 key = sh.keys[i];
        const u64 w = fixed_weight(key_value(key), r);
        if (key >= cut && w >= set.min_w) atomicAdd(&sh.mass[key_index(key) / kPart], w);
      }
      __syncthreads();
      if (tid < a.parts) mass = sh.mass[tid];
    }
  }
  draw_token<THREADS>(a, row, x, uniform, mass, cut, r, set, sh);
}

// Where the top_k of the tokens in `count` (LDS; there is one at least) end.
struct CountEnd {
  int bin;
  uint32_t above;  // tokens in the bins above it
  uint32_t need;   // and taken of it
};

struct CountShared {
  int scan[kSampleWaves];
  int bin, above;
};

template <int THREADS>
__device__ __forceinline__ CountEnd count_end(const uint32_t *count, int64_t top_k,
                                              CountShared &sh) {
  constexpr int kPer = kSampleBins / THREADS;
  const int tid = threadIdx.x;
  int c[kPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    c[i] = static_cast<int>(count[tid * kPer + i]);
    sum += c[i];
  }
  const int upto = wave_prefix(sum);
  if ((tid & (kWave - 1)) == kWave - 1) sh.scan[tid / kWave] = upto;
  __syncthreads();
  int at = upto - sum, all = 0;
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) {
    if (w < tid / kWave) at += sh.scan[w];
    all += sh.scan[w];
  }
  const int need = static_cast<int>(min(top_k, static_cast<int64_t>(all)));
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (at < need && need <= at + c[i]) {
      sh.bin = tid * kPer + i;
      sh.above = at;
    }
    at += c[i];
  }
  __syncthreads();
  return CountEnd{sh.bin, static_cast<uint32_t>(sh.above),
                  static_cast<uint32_t>(need - sh.above)};
}

constexpr int kTopFours = 160;  // vectors that a wave gathers

__device__ __forceinline__ int lanes_below(uint64_t which) {
  return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(which >> 32),
                                   __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(which), 0));
}

// A workgroup a chunk: its largest logit, and a list of the tokens in the bins
// (under that logit) of its top_k largest, which hold the row's.  Bound by
// latency for one row of 128256 (4.4 us) and by its reads for 64 (11.3 us with
// top-k 40, where the largest logits alone take 6.5); with every lane listing
// its own tokens, an atomic behind the other, 5.7 and 13.8.
__global__ __launch_bounds__(kChunkThreads) void sample_top_kernel(SampleArgs a) {
  __shared__ uint32_t s_bins[kSampleBins];
  __shared__ f32x4_at4 s_four[kChunkThreads / kWave][kTopFours];
  __shared__ int s_at[kChunkThreads / kWave][kTopFours];
  __shared__ float s_max[kChunkThreads / kWave];
  __shared__ CountShared s_end;
  __shared__ uint32_t s_count;
  const int chunk = static_cast<int>(blockIdx.x) % a.chunks;
  const int row = static_cast<int>(blockIdx.x) / a.chunks;
  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int wave = tid / kWave;
  const auto logits = row_chunk(a, row, chunk);
  const RowSettings set = row_settings(a, row);
  for (int i = tid; i < kSampleBins; i += kChunkThreads) s_bins[i] = 0;
  if (tid == 0) s_count = 0;
  float best = -INFINITY;
  logits.each([&](const f32x4_at4 &v, int, int) {
    best = nan_max(nan_max(best, nan_max(v[0], v[1])), nan_max(v[2], v[3]));
  });
  best = wave_nan_max(best);
  if (lane == 0) s_max[wave] = best;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kChunkThreads / kWave; ++w) best = nan_max(best, s_max[w]);
  if (tid == 0) a.chunk_max[static_cast<int64_t>(row) * a.chunks + chunk] = best;
  uint32_t *listed = a.bin_count + static_cast<int64_t>(row) * kSampleBins + chunk;
  if (set.greedy || no_token(best)) {  // uniform
    if (tid == 0) *listed = 0;
    return;
  }
  const RowScale r = row_scale(best, set, nullptr);
  // the largest of every four neighbours are enough to count: where top_k of
  // them end, top_k tokens have been passed
  auto four_bin = [&](const f32x4_at4 &v) {
    return weight_bin(log_weight(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), r));
  };
  logits.each([&](const f32x4_at4 &v, int, int) {
    const int b = four_bin(v);
    if (b < kSampleBins) atomicAdd(&s_bins[b], 1u);
  });
  __syncthreads();
  const CountEnd end = count_end<kChunkThreads>(s_bins, set.top_k, s_end);
  // fewer fours than top_k: at most kTopCap tokens, all listed
  const int last = end.above + end.need < set.top_k ? kSampleBins - 1 : end.bin;
  // a wave gathers its fours that hold such a token, so that its lanes take a
  // logit of these each
  int fours = 0;
  logits.each([&](const f32x4_at4 &v, int at, int) {
    const bool in = four_bin(v) <= last;
    const uint64_t which = __ballot(in);
    // (a lane that had no four before this one has not counted them)
    fours = __builtin_amdgcn_readfirstlane(fours);
    const int n = fours + lanes_below(which);
    if (in && n < kTopFours) {
      s_four[wave][n] = v;
      s_at[wave][n] = at;
    }
    fours += __popcll(which);
  });
  fours = __builtin_amdgcn_readfirstlane(fours);
  u64 *list = a.list + (static_cast<int64_t>(row) * a.chunks + chunk) * kTopCap;
  for (int first = 0; first < 4 * min(fours, kTopFours); first += kWave) {
    const int i = first + lane;
    const bool mine = i < 4 * min(fours, kTopFours);
    const float v = mine ? s_four[wave][i / 4][i % 4] : -INFINITY;
    const bool in = weight_bin(log_weight(v, r)) <= last;
    const uint64_t which = __ballot(in);
    uint32_t base = 0;
    if (lane == 0) base = atomicAdd(&s_count, static_cast<uint32_t>(__popcll(which)));
    const uint32_t n = __builtin_amdgcn_readfirstlane(base) + lanes_below(which);
    if (in && n < kTopCap)
      list[n] = topk_key(v, static_cast<uint32_t>(s_at[wave][i / 4] + i % 4));
  }
  // more than fit: the draw counts over the row
  if (lane == 0 && fours > kTopFours) atomicAdd(&s_count, kTopCap + 1);
  __syncthreads();
  if (tid == 0) *listed = s_count;
}

// One workgroup a row: bins of the chunks' lists under the row's largest logit
// give its top_k, which are sorted and cut as in the draw above.  At most kTopK
// tokens are left, and each finds the mass before it by itself.  Bound by its
// barriers: 7.8 us for 63 lists of top-k 40 or 64 rows of 16 lists.
constexpr int kTopHeld = 8;   // lists of which a wave holds the first keys: one a
constexpr int kTopTwo = 56;  // lane, and from this top_k on (ties come on top) two

template <int THREADS>
__global__ __launch_bounds__(THREADS) void sample_top_draw_kernel(SampleArgs a) {
  static_assert(kTopK <= THREADS, "a token a thread");
  constexpr int kWaves = THREADS / kWave;
  __shared__ DrawShared sh;
  __shared__ CountShared s_end;
  __shared__ uint32_t s_count, s_over;
  const int row = blockIdx.x;
  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int wave = tid / kWave;
  const float *x = a.logits + row * a.row_stride;
  const uint32_t *listed = a.bin_count + static_cast<int64_t>(row) * kSampleBins;
  const u64 *list = a.list + static_cast<int64_t>(row) * a.chunks * kTopCap;
  const bool two = a.top_k_value >= kTopTwo;
  u64 held[kTopHeld], more[kTopHeld];
  int count[kTopHeld];
#pragma unroll
  for (int j = 0; j < kTopHeld; ++j) {
    const int c = min(wave + kWaves * j, a.chunks - 1);
    count[j] = wave + kWaves * j < a.chunks ? static_cast<int>(listed[c]) : 0;
    held[j] = list[c * kTopCap + lane];
    if (two) more[j] = list[c * kTopCap + kWave + lane];
  }
  const float uniform = a.uniform[row];
  const RowSettings set = row_settings(a, row);
  const float mx = row_max(a, row);
  fill_table(sh.table);
  if (no_token(mx)) return store_no_token(a, row);
  if (set.greedy) return store_largest<THREADS>(a, row, x, mx, sh.first);
  for (int i = tid; i < kSampleBins; i += THREADS) sh.row.count[i] = 0;
  if (tid == 0) s_count = s_over = 0;
  __syncthreads();
  const RowScale r = row_scale(mx, set, sh.table);
  // f(key) for every listed token
  auto each = [&](auto f) {
    auto rest = [&](int c, int first, int n) {
#pragma unroll 1
      for (int i = first + lane; i < n; i += kWave) f(list[c * kTopCap + i]);
    };
#pragma unroll
    for (int j = 0; j < kTopHeld; ++j)
      if (lane < count[j]) f(held[j]);
    if (two) {  // uniform
#pragma unroll
      for (int j = 0; j < kTopHeld; ++j)
        if (kWave + lane < count[j]) f(more[j]);
    }
    const int known = two ? 2 * kWave : kWave;
#pragma unroll
    for (int j = 0; j < kTopHeld; ++j)
      if (count[j] > known) rest(wave + kWaves * j, known, count[j]);
#pragma unroll 1
    for (int c = wave + kWaves * kTopHeld; c < a.chunks; c += kWaves)
      if (listed[c] <= kTopCap) rest(c, 0, static_cast<int>(listed[c]));
  };
  // a list that did not fit has holes: its keys are nothing to work with
#pragma unroll
  for (int j = 0; j < kTopHeld; ++j)
    if (count[j] > kTopCap) {
      s_over = 1;
      count[j] = 0;
    }
  for (int c = kWaves * kTopHeld + tid; c < a.chunks; c += THREADS)
    if (listed[c] > kTopCap) s_over = 1;
  each([&](u64 key) {
    const int b = weight_bin(log_weight(key_value(key), r));
    if (b < kSampleBins) atomicAdd(&sh.row.count[b], 1u);
  });
  __syncthreads();
  bool over = s_over != 0;
  if (!over) {
    const CountEnd end = count_end<THREADS>(sh.row.count, set.top_k, s_end);
    each([&](u64 key) {  // (the list takes the place of the bins)
      if (weight_bin(log_weight(key_value(key), r)) > end.bin) return;
      const uint32_t n = atomicAdd(&s_count, 1u);
      if (n < kListMax) sh.keys[n] = key;
    });
    __syncthreads();
    const int n = static_cast<int>(s_count);
    over = n > kListMax;
    if (!over) {
      const RowEnds e{0, 0, 0, end.need, end.above, 0, end.bin, end.bin};
      u64 cut;
      if (n <= THREADS) {
        const u64 key = tid < n ? sh.keys[tid] : 0;
        __syncthreads();  // the sort writes sh.keys
        cut = list_cut<THREADS, 1>(nullptr, n, key, e, set, r, sh);
      } else {
        cut = list_cut<THREADS, kListMax / THREADS>(sh.keys, n, 0, e, set, r, sh);
      }
      // (sorted: the tokens that are left are the first)
      const int left = static_cast<int>(end.above + end.need);
      const u64 key = tid < left ? sh.keys[tid] : 0;
      u64 w = tid < left && key >= cut ? fixed_weight(key_value(key), r) : 0;
      w = w >= set.min_w ? w : 0;
      if (tid < left) sh.mass[tid] = w;
      __syncthreads();
      if (tid >= left) return;
      const uint32_t index = static_cast<uint32_t>(key_index(key));
      u64 total = 0, before = 0;
#pragma unroll 8
      for (int i = 0; i < left; ++i) {
        const u64 other = sh.mass[i];
        total += other;
        before += static_cast<uint32_t>(key_index(sh.keys[i])) < index ? other : 0;
      }
      const u64 target = target_of(uniform, total);
      if (before <= target && target < before + w)
        store_token(a, row, index, key_value(key), r, total);
      return;
    }
    __syncthreads();  // (the count takes the place of the list)
  }
  const u64 cut = counted_row<THREADS>(a, x, r, set, sh);
  draw_token<THREADS>(a, row, x, uniform, tid < a.parts ? sh.mass[tid] : 0, cut, r, set, sh);
}

// A row of at most kShortVocab logits in one launch: the row stays in the
// registers of one workgroup, its bins and its list in LDS.  Bound by its
// barriers: top-k 40 and top-p 0.95 of 4096 logits 11.5 us, of 64 rows of
// 16384 18.2, of 256 rows 20.2.  Four waves take rows of up to 4096: fewer to
// wait for.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void sample_short_kernel(SampleArgs a) {
  __shared__ DrawShared sh;
  constexpr int kWaves = THREADS / kWave;
  __shared__ float s_max[kWaves];
  __shared__ uint32_t s_count;
  const int row = blockIdx.x;
  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int wave = tid / kWave;
  const float *x = a.logits + row * a.row_stride;
  const Chunk<THREADS, kShortVecs> logits(x, 0, a.vocab);
  const float uniform = a.uniform[row];
  const RowSettings set = row_settings(a, row);
  fill_table(sh.table);
  for (int b = tid; b < kSampleBins; b += THREADS) {
    sh.row.count[b] = 0;
    sh.row.mass[b] = 0;
  }
  if (tid == 0) {
    s_count = 0;
    sh.first[0] = 0x7fffffff;
  }
  float mx = -INFINITY;
  logits.each([&](const f32x4_at4 &v, int, int) {
    mx = nan_max(nan_max(mx, nan_max(v[0], v[1])), nan_max(v[2], v[3]));
  });
  mx = wave_nan_max(mx);
  if (lane == 0) s_max[wave] = mx;
  __syncthreads();
#pragma unroll 4
  for (int w = 0; w < kWaves; ++w) mx = nan_max(mx, s_max[w]);
  if (no_token(mx)) return store_no_token(a, row);
  if (set.greedy) {
    int at = 0x7fffffff;
    logits.each([&](const f32x4_at4 &v, int first, int) {
#pragma unroll
      for (int i = 3; i >= 0; --i) at = v[i] == mx ? min(at, first + i) : at;
    });
    if (at != 0x7fffffff) atomicMin(&sh.first[0], at);
    __syncthreads();
    if (tid == 0) {
      a.ids[row] = sh.first[0];
      if (a.logprobs != nullptr) a.logprobs[row] = 0.0f;
    }
    return;
  }
  const RowScale r = row_scale(mx, set, sh.table);
  const bool use_k = set.use_k, use_p = set.use_p;
  u64 cut = 0;
  if (use_k || use_p) {
    logits.each([&](const f32x4_at4 &v, int, int) {
      add_to_bins(v, r, use_k, use_p, sh.row.count, sh.row.mass);
    });
    __syncthreads();
    const RowEnds e = find_ends(BinShare<THREADS>(sh.row.mass, sh.row.count, set), set);
    if (e.last_p >= 0 || e.last_k >= 0) {
      __syncthreads();  // the list takes the place of the bins
      logits.each([&](const f32x4_at4 &v, int at, int) {
        double t[4];
        int b[4];
        bins_of(v, r, t, b);
        list_of(v, at, b, e.first, e, sh.keys, &s_count);
      });
      __syncthreads();
      const int n = static_cast<int>(s_count);
      if (n > kListMax) {
        u64 live = 0, sum = 0;
        logits.each([&](const f32x4_at4 &v, int, int) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const u64 w = fixed_weight(v[i], r);
            live += w != 0 ? 1 : 0;
            sum += w;
          }
        });
        u64 live_all, mass_all;
        block_prefix<kWaves>(live, sh.scan, &live_all);
        block_prefix<kWaves>(sum, sh.scan, &mass_all);
        cut = counted_cut<THREADS>(x, a.vocab, r, set, mass_all, live_all, sh.row);
      } else if (n <= THREADS) {
        const u64 key = tid < n ? sh.keys[tid] : 0;
        __syncthreads();  // the sort writes sh.keys
        cut = list_cut<THREADS, 1>(nullptr, n, key, e, set, r, sh);
      } else {
        cut = list_cut<THREADS, kListMax / THREADS>(sh.keys, n, 0, e, set, r, sh);
      }
    }
  }
  // the draw: masses of the threads' vectors, in the order of their tokens
  // (vector j of all threads, then vector j + 1; the rest last)
  auto in_cut = [&](float logit, int i) {
    return topk_key(logit, static_cast<uint32_t>(i)) >= cut;
  };
  auto weight_of = [&](float logit, int i) {
    const u64 w = fixed_weight(logit, r);
    return w >= set.min_w && in_cut(logit, i) ? w : u64{0};
  };
  u64 sum[kShortVecs + 1];
#pragma unroll
  for (int j = 0; j < kShortVecs; ++j) {
    sum[j] = 0;
    if (logits.at(j) < logits.whole) {
      // (a cut leaves most vectors nothing)
      bool any = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) any |= in_cut(logits.v[j][i], logits.at(j) + i);
      if (any) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[j] += weight_of(logits.v[j][i], logits.at(j) + i);
      }
    }
    sum[j] = wave_prefix(sum[j]);
    if (lane == kWave - 1) sh.mass[j * kWaves + wave] = sum[j];
  }
  const int last = logits.whole + tid;
  sum[kShortVecs] = last < logits.end ? weight_of(logits.rest, last) : 0;
  sum[kShortVecs] = wave_prefix(sum[kShortVecs]);
  if (tid == kWave - 1) sh.mass[kShortVecs * kWaves] = sum[kShortVecs];
  __syncthreads();
  // prefix sums of the waves' masses: one a lane of the first waves
  constexpr int kParts = kShortVecs * kWaves + 1;
  u64 total;
  const u64 part = tid < kParts ? sh.mass[tid] : 0;
  const u64 upto = block_prefix<kWaves>(part, sh.scan, &total);
  if (tid < kParts) sh.mass[tid] = upto - part;
  __syncthreads();
  const u64 target = target_of(uniform, total);
#pragma unroll
  for (int j = 0; j <= kShortVecs; ++j) {
    if (j == kShortVecs && wave != 0) break;
    const u64 base = sh.mass[j * kWaves + (j < kShortVecs ? wave : 0)];
    // this thread's share of vector j: from the lane before it on
    u64 at = __shfl_up(sum[j], 1);
    at = base + (lane == 0 ? 0 : at);
    if (at <= target && target < base + sum[j]) {
      for (int i = j < kShortVecs ? logits.at(j) : last; i < a.vocab; ++i) {
        const u64 w = weight_of(x[i], i);
        if (target < at + w) {
          store_token(a, row, i, x[i], r, total);
          break;
        }
        at += w;
      }
    }
  }
}

// A row's chunks: enough of them to fill the device with few rows, as large
// as possible otherwise (fewer sums to join).
struct SamplePlan {
  int64_t chunk, chunks;
  int64_t parts;
  size_t max_bytes, mass_bytes, bin_mass_bytes, bin_count_bytes, ends_bytes, list_bytes,
      count_bytes;
  size_t bytes;  // of all of them
};

static int64_t chunks_wanted(int64_t rows) { return (kChunkWorkgroups + rows - 1) / rows; }

static SamplePlan sample_plan(int64_t rows, int64_t vocab) {
  SamplePlan p{};
  if (rows > kSliceRows) rows = kSliceRows;  // more rows go slice by slice
  const int64_t want = chunks_wanted(rows);
  p.chunk = (vocab + want - 1) / want;
  p.chunk = (p.chunk + kPart - 1) / kPart * kPart;
  if (p.chunk < kChunkMin) p.chunk = kChunkMin;
  if (p.chunk > kChunkMax) p.chunk = kChunkMax;
  p.chunks = (vocab + p.chunk - 1) / p.chunk;
  auto rounded = [](size_t bytes) { return (bytes + 255) / 256 * 256; };
  const size_t r = static_cast<size_t>(rows);
  p.max_bytes = rounded(r * p.chunks * sizeof(float));
  p.parts = (vocab + kPart - 1) / kPart;
  p.mass_bytes = rounded(r * p.parts * sizeof(u64));
  p.bin_mass_bytes = rounded(r * kSampleBins * sizeof(u64));
  p.bin_count_bytes = rounded(r * kSampleBins * sizeof(uint32_t));
  p.ends_bytes = rounded(r * sizeof(RowEnds));
  p.list_bytes = rounded(
      r * std::max<int64_t>(kListMax, p.chunks * kTopCap) * sizeof(u64));
  p.count_bytes = rounded(r * sizeof(uint32_t));
  p.bytes = p.max_bytes + p.mass_bytes + p.bin_mass_bytes + p.bin_count_bytes + p.ends_bytes +
            p.list_bytes + p.count_bytes;
  return p;
}

}  // namespace cascade

using namespace cascade;

extern "C" size_t cascade_sample_workspace_bytes(int64_t rows, int64_t vocab) {
  if (rows <= 0 || vocab <= 0 || vocab > kSampleMaxVocab || rows > 0x7fffffff) return 0;
  if (vocab <= kShortVocab) return 256;
  // enough for fewer rows too, which may be cut into more chunks, and for fewer
  // logits: their chunks are most where a smaller size of chunk ends
  size_t most = 0;
  for (int64_t r = rows < kSliceRows ? rows : kSliceRows; r >= 1; --r) {
    most = std::max(most, sample_plan(r, vocab).bytes);
    for (int64_t chunk = kChunkMin; chunk < kChunkMax; chunk += kPart) {
      const int64_t end = chunks_wanted(r) * chunk;
      if (end > kShortVocab && end < vocab) most = std::max(most, sample_plan(r, end).bytes);
    }
  }
  return most;
}

extern "C" int cascade_sample_f32(const float *logits, int64_t row_stride, int64_t rows,
                                  int64_t vocab, const float *uniform,
                                  const float *temperature, double temperature_value,
                                  const int32_t *top_k, int64_t top_k_value,
                                  const float *top_p, double top_p_value,
                                  const float *min_p, double min_p_value, int64_t *ids,
                                  float *logprobs, void *workspace,
                                  size_t workspace_bytes, void *stream) {
  if (logits == nullptr || uniform == nullptr || ids == nullptr || workspace == nullptr)
    return CASCADE_EINVAL;
  if (rows <= 0 || rows > 0x7fffffff || vocab <= 0 || row_stride < vocab) return CASCADE_EINVAL;
  if (vocab > kSampleMaxVocab) return CASCADE_ESHAPE;
  // NaN settings are refused too
  if ((top_p == nullptr && !(top_p_value >= 0.0)) || (min_p == nullptr && !(min_p_value >= 0.0)) ||
      (temperature == nullptr && !(temperature_value >= 0.0)))
    return CASCADE_EINVAL;
  const void *words[] = {logits, uniform, temperature, top_k, top_p, min_p, logprobs};
  for (const void *p : words)
    if (reinterpret_cast<uintptr_t>(p) & 3) return CASCADE_EALIGN;
  if ((reinterpret_cast<uintptr_t>(ids) & 7) || !aligned16(workspace)) return CASCADE_EALIGN;
  const bool short_rows = vocab <= kShortVocab;
  if (short_rows && rows > 0xffffffff / kSampleThreads) return CASCADE_ESHAPE;
  const SamplePlan p = short_rows ? SamplePlan{} : sample_plan(rows, vocab);
  if (workspace_bytes < (short_rows ? size_t{256} : p.bytes)) return CASCADE_EWORKSPACE;
  SampleArgs a{};
  a.row_stride = row_stride;
  a.vocab = static_cast<int32_t>(vocab);
  a.temperature_value = temperature_value;
  a.top_k_value = top_k_value;
  a.top_p_value = top_p_value;
  a.min_p_value = min_p_value;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (short_rows) {
    a.logits = logits;
    a.uniform = uniform;
    a.temperature = temperature;
    a.top_k = top_k;
    a.top_p = top_p;
    a.min_p = min_p;
    a.ids = ids;
    a.logprobs = logprobs;
    const dim3 grid(static_cast<unsigned>(rows));
    // as few waves as hold the row: every sum waits for all of them
    if (vocab <= 4 * 256 * kShortVecs)
      return launch_kernel(sample_short_kernel<256>, grid, dim3(256), 0, s, a);
    return launch_kernel(sample_short_kernel<kSampleThreads>, grid, dim3(kSampleThreads), 0,
                         s, a);
  }
  a.chunk = static_cast<int32_t>(p.chunk);
  a.chunks = static_cast<int32_t>(p.chunks);
  unsigned char *ws = static_cast<unsigned char *>(workspace);
  auto take = [&ws](size_t bytes) {
    unsigned char *part = ws;
    ws += bytes;
    return part;
  };
  a.chunk_max = reinterpret_cast<float *>(take(p.max_bytes));
  a.parts = static_cast<int32_t>(p.parts);
  a.part_mass = reinterpret_cast<u64 *>(take(p.mass_bytes));
  a.bin_mass = reinterpret_cast<u64 *>(take(p.bin_mass_bytes));
  a.bin_count = reinterpret_cast<uint32_t *>(take(p.bin_count_bytes));
  a.ends = reinterpret_cast<RowEnds *>(take(p.ends_bytes));
  a.list = reinterpret_cast<u64 *>(take(p.list_bytes));
  a.list_count = reinterpret_cast<uint32_t *>(take(p.count_bytes));
  // numbers for all rows that cut nothing need no lists
  const bool cuts = top_k != nullptr || top_k_value > 0 || top_p != nullptr ||
                    top_p_value < 1.0 || min_p != nullptr || min_p_value > 1.0;
  // a list of at most a key a thread is sorted in registers; more threads make
  // every sum dearer
  const bool few = top_k == nullptr && top_k_value <= kFewK;
  const bool top = top_k == nullptr && top_k_value > 0 && top_k_value <= kTopK;
  const dim3 block(kChunkThreads);
  for (int64_t first = 0; first < rows; first += kSliceRows) {
    const int64_t count = rows - first < kSliceRows ? rows - first : kSliceRows;
    a.logits = logits + first * row_stride;
    a.uniform = uniform + first;
    a.temperature = temperature != nullptr ? temperature + first : nullptr;
    a.top_k = top_k != nullptr ? top_k + first : nullptr;
    a.top_p = top_p != nullptr ? top_p + first : nullptr;
    a.min_p = min_p != nullptr ? min_p + first : nullptr;
    a.ids = ids + first;
    a.logprobs = logprobs != nullptr ? logprobs + first : nullptr;
    const dim3 grid(static_cast<unsigned>(count * p.chunks));
    const dim3 rows_grid(static_cast<unsigned>(count));
    if (top) {
      hipError_t e = launch_kernel(sample_top_kernel, grid, block, 0, s, a);
      if (e != hipSuccess) return e;
      e = launch_kernel(sample_top_draw_kernel<kFewThreads>, rows_grid, dim3(kFewThreads), 0,
                        s, a);
      if (e != hipSuccess) return e;
      continue;
    }
    hipError_t e = launch_kernel(sample_max_kernel, grid, block, 0, s, a);
    if (e != hipSuccess) return e;
    e = launch_kernel(sample_weigh_kernel, grid, block, 0, s, a);
    if (e != hipSuccess) return e;
    if (cuts) {
      e = launch_kernel(sample_collect_kernel, grid, block, 0, s, a);
      if (e != hipSuccess) return e;
    }
    e = few ? launch_kernel(sample_draw_kernel<kFewThreads>, rows_grid, dim3(kFewThreads), 0,
                            s, a)
            : launch_kernel(sample_draw_kernel<kSampleThreads>, rows_grid,
                            dim3(kSampleThreads), 0, s, a);
    if (e != hipSuccess) return e;
  }
  return 0;
}
