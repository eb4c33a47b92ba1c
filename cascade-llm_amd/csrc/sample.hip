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
// cut up.  A token below 2^-45 of the likeliest one is never drawn.  The
// cuts K and P are found by counting: histograms of 11 bits of the ordered
// logits, from the top down.
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
};

struct RowSettings {
  bool greedy;
  double scale;   // log2(e) / T
  int64_t top_k;  // <= 0: off
  double top_p;   // >= 1: off
  u64 min_w;      // smallest weight kept
};

__device__ __forceinline__ RowSettings row_settings(const SampleArgs &a, int row) {
  RowSettings r;
  const double t = a.temperature != nullptr ? static_cast<double>(a.temperature[row])
                                            : a.temperature_value;
  r.greedy = !(t > 0.0);
  r.scale = 1.4426950408889634 / t;
  r.top_k = a.top_k != nullptr ? static_cast<int64_t>(a.top_k[row]) : a.top_k_value;
  r.top_p = a.top_p != nullptr ? static_cast<double>(a.top_p[row]) : a.top_p_value;
  const double p = a.min_p != nullptr ? static_cast<double>(a.min_p[row]) : a.min_p_value;
  r.min_w = p > 0.0 ? static_cast<u64>(ceil(fmin(p, 1.0) * static_cast<double>(kWeightOne)))
                    : u64{0};
  if (p > 1.0) r.top_k = 1;  // none reaches it: the likeliest alone stays
  return r;
}

// 2^(44 + y) rounded to an integer, y <= 0; 0 below y = -45.  2^f for
// |f| <= 1/2 is the Taylor polynomial of e^(f ln 2) to the 12th power, whose
// remainder is below 2e-16.
__device__ __forceinline__ u64 fixed_exp2(double y) {
  if (!(y > -45.0)) return 0;
  const double n = rint(y);
  const double z = (y - n) * 0.6931471805599453;
  double p = 1.0 / 479001600.0;
  p = fma(p, z, 1.0 / 39916800.0);
  p = fma(p, z, 1.0 / 3628800.0);
  p = fma(p, z, 1.0 / 362880.0);
  p = fma(p, z, 1.0 / 40320.0);
  p = fma(p, z, 1.0 / 5040.0);
  p = fma(p, z, 1.0 / 720.0);
  p = fma(p, z, 1.0 / 120.0);
  p = fma(p, z, 1.0 / 24.0);
  p = fma(p, z, 1.0 / 6.0);
  p = fma(p, z, 0.5);
  p = fma(p, z, 1.0);
  p = fma(p, z, 1.0);
  return static_cast<u64>(ldexp(p, static_cast<int>(n) + kWeightBits) + 0.5);
}

// Weight of logit x in a row whose largest logit is mx: 2^44 for the largest
// itself (also where it is infinite), 0 for -inf.
__device__ __forceinline__ u64 fixed_weight(float x, float mx, double scale) {
  if (x == mx) return kWeightOne;
  if (x == -INFINITY) return 0;
  return fixed_exp2((static_cast<double>(x) - static_cast<double>(mx)) * scale);
}

// Inclusive prefix sum over the wave's lanes.
__device__ __forceinline__ u64 wave_prefix(u64 v, int lane) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const u64 o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// Inclusive prefix sum over the workgroup in thread order, and its total.
// Two barriers; `lds` may be reused after the second.
__device__ __forceinline__ u64 block_prefix(u64 v, u64 *lds, u64 *total) {
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = threadIdx.x / kWave;
  v = wave_prefix(v, lane);
  if (lane == kWave - 1) lds[wave] = v;
  __syncthreads();
  u64 before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSampleWaves; ++w) {
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
template <bool BY_MASS>
__device__ Cut find_cut(const float *x, int n, float mx, double scale, Cut in, u64 need,
                        SampleShared &sh, u64 *mass_kept) {
  const int tid = threadIdx.x;
  uint32_t prefix = 0, known = 0;  // the value's bits found so far
  u64 above_count = 0, above_mass = 0;
  u64 equal = 0, equal_mass = 0;
#pragma unroll 1
  for (int round = 0; round < 3; ++round) {
    const int shift = round == 0 ? 21 : round == 1 ? 10 : 0;
    const uint32_t bins = round == 2 ? 1024u : 2048u;
    for (int b = tid; b < kSampleBins; b += kSampleThreads) {
      sh.count[b] = 0;
      sh.mass[b] = 0;
    }
    __syncthreads();
    for (int i = tid; i < n; i += kSampleThreads) {
      const float v = x[i];
      const uint32_t o = ordered_bits(v);
      if ((o & known) != prefix || !keeps(in, o, i)) continue;
      const u64 w = fixed_weight(v, mx, scale);
      if (w == 0) continue;
      const uint32_t b = (o >> shift) & (bins - 1);
      atomicAdd(&sh.count[b], 1u);
      atomicAdd(&sh.mass[b], w);
    }
    __syncthreads();
    // thread t scans bins 2047 - 2 t and 2046 - 2 t, from the top down
    const int hi = kSampleBins - 1 - 2 * tid, lo = hi - 1;
    const u64 c0 = sh.count[hi], c1 = sh.count[lo];
    const u64 m0 = sh.mass[hi], m1 = sh.mass[lo];
    u64 total;
    const u64 c_end = block_prefix(c0 + c1, sh.scan, &total) + above_count;
    const u64 m_end = block_prefix(m0 + m1, sh.scan, &total) + above_mass;
    const u64 c_mid = c_end - c1, c_start = c_mid - c0;
    const u64 m_mid = m_end - m1, m_start = m_mid - m0;
    const u64 end = BY_MASS ? m_end : c_end, mid = BY_MASS ? m_mid : c_mid,
              start = BY_MASS ? m_start : c_start;
    if (start < need && need <= end) {
      const bool first = need <= mid;
      sh.found[0] = first ? hi : lo;
      sh.found[1] = first ? c_start : c_mid;
      sh.found[2] = first ? m_start : m_mid;
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
  Cut cut{prefix, 0xffffffffu};
  if (take < equal) {
    // the index of the take-th of them
    u64 seen = 0;
    for (int base = 0; base < n; base += kSampleThreads) {
      const int i = base + tid;
      const bool hit = i < n && ordered_bits(x[i]) == prefix;
      u64 total;
      const u64 at = seen + block_prefix(hit ? 1 : 0, sh.scan, &total);
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

// One workgroup a row.
__global__ __launch_bounds__(kSampleThreads) void sample_row_kernel(SampleArgs a) {
  __shared__ SampleShared sh;
  const int row = blockIdx.x;
  const int tid = threadIdx.x;
  const int n = a.vocab;
  const float *x = a.logits + row * a.row_stride;
  const RowSettings set = row_settings(a, row);

  // the largest key (its logit, and the lowest index that has it); a NaN
  // sorts above every number
  u64 best = 0;
  for (int i = tid; i < n; i += kSampleThreads) {
    const u64 key = topk_key(x[i], static_cast<uint32_t>(i));
    best = key > best ? key : best;
  }
  best = wave_max_u64(best);
  if ((tid & (kWave - 1)) == 0) sh.scan[tid / kWave] = best;
  __syncthreads();
  for (int w = 0; w < kSampleWaves; ++w) best = sh.scan[w] > best ? sh.scan[w] : best;
  __syncthreads();
  const float mx = key_value(best);
  const bool empty = mx != mx || mx == -INFINITY;
  if (empty || set.greedy) {
    if (tid == 0) {
      a.ids[row] = empty ? -1 : key_index(best);
      if (a.logprobs != nullptr) a.logprobs[row] = empty ? __builtin_nanf("") : 0.0f;
    }
    return;
  }

  // number and mass of the tokens that have a weight
  u64 live = 0, mass = 0;
  for (int i = tid; i < n; i += kSampleThreads) {
    const u64 w = fixed_weight(x[i], mx, set.scale);
    live += w != 0 ? 1 : 0;
    mass += w;
  }
  u64 live_all, mass_all;
  block_prefix(live, sh.scan, &live_all);
  block_prefix(mass, sh.scan, &mass_all);
  Cut cut{0u, 0xffffffffu};
  if (set.top_k > 0 && static_cast<u64>(set.top_k) < live_all)
    cut = find_cut<false>(x, n, mx, set.scale, cut, static_cast<u64>(set.top_k), sh, &mass_all);
  if (set.top_p < 1.0) {
    const double need = ceil(set.top_p * static_cast<double>(mass_all));
    u64 need_int = need >= 1.0 ? static_cast<u64>(need) : 1;
    need_int = need_int < mass_all ? need_int : mass_all;
    cut = find_cut<true>(x, n, mx, set.scale, cut, need_int, sh, &mass_all);
  }
  if (set.min_w > 0) {
    mass = 0;
    for (int i = tid; i < n; i += kSampleThreads) {
      const u64 w = fixed_weight(x[i], mx, set.scale);
      if (w >= set.min_w && keeps(cut, ordered_bits(x[i]), i)) mass += w;
    }
    block_prefix(mass, sh.scan, &mass_all);
  }
  // the draw
  double u = static_cast<double>(a.uniform[row]);
  u = u > 0.0 ? u : 0.0;  // NaN too
  const double t = u * static_cast<double>(mass_all);
  u64 target = t < static_cast<double>(mass_all) ? static_cast<u64>(t) : mass_all - 1;
  target = target < mass_all ? target : mass_all - 1;
  u64 seen = 0;
  for (int base = 0; base < n; base += kSampleThreads) {
    const int i = base + tid;
    u64 w = 0;
    if (i < n) {
      w = fixed_weight(x[i], mx, set.scale);
      if (w < set.min_w || !keeps(cut, ordered_bits(x[i]), i)) w = 0;
    }
    u64 total;
    const u64 end = seen + block_prefix(w, sh.scan, &total);
    if (w != 0 && end > target && end - w <= target) {
      a.ids[row] = i;
      if (a.logprobs != nullptr)
        a.logprobs[row] = static_cast<float>(
            log(static_cast<double>(w) / static_cast<double>(mass_all)));
    }
    seen += total;
    if (seen > target) break;  // uniform
  }
}

}  // namespace cascade

using namespace cascade;

extern "C" size_t cascade_sample_workspace_bytes(int64_t rows, int64_t vocab) {
  if (rows <= 0 || vocab <= 0 || vocab > kSampleMaxVocab || rows > 0xffff) return 0;
  return 256;
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
  if (rows <= 0 || rows > 0xffff || vocab <= 0 || row_stride < vocab) return CASCADE_EINVAL;
  if (vocab > kSampleMaxVocab) return CASCADE_ESHAPE;
  // NaN settings are refused too
  if ((top_p == nullptr && !(top_p_value >= 0.0)) || (min_p == nullptr && !(min_p_value >= 0.0)) ||
      (temperature == nullptr && !(temperature_value >= 0.0)))
    return CASCADE_EINVAL;
  const void *words[] = {logits, uniform, temperature, top_k, top_p, min_p, logprobs};
  for (const void *p : words)
    if (reinterpret_cast<uintptr_t>(p) & 3) return CASCADE_EALIGN;
  if ((reinterpret_cast<uintptr_t>(ids) & 7) || !aligned16(workspace)) return CASCADE_EALIGN;
  if (workspace_bytes < cascade_sample_workspace_bytes(rows, vocab)) return CASCADE_EWORKSPACE;
  const SampleArgs a{logits, row_stride, static_cast<int32_t>(vocab), uniform,
                     temperature, temperature_value, top_k, top_k_value, top_p,
                     top_p_value, min_p, min_p_value, ids, logprobs};
  return launch_kernel(sample_row_kernel, dim3(static_cast<unsigned>(rows)),
                       dim3(kSampleThreads), 0, static_cast<hipStream_t>(stream), a);
}
