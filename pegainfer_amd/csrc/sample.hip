// Next tokens from logits on MI355X (gfx950): temperature, min-p, top-k, top-p and a draw with a
// given uniform number, for each row l[0 .. V).
//
//   w[v] = e^((l[v] - max l) / T)             zero below e^-28, and below min_p
//   order: by l descending, ties by v ascending
//   top-k: the first k of the order keep their weight
//   top-p: then those with less than p of what is left before them in the order
//   token = the first v, in index order, with w[0] + .. + w[v] > u * (sum of w)
//   logprob = ln(w[token] / sum of w)
//
// T <= 0 takes the first of the order.  A NaN counts as -inf and is never drawn; rows with nothing
// but those give token -1 and logprob -inf.  With +inf logits these alone have weight.
//
// Weights are whole multiples of 2^-44, rounded once from 64 bits, and their sums are of 64-bit
// integers: exact in any order, so that a row's token depends on nothing but its inputs, and every
// comparison is of exact sums (the weights' rounding moves a border by 10^-11 at most).
//
// No sort.  A histogram of the weights' logarithms (counts and masses in LDS) finds the bin in which a cut falls,
// and histograms of the keys inside the bin narrow it to one key; equal keys are cut by index.
#include "common.h"
#include "pega_moe.h"

namespace pega {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 1024;
constexpr int kList = 4096;            // elements of a bin kept in LDS
constexpr int kParts = 128;            // of a row, whose masses the draw goes over first
constexpr int kMaxVocab = 1 << 19;     // sums of weights stay below 2^63
constexpr double kRange = 28.0;        // smaller weights than e^-28 are zero
constexpr double kLog2e = 1.4426950408889634;
constexpr double kBinsPerOctave = kBins / (kRange * kLog2e + 0.01);

typedef unsigned long long u64;
constexpr u64 kNoMass = u64{1} << 63;  // more than any sum of weights, less than 2^64 by more than a weight
constexpr uint32_t kNoCount = 0xffffffffu;

struct SampleArgs {
  const void* logits;
  long long stride;  // elements from row to row
  int rows, vocab;
  const float *u, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  int32_t* tokens;
  float* logprobs;
};

__device__ __forceinline__ float clean(float l) { return l == l ? l + 0.0f : -__builtin_inff(); }  // -0 is 0

// Floats in the order of their values.
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t b = __builtin_bit_cast(uint32_t, l);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <typename T>
struct Row {
  const T* p;
  int n;
  static constexpr int kVec = 16 / sizeof(T);

  static __device__ __forceinline__ float value(uint4 q, int e) {
    if constexpr (sizeof(T) == 4)
      return clean(__builtin_bit_cast(float, e == 0 ? q.x : e == 1 ? q.y : e == 2 ? q.z : q.w));
    const uint32_t w = (e >> 1) == 0 ? q.x : (e >> 1) == 1 ? q.y : (e >> 1) == 2 ? q.z : q.w;
    return clean(e & 1 ? bf_hi(w) : bf_lo(w));
  }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (sizeof(T) == 4) return clean(p[i]);
    else return clean(bf2f(p[i]));
  }
  // f(i, l[i]) for i in [from, to), over `threads` threads: 16-byte loads, four in flight, of what is
  // aligned, element by element before and after
  template <typename F>
  __device__ __forceinline__ void each(int from, int to, int tid, int threads, F f) const {
    const T* q = p + from;
    const int lead = static_cast<int>((16u - (reinterpret_cast<uintptr_t>(q) & 15u)) & 15u) / static_cast<int>(sizeof(T));
    const int head = min(to - from, lead), vecs = (to - from - head) / kVec;
    if (tid < head) f(from + tid, at(from + tid));
    const uint4* v = reinterpret_cast<const uint4*>(q + head);
    const int first = from + head;
    int i = tid;
    for (; i + 3 * threads < vecs; i += 4 * threads) {
      uint4 r[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) r[j] = v[i + j * threads];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < kVec; ++e) f(first + (i + j * threads) * kVec + e, value(r[j], e));
    }
    for (; i < vecs; i += threads) {
      const uint4 r = v[i];
#pragma unroll
      for (int e = 0; e < kVec; ++e) f(first + i * kVec + e, value(r, e));
    }
    const int rest = first + vecs * kVec + tid;
    if (rest < to) f(rest, at(rest));
  }
};

// What turns a logit into a weight.
struct Scale {
  double max, least, per;  // the row's maximum, the least l - max that has weight, log2(e) / T
  bool infinite;           // the maximum is +inf

  __device__ __forceinline__ double below(float l) const {
    if (infinite) return l == __builtin_inff() ? 0.0 : -__builtin_inf();
    return static_cast<double>(l) - max;
  }
  __device__ __forceinline__ bool live(double d) const { return d >= least && d != -__builtin_inf(); }
  // 2^(d per + 44), rounded to a whole number
  __device__ __forceinline__ u64 weight(double d) const {
    const double x = d * per, n = __builtin_rint(x), r = (x - n) * 0.6931471805599453;
    double e = 1.0 / 479001600.0;  // 1/12!; what follows is 2^-52 of the sum at |r| <= ln 2 / 2
    e = __builtin_fma(e, r, 1.0 / 39916800.0);
    e = __builtin_fma(e, r, 1.0 / 3628800.0);
    e = __builtin_fma(e, r, 1.0 / 362880.0);
    e = __builtin_fma(e, r, 1.0 / 40320.0);
    e = __builtin_fma(e, r, 1.0 / 5040.0);
    e = __builtin_fma(e, r, 1.0 / 720.0);
    e = __builtin_fma(e, r, 1.0 / 120.0);
    e = __builtin_fma(e, r, 1.0 / 24.0);
    e = __builtin_fma(e, r, 1.0 / 6.0);
    e = __builtin_fma(e, r, 0.5);
    e = __builtin_fma(e, r, 1.0);
    e = __builtin_fma(e, r, 1.0);
    const u64 pow = static_cast<u64>(static_cast<int>(n) + 44 + 1023) << 52;
    const double whole = __builtin_fma(e, __builtin_bit_cast(double, pow), 0x1p52);
    return __builtin_bit_cast(u64, whole) & 0xfffffffffffffull;
  }
  // bins of equal width in the logarithm, the largest weights in bin 0
  __device__ __forceinline__ int bin(double d) const {
    return min(kBins - 1, static_cast<int>(-d * per * kBinsPerOctave));
  }
};

struct Shared {
  u64 mass[kBins];
  uint32_t count[kBins];
  uint32_t key[kList];
  int32_t index[kList];
  u64 wave_mass[kWaves];
  uint32_t wave_count[kWaves], wave_b[kWaves];
  u64 found_mass;
  uint32_t found_count;
  int found, last, listed;
};

// Inclusive sums over the workgroup's threads, in their order.
__device__ __forceinline__ void block_scan(Shared& s, uint32_t& count, u64& mass, int tid) {
  const int lane = tid & 63, wave = tid >> 6;
#pragma unroll
  for (int by = 1; by < 64; by <<= 1) {
    const uint32_t c = __shfl_up(count, by);
    const u64 m = __shfl_up(mass, by);
    if (lane >= by) count += c, mass += m;
  }
  __syncthreads();  // the places of an earlier scan have been read
  if (lane == 63) s.wave_count[wave] = count, s.wave_mass[wave] = mass;
  __syncthreads();
  for (int w = 0; w < wave; ++w) count += s.wave_count[w], mass += s.wave_mass[w];
}

// The least and largest over the workgroup.
__device__ __forceinline__ void block_range(Shared& s, uint32_t& lo, uint32_t& hi, int tid) {
#pragma unroll
  for (int by = 32; by > 0; by >>= 1) {
    lo = min(lo, static_cast<uint32_t>(__shfl_xor(lo, by)));
    hi = max(hi, static_cast<uint32_t>(__shfl_xor(hi, by)));
  }
  __syncthreads();
  if ((tid & 63) == 0) s.wave_count[tid >> 6] = lo, s.wave_b[tid >> 6] = hi;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) lo = min(lo, s.wave_count[w]), hi = max(hi, s.wave_b[w]);
}

__device__ __forceinline__ void clear_bins(Shared& s, int tid) {
  __syncthreads();
  s.count[tid] = 0, s.mass[tid] = 0;
  __syncthreads();
}

// A cut of the order: the first `count` elements, or those with less than `mass` before them,
// whichever is fewer (each at least one).
struct Target {
  uint32_t count;
  u64 mass;
};

// The bin in which the cut falls, given what lies before bin 0; on return what lies before that bin.
// The last bin that is not empty if the cut lies past all of them.
__device__ __forceinline__ int find_bin(Shared& s, const Target& t, uint32_t& before, u64& mass_before, int tid) {
  const uint32_t own = s.count[tid];
  const u64 own_mass = s.mass[tid];
  uint32_t c = own;
  u64 m = own_mass;
  block_scan(s, c, m, tid);
  c += before, m += mass_before;
  if (tid == 0) s.found = -1;
  __syncthreads();
  // the first bin with which either limit is reached: the bins before it do not reach them
  const bool reached = own && (c >= t.count || m >= t.mass);
  const bool earlier = c - own >= t.count || m - own_mass >= t.mass;
  if (reached && !earlier) s.found = tid, s.found_count = c - own, s.found_mass = m - own_mass;
  __syncthreads();
  const int found = s.found;
  if (found >= 0) before = s.found_count, mass_before = s.found_mass;
  return found;
}

// Keep what has a key above `key`, and of those at it the ones with an index up to `index`.
struct Cut {
  uint32_t key;
  int32_t index;
  u64 mass;  // of what is kept
  __device__ __forceinline__ bool keeps(float l, int i) const {
    const uint32_t k = key_of(l);
    return k > key || (k == key && i <= index);
  }
};

// Where the cut falls in the histogram's bin `bin`, of which before and mass_before lie ahead.
template <typename T>
__device__ Cut resolve(Shared& s, const Row<T>& row, const Scale& scale, const Target& t, int bin,
                       uint32_t before, u64 mass_before, const Cut& inside, int tid) {
  if (tid == 0) s.listed = 0;
  __syncthreads();
  row.each(0, row.n, tid, kThreads, [&](int i, float l) {
    const double d = scale.below(l);
    if (!scale.live(d) || scale.bin(d) != bin || !inside.keeps(l, i)) return;
    const int at = atomicAdd(&s.listed, 1);
    if (at < kList) s.key[at] = key_of(l), s.index[at] = i;
  });
  __syncthreads();
  const int listed = s.listed;
  const bool whole = listed <= kList;
  // f(key, index) of the bin's elements, from the list or from the row
  const auto each = [&](auto f) {
    if (whole) {
      for (int i = tid; i < listed; i += kThreads) f(s.key[i], s.index[i]);
    } else {
      row.each(0, row.n, tid, kThreads, [&](int i, float l) {
        const double d = scale.below(l);
        if (scale.live(d) && scale.bin(d) == bin && inside.keeps(l, i)) f(key_of(l), i);
      });
    }
  };
  const auto value_of = [](uint32_t k) {
    return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
  };
  uint32_t lo = 0xffffffffu, hi = 0;
  each([&](uint32_t k, int) { lo = min(lo, k), hi = max(hi, k); });
  block_range(s, lo, hi, tid);
  uint32_t ties = 0;
  while (true) {  // the range falls to a 1024th each time
    int shift = 0;
    while (((hi - lo) >> shift) >= kBins) ++shift;
    clear_bins(s, tid);
    each([&](uint32_t k, int) {
      if (k < lo || k > hi) return;
      const uint32_t b = (hi - k) >> shift;
      atomicAdd(&s.count[b], 1u);
      atomicAdd(&s.mass[b], scale.weight(scale.below(value_of(k))));
    });
    __syncthreads();
    const int b = find_bin(s, t, before, mass_before, tid);
    ties = s.count[b];
    hi = hi - (static_cast<uint32_t>(b) << shift);
    if (shift == 0) break;
    const uint32_t span = (1u << shift) - 1u;
    lo = hi - lo > span ? hi - span : lo;
    if (lo == hi) break;
  }
  Cut cut;
  cut.key = hi;
  const u64 w = scale.weight(scale.below(value_of(hi)));
  const u64 by_mass = (t.mass - mass_before + w - 1) / w;
  const uint32_t keep = static_cast<uint32_t>(min(static_cast<u64>(min(t.count - before, ties)), max(by_mass, u64{1})));
  cut.mass = mass_before + keep * w;
  cut.index = row.n;
  if (keep < ties) {  // the keep-th smallest index among them
    uint32_t first = 0, last = static_cast<uint32_t>(row.n - 1), passed = 0;
    while (true) {
      int shift = 0;
      while (((last - first) >> shift) >= kBins) ++shift;
      clear_bins(s, tid);
      each([&](uint32_t k, int i) {
        const uint32_t at = static_cast<uint32_t>(i);
        if (k == hi && at >= first && at <= last) atomicAdd(&s.count[(at - first) >> shift], 1u);
      });
      __syncthreads();
      u64 none = 0;
      const int b = find_bin(s, Target{keep, kNoMass}, passed, none, tid);
      first += static_cast<uint32_t>(b) << shift;
      if (shift == 0) break;
      last = min(last, first + (1u << shift) - 1u);
    }
    cut.index = static_cast<int>(first);
  }
  __syncthreads();
  return cut;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs p) {
  __shared__ Shared s;
  const int tid = threadIdx.x, row_id = blockIdx.x;
  const Row<T> row{static_cast<const T*>(p.logits) + row_id * p.stride, p.vocab};
  uint32_t least = 0xffffffffu, most = 0;
  row.each(0, row.n, tid, kThreads, [&](int, float l) { most = max(most, key_of(l)); });
  block_range(s, least, most, tid);
  const float top = __builtin_bit_cast(float, most & 0x80000000u ? most & 0x7fffffffu : ~most);
  if (top == -__builtin_inff()) {
    if (tid == 0) {
      p.tokens[row_id] = -1;
      if (p.logprobs) p.logprobs[row_id] = -__builtin_inff();
    }
    return;
  }
  float temp = p.temperature ? p.temperature[row_id] : 1.0f;
  const bool greedy = !(temp > 0.0f);
  temp = greedy ? 1.0f : fminf(temp, 3.40282347e38f);
  const float min_p = p.min_p ? p.min_p[row_id] : 0.0f;
  const float top_p = p.top_p ? p.top_p[row_id] : 1.0f;
  const int k = greedy ? 1 : p.top_k ? p.top_k[row_id] : 0;
  Scale scale;
  scale.max = top;
  scale.infinite = top == __builtin_inff();
  scale.per = kLog2e / temp;
  scale.least = -kRange * temp;
  if (min_p > 0.0f) scale.least = fmax(scale.least, temp * ::log(static_cast<double>(fminf(min_p, 1.0f))));

  // the histogram, and each part's mass for the draw
  clear_bins(s, tid);
  row.each(0, row.n, tid, kThreads, [&](int, float l) {
    const double d = scale.below(l);
    if (!scale.live(d)) return;
    const int b = scale.bin(d);
    atomicAdd(&s.count[b], 1u);
    atomicAdd(&s.mass[b], scale.weight(d));
  });
  __syncthreads();
  const uint32_t own = s.count[tid];
  const u64 own_mass = s.mass[tid];
  uint32_t live = own;
  u64 total = own_mass;
  block_scan(s, live, total, tid);
  if (tid == kThreads - 1) s.found_count = live, s.found_mass = total;
  __syncthreads();
  live = s.found_count, total = s.found_mass;
  Cut cut{0, row.n, total};
  if (k > 0 && static_cast<uint32_t>(k) < live) {
    const Target t{static_cast<uint32_t>(k), kNoMass};
    uint32_t before = 0;
    u64 mass_before = 0;
    const int b = find_bin(s, t, before, mass_before, tid);
    cut = resolve(s, row, scale, t, b, before, mass_before, cut, tid);
    total = cut.mass;
    s.count[tid] = own, s.mass[tid] = own_mass;
    __syncthreads();
  }
  if (top_p < 1.0f) {
    const double want = static_cast<double>(fmaxf(top_p, 0.0f)) * static_cast<double>(total);
    const u64 mass = max(static_cast<u64>(__builtin_ceil(want)), u64{1});
    const Target t{kNoCount, min(mass, total)};
    uint32_t before = 0;
    u64 mass_before = 0;
    const int b = find_bin(s, t, before, mass_before, tid);
    cut = resolve(s, row, scale, t, b, before, mass_before, cut, tid);
    total = cut.mass;
  }
  // The draw: masses of kParts parts of the row, then of the elements of the part that it falls in.
  const float given = p.u[row_id];
  const double want = given > 0.0f ? static_cast<double>(given) * static_cast<double>(total) : 0.0;
  const auto kept = [&](int i, float l) -> u64 {
    if (!cut.keeps(l, i)) return 0;
    const double d = scale.below(l);
    return scale.live(d) ? scale.weight(d) : 0;
  };
  const int part = ceil_div(row.n, kParts), lane = tid & 63, wave = tid >> 6;
  clear_bins(s, tid);
  for (int i = wave; i < kParts; i += kWaves) {
    u64 m = 0;
    const int from = min(i * part, row.n), to = min(from + part, row.n);
    row.each(from, to, lane, 64, [&](int at, float l) { m += kept(at, l); });
#pragma unroll
    for (int by = 32; by > 0; by >>= 1) m += __shfl_xor(m, by);
    if (lane == 0) s.mass[i] = m;
  }
  __syncthreads();
  uint32_t none = 0;
  const u64 part_mass = s.mass[tid];
  u64 sum = part_mass;
  block_scan(s, none, sum, tid);
  if (tid == 0) s.found = -1, s.last = -1;
  __syncthreads();
  // the first part with more than `want`, or the last one with any mass (u = 1 and its like)
  if (part_mass && static_cast<double>(sum) > want && !(static_cast<double>(sum - part_mass) > want))
    s.found = tid, s.found_mass = sum - part_mass;
  if (part_mass && sum == total) s.last = tid;
  __syncthreads();
  const bool past = s.found < 0;
  const int begin = (past ? s.last : s.found) * part, end = min(begin + part, row.n);
  const u64 ahead = past ? 0 : s.found_mass;
  const int each = ceil_div(part, kThreads), from = begin + tid * each;
  u64 mine = 0;
  for (int i = from; i < min(from + each, end); ++i) mine += kept(i, row.at(i));
  u64 until = mine;
  block_scan(s, none, until, tid);
  if (tid == kThreads - 1) s.found_mass = until;
  __syncthreads();
  const u64 all = s.found_mass;
  // of the threads with mass the one in which the sum passes `want`, or the last
  u64 at = ahead + until - mine;
  const bool here = past ? mine && until == all
                         : mine && static_cast<double>(at + mine) > want && !(static_cast<double>(at) > want);
  if (here) {
    int token = -1;
    for (int i = from; i < min(from + each, end); ++i) {
      const u64 w = kept(i, row.at(i));
      if (!w) continue;
      at += w;
      token = i;
      if (!past && static_cast<double>(at) > want) break;
    }
    p.tokens[row_id] = token;
    if (p.logprobs) {
      const double d = scale.below(row.at(token));
      p.logprobs[row_id] = static_cast<float>(d / temp - ::log(static_cast<double>(total) * 0x1p-44));
    }
  }
}

}  // namespace
}  // namespace pega

using namespace pega;

PEGA_API long long pega_sample_workspace_bytes(int rows, int vocab) {
  return rows <= 0 || vocab <= 0 ? 0 : 16LL * rows;
}

// No reference counterpart here: the reference samples outside the expert path.
PEGA_API int pega_sample_tokens(const void* logits, bool logits_bf16, long long row_stride, int rows,
                                int vocab, const float* uniform, const float* temperature,
                                const int32_t* top_k, const float* top_p, const float* min_p,
                                int32_t* tokens, float* logprobs, void* workspace,
                                long long workspace_bytes, hipStream_t stream) {
  if (rows < 0 || vocab <= 0 || row_stride < vocab)
    return fail(kInvalidValue, "sample_tokens: bad sizes (rows=%d vocab=%d stride=%lld)", rows, vocab, row_stride);
  if (vocab > kMaxVocab) return fail(kNotSupported, "sample_tokens: at most %d tokens, got %d", kMaxVocab, vocab);
  if (rows == 0) return kSuccess;  // empty tensors have no address
  if (!logits || !uniform || !tokens || !workspace) return fail(kInvalidValue, "sample_tokens: null pointer");
  if (workspace_bytes < pega_sample_workspace_bytes(rows, vocab))
    return fail(kInvalidValue, "sample_tokens: a workspace of %lld bytes, %lld needed", workspace_bytes,
                pega_sample_workspace_bytes(rows, vocab));
  if ((reinterpret_cast<uintptr_t>(workspace) & 15u) ||
      (reinterpret_cast<uintptr_t>(logits) & (logits_bf16 ? 1u : 3u)))
    return fail(kNotSupported, "sample_tokens: the workspace must be 16-byte aligned, logits by their type");
  const long long logit_bytes = ((rows - 1) * row_stride + vocab) * (logits_bf16 ? 2 : 4);
  struct Span { const void* p; long long bytes; };
  const Span outs[3] = {{tokens, 4LL * rows}, {logprobs, 4LL * rows}, {workspace, workspace_bytes}};
  const Span ins[6] = {{logits, logit_bytes}, {uniform, 4LL * rows}, {temperature, 4LL * rows},
                       {top_k, 4LL * rows}, {top_p, 4LL * rows}, {min_p, 4LL * rows}};
  for (int o = 0; o < 3; ++o) {
    for (const Span& in : ins)
      if (overlap(outs[o].p, outs[o].bytes, in.p, in.bytes))
        return fail(kInvalidValue, "sample_tokens: an output overlaps an input");
    for (int i = 0; i < o; ++i)
      if (overlap(outs[o].p, outs[o].bytes, outs[i].p, outs[i].bytes))
        return fail(kInvalidValue, "sample_tokens: two outputs overlap");
  }
  const SampleArgs p{logits, row_stride, rows, vocab, uniform, temperature, top_p, min_p, top_k, tokens, logprobs};
  if (logits_bf16) hipLaunchKernelGGL(sample_kernel<uint16_t>, dim3(rows), dim3(kThreads), 0, stream, p);
  else hipLaunchKernelGGL(sample_kernel<float>, dim3(rows), dim3(kThreads), 0, stream, p);
  return launch_status("sample_tokens");
}
