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
// comparison is of exact sums with a share of the whole in 64-bit floating point.  The weights' rounding,
// 2^-45 each, moves a border by V 2^-45 of the sum at most: where nearly all are equal and small, by
// 4.7e-9 with 163840 of them.
//
// No sort.  A histogram of the weights' logarithms (counts and masses in LDS) finds the bin in which
// each cut falls; its elements are listed, and compared with each other or, where they are many,
// narrowed down by histograms of their keys; equal keys are cut by index.  A row is read two or three
// times: for its largest logit, then for the histogram, then for the list and the masses of what is
// kept whole.  Where k is small (its bound: the threads of the first pass) the histogram falls away:
// each thread of the first pass leaves its own largest, the k-th largest of these is a bound below
// which nothing is kept, and what lies above it is listed at once.
//
// What bounds it: the first pass, memory (256 rows of 163840 fp32 logits, 168 MB, 32 us, 5.2 TB/s).
// The others read what the first left in the caches and are bound by the vector units, a chain of 12
// products in 64 bits for each weight (the histogram 40 us of those rows, the third pass 27 us; 14 us
// for the cuts; together 116).  One row is bound by latency alone: launches of 4.3, 9.5 and 7.8 us.
// So a row is split over up to 16 workgroups, of 512 threads as there are bins (of 1024 threads with
// more than 64 registers one fitted a CU).  One workgroup a row for everything took 268 us for one row
// and 317 for 256.  The passes' bodies are loops of few instructions, not unrolled: these kernels are
// short enough for a CU's instruction fetches to show.
#include "common.h"
#include "pega_moe.h"

namespace pega {
namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kBins = kThreads;        // one a thread
// Elements of the cuts' bins kept in LDS.  With 4096 three workgroups fit a CU; with 3200 four do, which is no
// faster (256 rows 112.5 and 113.7 us), and with 2048 some rows are over it (233).  A row over it is gone over by one
// workgroup, element by element: with top-p 0.9 over 163840 normal logits of sigma / T = 0.75 and less, one row takes
// 398 to 441 us (38 with 2.2), 256 rows 721 to 737 (180), and 256 rows with one such among them 621.
constexpr int kList = 4096;
constexpr int kMaxSplit = 16;          // workgroups of a row
constexpr int kMaxParts = 256;         // of a row, whose masses the draw goes over first (a multiple of kMaxSplit)
constexpr int kFlight = 4;             // vectors of a thread in flight
constexpr int kMaxFew = 1024;          // so few fit the list with room for what shares the last one's bin
constexpr int kPairs = kThreads / 4;   // candidates that are compared with each other, by four threads each
constexpr int kWorkgroups = 1024;      // of a launch, where rows are fewer
constexpr int kFewWorkgroups = 256;    // no more than one a CU
constexpr int kMaxRows = 256;          // of a round of launches, which bounds the workspace
constexpr int kMaxVocab = 1 << 19;     // sums of weights: at most 2^63
constexpr double kRange = 28.0;        // smaller weights than e^-28 are zero
constexpr double kLog2e = 1.4426950408889634;
constexpr double kBinsPerOctave = kBins / (kRange * kLog2e + 0.01);

typedef unsigned long long u64;
constexpr u64 kOne = u64{1} << 44;              // the largest logit's weight
constexpr u64 kNoMass = (u64{1} << 63) + kOne;  // more than any sum of weights; one more weight fits on top
static_assert(kNoMass > kMaxVocab * kOne && kNoMass + kOne > kNoMass, "sums of weights");
constexpr uint32_t kNoCount = 0xffffffffu;

struct SampleArgs {
  const void* logits;
  long long stride;  // elements from row to row
  int rows, vocab;
  const float *u, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  int32_t* tokens;
  float* logprobs;
  bool has_temperature, has_top_p, has_min_p, has_top_k;
};

__device__ __forceinline__ float clean(float l) { return l == l ? l : -__builtin_inff(); }

// Floats in the order of their values.
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t b = __builtin_bit_cast(uint32_t, l + 0.0f);  // -0 is 0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// A logit and its index in one number: the larger, the further ahead in the order.
__device__ __forceinline__ u64 place(float l, int i) {
  return static_cast<u64>(key_of(l)) << 32 | (0xffffffffu - static_cast<uint32_t>(i));
}

// A row as vectors of 16 bytes, wherever it starts (the loads need no alignment); the last one reaches back to
// end with the row.  Rows shorter than a vector go element by element.
template <typename T>
struct Row {
  static constexpr int kVec = 16 / static_cast<int>(sizeof(T));
  const T* p;
  int n, vecs;  // elements, vectors

  __device__ __forceinline__ Row(const T* row, int size) : p(row), n(size), vecs(ceil_div(size, kVec)) {}
  static __device__ __forceinline__ float value(uint4 q, int e) {
    if constexpr (sizeof(T) == 4)
      return __builtin_bit_cast(float, e == 0 ? q.x : e == 1 ? q.y : e == 2 ? q.z : q.w);
    const uint32_t w = (e >> 1) == 0 ? q.x : (e >> 1) == 1 ? q.y : (e >> 1) == 2 ? q.z : q.w;
    return e & 1 ? bf_hi(w) : bf_lo(w);
  }
  // Whether a comparison holds for an element of one of the wave's vectors.  By comparisons, which no NaN passes, and
  // by their lane masks: the maximum of a number and a signaling NaN is a NaN, which would hide the numbers beside it,
  // and the compiler makes such a maximum out of comparisons that are joined in a lane.
  template <typename C>
  static __device__ __forceinline__ bool any(uint4 q, C holds) {
    u64 found = 0;
#pragma unroll
    for (int e = 0; e < kVec; ++e) found |= __builtin_amdgcn_ballot_w64(holds(value(q, e)));
    return found != 0;
  }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (sizeof(T) == 4) return clean(p[i]);
    else return clean(bf2f(p[i]));
  }
  __device__ __forceinline__ int start(int v) const { return min(v * kVec, n - kVec); }
  __device__ __forceinline__ uint4 load(int v) const {  // past the last: the last
    uint4 q;
    __builtin_memcpy(&q, p + start(min(v, vecs - 1)), 16);
    return q;
  }
  // The place of this thread's first in the order among the vectors in [from, to), over `threads` threads,
  // each element once.
  __device__ __forceinline__ u64 best(int from, int to, int tid, int threads) const {
    float top = -__builtin_inff();
    int at = -1;
    if (n < kVec) {
      if (from == 0 && tid < n) top = this->at(tid), at = tid;
      return place(top, at);
    }
    for (int v = from + tid; v < to; v += kFlight * threads) {
      uint4 q[kFlight];
#pragma unroll
      for (int j = 0; j < kFlight; ++j) q[j] = load(v + j * threads);
#pragma unroll
      for (int j = 0; j < kFlight; ++j) {
        // seldom passed: later elements of one value are behind it
        if (!any(q[j], [&](float l) { return l > top; })) continue;
        const int vec = v + j * threads, i = start(min(vec, vecs - 1)), own = vec * kVec - i;
#pragma unroll
        for (int e = 0; e < kVec; ++e)
          if (vec < to && e >= own && value(q[j], e) > top) top = value(q[j], e), at = i + e;
      }
    }
    return place(top, at);
  }
  // f(i, l[i]) for the vectors' elements with l >= low (a NaN has not), over `threads` threads with
  // kFlight loads in flight each.  f is there four times, not once for each element in flight.
  // after(base): once for each round of vectors base .. base + threads - 1, by all threads.
  template <typename F, typename A>
  __device__ __forceinline__ void each(int from, int to, int tid, int threads, float low, F f, A after) const {
    if (n < kVec) {
      if (from == 0 && from < to) {
        each_plain(tid, threads, low, f);
        after(from);
      }
      return;
    }
    uint4 q[kFlight];
#pragma unroll
    for (int j = 0; j < kFlight; ++j) q[j] = load(from + tid + j * threads);
#pragma unroll 1
    for (int base = from; base < to; base += threads) {
      const int v = base + tid;
      uint4 now = q[0];
#pragma unroll
      for (int j = 0; j + 1 < kFlight; ++j) q[j] = q[j + 1];
      q[kFlight - 1] = load(v + kFlight * threads);
      if (v < to && any(now, [&](float l) { return l >= low; })) {
        const int first = start(v);
        // the last vector may reach back over the one before, whose elements are not its own
        const int own = v * kVec - first;
        int i = first;
#pragma unroll 1
        for (int w = 0; w < kVec; w += 4) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float l = value(now, e);
            if (l >= low && i + e - first >= own) f(i + e, l);
          }
          i += 4;
          now = make_uint4(now.z, now.w, now.x, now.y);
        }
      }
      after(base);
    }
  }
  // The same, element by element: where speed does not count.
  template <typename F>
  __device__ __forceinline__ void each_plain(int tid, int threads, float low, F f) const {
#pragma unroll 1
    for (int i = tid; i < n; i += threads) {
      const float l = at(i);
      if (l >= low) f(i, l);
    }
  }
};

// 2^r = sum of (r ln 2)^k / k!, for |r| <= 1/2; what follows k = 12 is 2^-52 of the sum.  The
// coefficients stand in scalar registers, made in front of a loop: from vector registers each would be
// moved in front of its product (78 against 98 us for 256 rows of 163840 weights).
struct Powers {
  double c[12] = {0x1.c3bd650fc2986p-36, 0x1.e8cac7351bb25p-32, 0x1.e4cf5158b8ecap-28,
                  0x1.b5253d395e7c4p-24, 0x1.62c0223a5c824p-20, 0x1.ffcbfc588b0c7p-17,
                  0x1.430912f86c787p-13, 0x1.5d87fe78a6731p-10, 0x1.3b2ab6fba4e77p-7,
                  0x1.c6b08d704a0c0p-5, 0x1.ebfbdff82c58fp-3, 0x1.62e42fefa39efp-1};
  __device__ __forceinline__ Powers() {
#pragma unroll
    for (int i = 0; i < 12; ++i) asm("" : "+s"(c[i]));
  }
  __device__ __forceinline__ double of(double r) const {
    double e = c[0];
#pragma unroll
    for (int i = 1; i < 12; ++i) e = __builtin_fma(e, r, c[i]);
    return __builtin_fma(e, r, 1.0);
  }
};

// What turns a logit into a weight.
struct Scale {
  // the row's maximum, the least l - max that has weight, log2(e) / T, and bins for a unit of l
  double max, least, per, bins;
  bool infinite;           // the maximum is +inf

  // l - max; of an infinite maximum 0 and, for all else, -inf
  __device__ __forceinline__ double below(float l) const { return __builtin_fmin(static_cast<double>(l) - max, 0.0); }
  __device__ __forceinline__ bool live(double d) const { return d >= least; }  // (least is finite)
  // 2^(d per + 44), rounded to a whole number
  __device__ __forceinline__ u64 weight(double d, const Powers& powers = Powers()) const {
    const double x = d * per, n = __builtin_rint(x), r = x - n;
    const double e = powers.of(r);
    const u64 pow = static_cast<u64>(static_cast<int>(n) + 44 + 1023) << 52;
    const double whole = __builtin_fma(e, __builtin_bit_cast(double, pow), 0x1p52);
    return __builtin_bit_cast(u64, whole) & 0xfffffffffffffull;
  }
  // bins of equal width in the logarithm, the largest weights in bin 0
  __device__ __forceinline__ double position(double d) const { return -d * bins; }
  __device__ __forceinline__ int bin(double d) const { return min(kBins - 1, static_cast<int>(position(d))); }
  // above every d of a bin, below every one
  __device__ __forceinline__ double inner(int b) const { return -b / bins * (1 - 0x1p-30); }
  __device__ __forceinline__ double edge(int b) const { return -(b + 1) / bins * (1 + 0x1p-30); }
  // A float below every logit l with below(l) >= d, so that what it leaves out is never live, and one above all with
  // below(l) < d.  The first leaves room for the rounding of l - max, up to 2^-53 |d|, beside which max + d may be next
  // to nothing; the sum's own rounding is relative to it.
  __device__ __forceinline__ float bound(double d) const {
    if (infinite) return __builtin_inff();
    const float f = static_cast<float>(max + d - (__builtin_fabs(max) + __builtin_fabs(d)) * 0x1p-50);
    return f - __builtin_fabsf(f) * 0x1p-22f - 0x1p-126f;
  }
  __device__ __forceinline__ float over(double d) const {
    const float f = static_cast<float>(max + d);
    return f + __builtin_fabsf(f) * 0x1p-22f + 0x1p-126f;
  }
};

struct Shared {
  u64 mass[kBins];  // the row's histogram
  uint32_t count[kBins];
  __align__(16) u64 fine_mass[kBins];  // a narrower one inside a bin of it
  uint32_t fine_count[kBins];
  u64 part[kMaxParts];  // masses of the row's parts
  uint32_t key[kList];  // elements of the bins in which the cuts fall
  int32_t index[kList];
  u64 wave_mass[16];
  uint32_t wave_count[16];
  u64 found_mass;
  uint32_t found_count;
  int found, last, listed;
};

// Lane moves without an "old" operand; lanes that nothing reaches, or outside the rows of the mask, get 0.
template <int kCtrl, int kRows>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kCtrl, kRows, 0xF, false));
}
template <int kCtrl, int kRows = 0xF>
__device__ __forceinline__ u64 dpp64(u64 v) {
  return static_cast<u64>(dpp<kCtrl, kRows>(static_cast<uint32_t>(v >> 32))) << 32 | dpp<kCtrl, kRows>(static_cast<uint32_t>(v));
}
// Inclusive sums over 16 lanes, over the wave's 64.
__device__ __forceinline__ u64 scan16(u64 v) {
  v += dpp64<0x111>(v);  // row_shr:1, 2, 4, 8
  v += dpp64<0x112>(v);
  v += dpp64<0x114>(v);
  return v + dpp64<0x118>(v);
}
__device__ __forceinline__ uint32_t scan16(uint32_t v) {
  v += dpp<0x111, 0xF>(v);
  v += dpp<0x112, 0xF>(v);
  v += dpp<0x114, 0xF>(v);
  return v + dpp<0x118, 0xF>(v);
}
__device__ __forceinline__ u64 scan64(u64 v) {
  v = scan16(v);
  v += dpp64<0x142, 0xA>(v);         // row_bcast:15 into rows 1 and 3
  return v + dpp64<0x143, 0xC>(v);   // row_bcast:31 into rows 2 and 3
}
__device__ __forceinline__ uint32_t scan64(uint32_t v) {
  v = scan16(v);
  v += dpp<0x142, 0xA>(v);
  return v + dpp<0x143, 0xC>(v);
}
__device__ __forceinline__ u64 lane64(u64 v, int lane) {
  const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(v)), lane));
  const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(v >> 32)), lane));
  return static_cast<u64>(hi) << 32 | lo;
}

// Inclusive sums over the workgroup's threads, in their order.
__device__ __forceinline__ void block_scan(Shared& s, uint32_t& count, u64& mass, int tid) {
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  count = scan64(count), mass = scan64(mass);
  __syncthreads();  // the places of an earlier scan have been read
  if (lane == 63) s.wave_count[wave] = count, s.wave_mass[wave] = mass;
  __syncthreads();
  const uint32_t c = scan16(s.wave_count[lane & 15]);
  const u64 m = scan16(s.wave_mass[lane & 15]);
  if (wave > 0) {
    count += static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(c), wave - 1));
    mass += lane64(m, wave - 1);
  }
}

// The largest over the workgroup, in each thread.
__device__ __forceinline__ u64 block_max(u64* wave_max, u64 v, int tid) {
  const auto max16 = [](u64 x) {
    x = max(x, dpp64<0xB1>(x));     // quad_perm [1,0,3,2]
    x = max(x, dpp64<0x4E>(x));     // quad_perm [2,3,0,1]
    x = max(x, dpp64<0x141>(x));    // row_half_mirror
    return max(x, dpp64<0x140>(x)); // row_mirror
  };
  v = max16(v);
  v = max(max(lane64(v, 0), lane64(v, 16)), max(lane64(v, 32), lane64(v, 48)));
  __syncthreads();
  if ((tid & 63) == 0) wave_max[tid >> 6] = v;
  __syncthreads();
  return lane64(max16(wave_max[tid & (kWaves - 1)]), 0);
}

// A cut of the order: the first `count` elements, or those with less than `mass` before them,
// whichever is fewer (each at least one).
struct Target {
  uint32_t count;
  u64 mass;
};

// A histogram's bin of this thread, and the sums up to and with it.
struct Bin {
  uint32_t own, count;
  u64 own_mass, mass;
};
__device__ __forceinline__ Bin scan_bins(Shared& s, const uint32_t* count, const u64* mass, int tid) {
  Bin b{count[tid], count[tid], mass[tid], mass[tid]};
  block_scan(s, b.count, b.mass, tid);
  return b;
}

// The bin in which the cut falls, given what lies before bin 0; on return what lies before that bin.  -1 if
// the bins do not reach it.
__device__ __forceinline__ int find_bin(Shared& s, const Bin& bin, const Target& t, uint32_t& before,
                                        u64& mass_before, int tid) {
  const uint32_t c = bin.count + before;
  const u64 m = bin.mass + mass_before;
  __syncthreads();  // what an earlier call found has been read
  if (tid == 0) s.found = -1;
  __syncthreads();
  const bool reached = bin.own && (c >= t.count || m >= t.mass);
  const bool earlier = c - bin.own >= t.count || m - bin.own_mass >= t.mass;
  if (reached && !earlier) s.found = tid, s.found_count = c - bin.own, s.found_mass = m - bin.own_mass;
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
  __device__ __forceinline__ bool keeps(uint32_t k, int i) const {
    return k > key || (k == key && i <= index);
  }
};

// What a row asks for, and what its largest logit makes of that.
struct Request {
  Scale scale;
  double temp;
  float top_p, u;
  int k;        // 0: all
  bool none;    // no logit above -inf
  bool first;   // the first of the order alone
  bool few;     // a small k: all that its cut leaves is listed without a histogram of the row
  __device__ __forceinline__ bool cuts() const { return k > 0 || top_p < 1.0f; }
  __device__ __forceinline__ bool settled() const { return none || first; }
  // whether scan leaves nothing but the draw
  __device__ __forceinline__ bool scanned() const { return settled() || few || !cuts(); }
};

__device__ __forceinline__ float value_of(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// splits: of the row
__device__ __forceinline__ Request request(const SampleArgs& p, int row, u64 best, int splits) {
  Request q;
  const float top = value_of(static_cast<uint32_t>(best >> 32));
  // (loads side by side: a missing one's pointer is u's)
  const float temp = p.has_temperature ? p.temperature[row] : 1.0f;
  const float min_p = p.has_min_p ? p.min_p[row] : 0.0f;
  const bool greedy = !(temp > 0.0f);
  q.k = greedy ? 1 : p.has_top_k ? max(p.top_k[row], 0) : 0;
  q.first = q.k == 1;
  q.few = q.k > 0 && q.k <= min(kMaxFew, splits * (kThreads / 2));
  q.none = top == -__builtin_inff();
  q.top_p = p.has_top_p ? p.top_p[row] : 1.0f;
  q.u = p.u[row];
  q.temp = greedy ? 1.0 : static_cast<double>(fminf(temp, 3.40282347e38f));
  q.scale.max = top;
  q.scale.infinite = top == __builtin_inff();
  q.scale.per = kLog2e / q.temp;
  q.scale.bins = q.scale.per * kBinsPerOctave;
  q.scale.least = -kRange * q.temp;
  if (min_p > 0.0f)
    q.scale.least = fmax(q.scale.least, q.temp * ::log(static_cast<double>(fminf(min_p, 1.0f))));
  return q;
}

__device__ __forceinline__ void write(const SampleArgs& p, int row, int token, float logprob) {
  p.tokens[row] = token;
  if (p.logprobs) p.logprobs[row] = logprob;
}

// One element's share of the histogram.
__device__ __forceinline__ void count_in(Shared& s, const Scale& scale, float l, const Powers& powers) {
  const double d = scale.below(l);
  if (!scale.live(d)) return;
  const int b = scale.bin(d);
  atomicAdd(&s.count[b], 1u);
  atomicAdd(&s.mass[b], scale.weight(d, powers));
}

// The histogram of vectors [from, to).
template <typename R>
__device__ __forceinline__ void histogram(Shared& s, const R& row, const Scale& scale, int from,
                                          int to, int tid) {
  s.count[tid] = 0, s.mass[tid] = 0;
  __syncthreads();
  const Powers powers;
  row.each(from, to, tid, kThreads, scale.bound(scale.least),
           [&](int, float l) { count_in(s, scale, l, powers); }, [](int) {});
  __syncthreads();
}

// Which bins the cuts fall in.
struct Plan {
  uint32_t live;    // elements with weight
  u64 total;        // and their mass
  bool by_k, by_p;  // cuts that leave something out
  int sure;         // bins before it are kept whole
  int k_bin, p_first, p_last;  // of the cuts, -1 without one; the p cut's within a range
  uint32_t candidates;         // elements of those bins
  uint32_t k_before, p_before;  // elements and masses ahead of k_bin and of p_last
  u64 k_mass, p_mass;
  __device__ __forceinline__ bool has(int b) const { return b == k_bin || (b >= p_first && b <= p_last); }
};

__device__ __forceinline__ Plan no_plan() { return Plan{0, 0, false, false, kBins, -1, -1, -2, 0, 0, 0, 0, 0}; }

__device__ __forceinline__ u64 p_target(float p, u64 total) {
  const double want = static_cast<double>(fmaxf(p, 0.0f)) * static_cast<double>(total);
  return min(max(static_cast<u64>(__builtin_ceil(want)), u64{1}), total);
}

__device__ __forceinline__ Plan make_plan(Shared& s, const Request& q, const Bin& bin, int tid) {
  Plan plan = no_plan();
  __syncthreads();
  if (tid == kThreads - 1) s.found_count = bin.count, s.found_mass = bin.mass;
  __syncthreads();
  plan.live = s.found_count, plan.total = s.found_mass;
  plan.by_k = q.k > 0 && static_cast<uint32_t>(q.k) < plan.live;
  plan.by_p = q.top_p < 1.0f;
  u64 least = plan.total, most = plan.total;  // what the k cut leaves
  uint32_t before = 0;
  if (plan.by_k) {
    least = 0;
    plan.k_bin = find_bin(s, bin, Target{static_cast<uint32_t>(q.k), kNoMass}, before, least, tid);
    most = least + s.mass[plan.k_bin];
    plan.k_before = before, plan.k_mass = least;
    plan.sure = plan.k_bin;
    plan.candidates = s.count[plan.k_bin];
  }
  if (plan.by_p) {
    before = 0;
    u64 mass_before = 0;
    plan.p_last = find_bin(s, bin, Target{kNoCount, p_target(q.top_p, most)}, before, mass_before, tid);
    const uint32_t until = before + s.count[plan.p_last];
    plan.p_before = before, plan.p_mass = mass_before;
    if (plan.by_k) {
      before = 0, mass_before = 0;
      plan.p_first = find_bin(s, bin, Target{kNoCount, p_target(q.top_p, max(least, u64{1}))}, before, mass_before, tid);
    } else {
      plan.p_first = plan.p_last;
    }
    plan.sure = plan.p_first;
    plan.candidates = until - before + (plan.k_bin > plan.p_last ? s.count[plan.k_bin] : 0u);
  }
  return plan;
}

// The plan of a row with a small k.  `keys(i)` for i < n are the largest of disjoint parts of the row, so the
// k-th largest of them is no larger than the k-th largest logit: all bins down to its bin are listed.
template <typename K>
__device__ __forceinline__ Plan few_plan(Shared& s, const Request& q, int n, const K& keys, int tid) {
  s.count[tid] = 0, s.mass[tid] = 0;
  __syncthreads();
#pragma unroll 1
  for (int i = 0; i < n; i += 8) {
    uint32_t k[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) k[j] = keys(min(i + j, n - 1));  // in flight together
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const double d = q.scale.below(value_of(k[j]));
      if (i + j < n && q.scale.live(d)) atomicAdd(&s.count[q.scale.bin(d)], 1u);
    }
  }
  __syncthreads();
  uint32_t before = 0;
  u64 none = 0;
  const int b = find_bin(s, scan_bins(s, s.count, s.mass, tid), Target{static_cast<uint32_t>(q.k), kNoMass}, before,
                         none, tid);
  Plan plan = no_plan();
  plan.by_p = q.top_p < 1.0f;
  plan.sure = 0;
  plan.p_first = 0, plan.p_last = b < 0 ? kBins - 1 : b;  // fewer than k parts with weight: everything that has any
  return plan;
}

// Of the parts first .. end - 1, `part` vectors each, the elements of the cuts' bins into the list, and the
// masses of what lies before those bins.
template <typename R>
__device__ __forceinline__ void pick(Shared& s, const R& row, const Scale& scale, const Plan& plan,
                                     int part, int first, int end, int tid) {
  const int lane = tid & 63, wave = tid >> 6;
  __syncthreads();
  if (tid == 0) s.listed = 0;
  __syncthreads();
  const bool gather = plan.candidates <= kList, all = plan.sure == kBins;
  const int lowest = all ? kBins - 1 : max(plan.k_bin, plan.p_last);
  const float low = fmaxf(scale.bound(scale.least), scale.bound(scale.edge(lowest)));
  // a wave's parts in one run, so that its loads stay in flight from one to the next
  const int each_wave = ceil_div(end - first, kWaves), mine = first + wave * each_wave;
  const int from = mine * part, to = min(min(mine + each_wave, end) * part, row.vecs);
  if (lane < each_wave && mine + lane < end) s.part[mine + lane] = 0;
  // from here on a logit is surely in the bins that are kept whole
  const float whole = all ? scale.over(scale.least) : plan.sure == 0 ? __builtin_nanf("") : scale.over(scale.inner(plan.sure));
  u64 m = 0;
  const Powers powers;
  row.each(from, to, lane, 64, low, [&](int at, float l) {
    const double d = scale.below(l);
    if (l >= whole) {
      m += scale.weight(d, powers);
      return;
    }
    if (!scale.live(d)) return;
    const int b = scale.bin(d);
    if (b < plan.sure) {
      m += scale.weight(d, powers);
    } else if (gather && plan.has(b)) {
      const int to_list = atomicAdd(&s.listed, 1);
      if (to_list < kList) s.key[to_list] = key_of(l), s.index[to_list] = at;
    }
  }, [&](int base) {
    if ((base + 64 - from) % part != 0 && base + 64 < to) return;
    const u64 sum = scan64(m);
    if (lane == 63) s.part[base / part] = sum;
    m = 0;
  });
  __syncthreads();
}

// Where a cut falls among n <= kPairs elements of which mine() are meant: each against all others, four
// threads to one, a fourth of them each.
template <typename M>
__device__ __forceinline__ Cut resolve_pairs(Shared& s, const uint32_t* key, const int32_t* index, int n, const M& mine,
                                             const Scale& scale, const Target& t, uint32_t before, u64 mass_before,
                                             int tid) {
  const int own = tid >> 2, quarter = tid & 3;
  const uint32_t k = key[min(own, n - 1)];
  const int i = index[min(own, n - 1)];
  const bool ours = own < n && mine(k, i);
  const u64 at = ours ? place(value_of(k), i) : 0;  // 0: not meant, or past the last: ahead of nothing
  const u64 w = ours ? scale.weight(scale.below(value_of(k))) : 0;
  __syncthreads();
  if (quarter == 0) s.fine_mass[2 * own] = at, s.fine_mass[2 * own + 1] = w;
  __syncthreads();
  uint32_t c = 0;
  u64 m = 0;
  const int n4 = (n + 3) >> 2;
#pragma unroll 8
  for (int j = 0; j < n4; ++j) {
    const ulonglong2 other = *reinterpret_cast<const ulonglong2*>(&s.fine_mass[2 * (4 * j + quarter)]);
    const bool ahead = other.x > at;
    c += ahead ? 1u : 0u, m += ahead ? other.y : 0;
  }
  c += dpp<0xB1, 0xF>(c), m += dpp64<0xB1>(m);
  c += dpp<0x4E, 0xF>(c), m += dpp64<0x4E>(m);
  before += c, mass_before += m;
  if (ours && quarter == 0 && before < t.count && mass_before < t.mass &&
      (before + 1 >= t.count || mass_before + w >= t.mass))
    s.found = own, s.found_mass = mass_before + w;
  __syncthreads();
  const Cut cut{key[s.found], index[s.found], s.found_mass};
  __syncthreads();
  return cut;
}

// Where a cut falls in bin `bin` (-1: among all candidates), of which before and mass_before lie ahead.  each(f) calls f(key, index)
// for the candidates, `listed` of them from the list (more than it holds: from the row).
template <typename E>
__device__ Cut resolve(Shared& s, const E& each, int listed, const Scale& scale, const Target& t, int bin,
                       uint32_t before, u64 mass_before, const Cut& inside, int tid) {
  const auto mine = [&](uint32_t k, int i) {
    return (bin < 0 || scale.bin(scale.below(value_of(k))) == bin) && inside.keeps(k, i);
  };
  if (listed <= kPairs)
    return resolve_pairs(s, s.key, s.index, listed, mine, scale, t, before, mass_before, tid);
  // the bin in 512 steps of its logarithm (all candidates: by their bins), and the elements of the one step
  const auto step_of = [&](uint32_t k) {
    const double d = scale.below(value_of(k));
    return bin < 0 ? scale.bin(d) : min(kBins - 1, max(0, static_cast<int>((scale.position(d) - bin) * kBins)));
  };
  __syncthreads();
  s.fine_count[tid] = 0, s.fine_mass[tid] = 0;
  if (tid == 0) s.last = 0;
  __syncthreads();
  each([&](uint32_t k, int i) {
    if (!mine(k, i)) return;
    const int b = step_of(k);
    atomicAdd(&s.fine_count[b], 1u);
    atomicAdd(&s.fine_mass[b], scale.weight(scale.below(value_of(k))));
  });
  __syncthreads();
  const int step = find_bin(s, scan_bins(s, s.fine_count, s.fine_mass, tid), t, before, mass_before, tid);
  const int left = static_cast<int>(s.fine_count[step]);
  __syncthreads();
  if (left <= kPairs) {
    uint32_t* key = s.fine_count;
    int32_t* index = reinterpret_cast<int32_t*>(s.fine_count + kPairs);
    each([&](uint32_t k, int i) {
      if (!mine(k, i) || step_of(k) != step) return;
      const int at = atomicAdd(&s.last, 1);
      key[at] = k, index[at] = i;
    });
    __syncthreads();
    return resolve_pairs(s, key, index, left, [](uint32_t, int) { return true; }, scale, t, before, mass_before, tid);
  }
  // many equal or nearly so
  Cut cut;
  u64 up = 0, down = 0;
  each([&](uint32_t k, int i) {
    if (mine(k, i) && step_of(k) == step) up = max(up, static_cast<u64>(k)), down = max(down, static_cast<u64>(~k));
  });
  uint32_t hi = static_cast<uint32_t>(block_max(s.wave_mass, up, tid));
  uint32_t lo = ~static_cast<uint32_t>(block_max(s.wave_mass, down, tid));
  uint32_t ties = 0;
  while (true) {  // the range falls to a 512th each time
    int shift = 0;
    while (((hi - lo) >> shift) >= kBins) ++shift;
    __syncthreads();
    s.fine_count[tid] = 0, s.fine_mass[tid] = 0;
    __syncthreads();
    each([&](uint32_t k, int i) {
      if (k < lo || k > hi || !mine(k, i)) return;  // (of this step: lo and hi are)
      const uint32_t b = (hi - k) >> shift;
      atomicAdd(&s.fine_count[b], 1u);
      atomicAdd(&s.fine_mass[b], scale.weight(scale.below(value_of(k))));
    });
    __syncthreads();
    const int b = find_bin(s, scan_bins(s, s.fine_count, s.fine_mass, tid), t, before, mass_before, tid);
    ties = s.fine_count[b];
    hi = hi - (static_cast<uint32_t>(b) << shift);
    if (shift == 0) break;
    const uint32_t span = (1u << shift) - 1u;
    lo = hi - lo > span ? hi - span : lo;
  }
  cut.key = hi;
  const u64 w = scale.weight(scale.below(value_of(hi)));
  const u64 by_mass = (t.mass - mass_before + w - 1) / w;
  const uint32_t keep = static_cast<uint32_t>(min(static_cast<u64>(min(t.count - before, ties)), max(by_mass, u64{1})));
  cut.mass = mass_before + keep * w;
  cut.index = 0x7fffffff;
  if (keep < ties) {  // the keep-th smallest index among them
    uint32_t first = 0, last = kMaxVocab - 1, passed = 0;
    while (true) {
      int shift = 0;
      while (((last - first) >> shift) >= kBins) ++shift;
      __syncthreads();
      s.fine_count[tid] = 0, s.fine_mass[tid] = 0;
      __syncthreads();
      each([&](uint32_t k, int i) {
        const uint32_t at = static_cast<uint32_t>(i);
        if (k == hi && at >= first && at <= last && inside.keeps(k, i)) atomicAdd(&s.fine_count[(at - first) >> shift], 1u);
      });
      __syncthreads();
      u64 none = 0;
      const int b = find_bin(s, scan_bins(s, s.fine_count, s.fine_mass, tid), Target{keep, kNoMass}, passed, none, tid);
      first += static_cast<uint32_t>(b) << shift;
      if (shift == 0) break;
      last = first + (1u << shift) - 1u;
    }
    cut.index = static_cast<int>(first);
  }
  __syncthreads();
  return cut;
}

// A row whose candidates are too many for the list, by one workgroup from its histogram on.
template <typename R>
__device__ __forceinline__ void again(Shared& s, const R& row, const Request& q, Plan& plan, Bin& bin, int part,
                                   int parts, int tid) {
  const float low = q.scale.bound(q.scale.least);
  s.count[tid] = 0, s.mass[tid] = 0;
  if (tid < parts) s.part[tid] = 0;
  __syncthreads();
  row.each_plain(tid, kThreads, low, [&](int, float l) { count_in(s, q.scale, l, Powers()); });
  __syncthreads();
  bin = scan_bins(s, s.count, s.mass, tid);
  plan = make_plan(s, q, bin, tid);
  if (tid == 0) s.listed = 0;
  __syncthreads();
  row.each_plain(tid, kThreads, low, [&](int i, float l) {
    const double d = q.scale.below(l);
    if (!q.scale.live(d)) return;
    const int b = q.scale.bin(d);
    if (b < plan.sure) {
      atomicAdd(&s.part[i / (part * R::kVec)], q.scale.weight(d));
    } else if (plan.has(b)) {
      const int at = atomicAdd(&s.listed, 1);
      if (at < kList) s.key[at] = key_of(l), s.index[at] = i;
    }
  });
  __syncthreads();
}

// The cuts and the draw, once the histogram, the list and the parts' masses are there.
template <typename R>
__device__ __forceinline__ void finish(Shared& s, const SampleArgs& p, int row_id, const R& row, const Request& q,
                                       Plan plan, Bin bin, int part, int parts, int tid) {
  const Scale& scale = q.scale;
  const bool few = q.few && plan.candidates <= kList;
  // (fewer than k listed are all that have weight; k or more may not be)
  if (few) plan.by_k = plan.candidates >= static_cast<uint32_t>(q.k);
  else if (q.few) again(s, row, q, plan, bin, part, parts, tid);
  const int listed = static_cast<int>(plan.candidates);
  const auto each = [&](auto f) {
    // one loop for both, so that f is there once
    const bool list = listed <= kList;
#pragma unroll 1
    for (int i = tid; i < (list ? listed : row.n); i += kThreads) {
      uint32_t k;
      int at = i;
      if (list) {
        k = s.key[i], at = s.index[i];
      } else {
        const float l = row.at(i);
        const double d = scale.below(l);
        if (!scale.live(d) || !plan.has(scale.bin(d))) continue;
        k = key_of(l);
      }
      f(k, at);
    }
  };
  Cut cut{0, 0x7fffffff, plan.total};
#pragma unroll 1
  for (int which = plan.by_k ? 0 : 1; which < (plan.by_p ? 2 : 1); ++which) {  // the k cut, the p cut
    const bool pairs = few && plan.by_k && listed <= kPairs;  // the k cut has summed up what it leaves
    if (which == 1 && few && !pairs) {  // the masses of what is left
      __syncthreads();
      s.count[tid] = 0, s.mass[tid] = 0;
      __syncthreads();
      each([&](uint32_t k, int i) {
        if (cut.keeps(k, i)) count_in(s, scale, value_of(k), Powers());
      });
      __syncthreads();
      bin = scan_bins(s, s.count, s.mass, tid);
      if (tid == kThreads - 1) s.found_mass = bin.mass;
      __syncthreads();
      cut.mass = s.found_mass;
    }
    const Target t = which == 0 ? Target{static_cast<uint32_t>(q.k), kNoMass} : Target{kNoCount, p_target(q.top_p, cut.mass)};
    uint32_t before = which == 0 ? plan.k_before : plan.p_before;
    u64 mass_before = which == 0 ? plan.k_mass : plan.p_mass;
    int b = which == 0 ? plan.k_bin : plan.p_last;  // (few: -1, nothing ahead)
    if (which == 1 && (few || plan.by_k)) {
      before = 0, mass_before = 0;
      b = pairs ? -1 : find_bin(s, bin, t, before, mass_before, tid);
    }
    cut = resolve(s, each, listed, scale, t, b, before, mass_before, cut, tid);
  }
  if (plan.sure < kBins) {
    each([&](uint32_t k, int i) {
      if (!cut.keeps(k, i)) return;
      const double d = scale.below(value_of(k));
      if (scale.bin(d) >= plan.sure) atomicAdd(&s.part[i / (part * R::kVec)], scale.weight(d));
    });
  }
  __syncthreads();
  // the first part with which the sum passes u times the whole, or the last one with any mass
  uint32_t none = 0;
  const u64 part_mass = tid < parts ? s.part[tid] : 0;
  u64 sum = part_mass;
  block_scan(s, none, sum, tid);
  if (tid == kThreads - 1) s.found_mass = sum;
  if (tid == 0) s.found = -1;
  __syncthreads();
  const u64 total = s.found_mass;
  const double want = q.u > 0.0f ? static_cast<double>(q.u) * static_cast<double>(total) : 0.0;
  const auto passes = [&](u64 v) { return static_cast<double>(v) > want; };
  if (part_mass && passes(sum) && !passes(sum - part_mass)) s.found = tid;
  if (part_mass && sum == total) s.last = tid;
  __syncthreads();
  const bool past = s.found < 0;
  const int chosen = past ? s.last : s.found;
  if (tid == chosen) s.found_mass = sum - part_mass;
  // its elements in index order, `span` to a thread
  const int size = part * R::kVec, begin = chosen * size, end = min(begin + size, row.n);
  const int span = ceil_div(size, kThreads), from = begin + tid * span, to = min(from + span, end);
  const auto kept = [&](int i) -> u64 {
    const float l = row.at(i);
    const double d = scale.below(l);
    return cut.keeps(key_of(l), i) && scale.live(d) ? scale.weight(d) : 0;
  };
  u64 mine = 0;
  for (int i = from; i < to; ++i) mine += kept(i);
  u64 until = mine;
  block_scan(s, none, until, tid);
  until += s.found_mass;
  const u64 chosen_end = s.part[chosen] + s.found_mass;
  if (mine && (past ? until == chosen_end : passes(until) && !passes(until - mine))) {
    u64 at = until - mine;
    int token = -1;
    for (int i = from; i < to; ++i) {
      const u64 w = kept(i);
      if (!w) continue;
      at += w;
      token = i;
      if (!past && passes(at)) break;
    }
    write(p, row_id, token,
          static_cast<float>(scale.below(row.at(token)) / q.temp - ::log(static_cast<double>(total) * 0x1p-44)));
  }
}

template <typename T>
__device__ __forceinline__ Row<T> row_of(const SampleArgs& p, int row) {
  return Row<T>(static_cast<const T*>(p.logits) + row * p.stride, p.vocab);
}

__device__ __forceinline__ void write_settled(const SampleArgs& p, const Request& q, int row, u64 best) {
  if (q.none) write(p, row, -1, -__builtin_inff());
  else write(p, row, static_cast<int>(0xffffffffu - static_cast<uint32_t>(best)), 0.0f);
}

// Several workgroups (splits) a row, in three launches or four:
//   best   the first of the order in each split, and each thread's largest
//   scan   rows with a small k: the list; rows without cuts: the parts' masses; others: the histogram
//   pick   those others: the list and the parts' masses
//   draw   a workgroup a row: the cuts and the draw
// What they hand on, for each row:
struct Hand {
  u64 best[kMaxSplit];
  Request request;  // from scan on
  Plan plan;
  uint32_t listed, done;  // elements in the list, workgroups of the draw that have listed theirs
  u64 part[kMaxParts];
  uint32_t key[kList];
  int32_t index[kList];
};
struct Histogram {  // of each split; before scan its threads' largest keys
  u64 mass[kBins];
  uint32_t count[kBins];
};
struct SplitArgs {
  SampleArgs p;
  Hand* hand;
  Histogram* hist;
  int splits, part, parts;  // parts: of the row, a multiple of splits
};

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_best_kernel(SplitArgs a) {
  __shared__ u64 wave_max[kWaves];  // (all that it needs: with Shared 114.4 us for 256 rows, without 112.5)
  const int tid = threadIdx.x, row_id = blockIdx.y, split = blockIdx.x;
  const Row<T> row = row_of<T>(a.p, row_id);
  const int per = a.parts / a.splits * a.part;
  const int from = split * per, to = min(from + per, row.vecs);
  const u64 own = row.best(from, to, tid, kThreads);
  a.hist[static_cast<long long>(row_id) * a.splits + split].count[tid] = static_cast<uint32_t>(own >> 32);
  const u64 best = block_max(wave_max, own, tid);
  Hand& h = a.hand[row_id];
  if (tid == 0) {
    h.best[split] = best;
    if (split == 0) h.listed = 0, h.done = 0;
  }
}

__device__ __forceinline__ u64 best_of(const Hand& h, int splits) {
  u64 best = 0;
#pragma unroll
  for (int i = 0; i < kMaxSplit; ++i) best = max(best, h.best[min(i, splits - 1)]);
  return best;
}

// Between workgroups of a launch: device-coherent (the L2 is per XCD).
template <typename V>
__device__ __forceinline__ void store_coherent(V* p, V v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename V>
__device__ __forceinline__ V load_coherent(const V* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// A split's share of the list and of the parts' masses.
template <typename T>
__device__ __forceinline__ void hand_over(Shared& s, const SplitArgs& a, Hand& hand, const Row<T>& row, const Request& q,
                                          const Plan& plan, int split, int splits, int tid) {
  const int per = a.parts / splits, first = split * per;
  pick(s, row, q.scale, plan, a.part, first, first + per, tid);
  if (tid < per) store_coherent(&hand.part[first + tid], s.part[first + tid]);
  const int listed = s.listed;
  if (listed == 0) return;
  if (tid == 0) s.last = static_cast<int>(atomicAdd(&hand.listed, static_cast<uint32_t>(listed)));
  __syncthreads();
  for (int i = tid; i < min(listed, kList) && s.last + i < kList; i += kThreads) {
    store_coherent(&hand.key[s.last + i], s.key[i]);
    store_coherent(&hand.index[s.last + i], s.index[i]);
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_scan_kernel(SplitArgs a) {
  __shared__ Shared s;
  const int tid = threadIdx.x, row_id = blockIdx.y, split = blockIdx.x;
  const Row<T> row = row_of<T>(a.p, row_id);
  Hand& hand = a.hand[row_id];
  const u64 best = best_of(hand, a.splits);
  const Request q = request(a.p, row_id, best, a.splits);
  const bool writes = split == 0 && tid == 0;
  if (writes) hand.request = q;
  if (q.settled()) {
    if (writes) write_settled(a.p, q, row_id, best);
    return;
  }
  Histogram* h = a.hist + static_cast<long long>(row_id) * a.splits;
  if (q.cuts() && !q.few) {
    const int per = a.parts / a.splits * a.part;
    const int from = split * per, to = min(from + per, row.vecs);
    histogram(s, row, q.scale, from, to, tid);
    h[split].count[tid] = s.count[tid], h[split].mass[tid] = s.mass[tid];
    return;
  }
  const Plan plan = q.few ? few_plan(s, q, a.splits, [&](int i) { return h[i].count[tid]; }, tid) : no_plan();
  if (writes) hand.plan = plan;
  hand_over(s, a, hand, row, q, plan, split, a.splits, tid);
}

// The row's histogram, and the plan that follows from it.
__device__ __forceinline__ Plan planned(Shared& s, const SplitArgs& a, int row_id, const Request& q, Bin& bin,
                                        int tid) {
  const Histogram* h = a.hist + static_cast<long long>(row_id) * a.splits;
  uint32_t c = 0;
  u64 m = 0;
#pragma unroll 1
  for (int i = 0; i < a.splits; i += 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // four in flight
      const Histogram& from = h[min(i + j, a.splits - 1)];
      const uint32_t count = from.count[tid];
      const u64 mass = from.mass[tid];
      if (i + j < a.splits) c += count, m += mass;
    }
  }
  s.count[tid] = c, s.mass[tid] = m;
  __syncthreads();
  bin = scan_bins(s, s.count, s.mass, tid);
  return make_plan(s, q, bin, tid);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_pick_kernel(SplitArgs a) {
  __shared__ Shared s;
  const int tid = threadIdx.x, row_id = blockIdx.y, split = blockIdx.x;
  const Row<T> row = row_of<T>(a.p, row_id);
  Hand& hand = a.hand[row_id];
  const Request q = hand.request;
  if (q.scanned()) return;
  Bin bin{};
  const Plan plan = planned(s, a, row_id, q, bin, tid);
  if (split == 0 && tid == 0) hand.plan = plan;
  hand_over(s, a, hand, row, q, plan, split, gridDim.x, tid);
}

// kPicks: with pick's work in front, and the row's last workgroup to go on.
template <typename T, bool kPicks>
__global__ __launch_bounds__(kThreads) void sample_draw_kernel(SplitArgs a) {
  __shared__ Shared s;
  const int tid = threadIdx.x, row_id = blockIdx.y, split = blockIdx.x;
  const Row<T> row = row_of<T>(a.p, row_id);
  Hand& hand = a.hand[row_id];
  const Request q = hand.request;
  if (q.settled() || (q.scanned() && split > 0)) return;
  Bin bin{};
  Plan plan;
  if (kPicks && !q.scanned()) {
    plan = planned(s, a, row_id, q, bin, tid);
    hand_over(s, a, hand, row, q, plan, split, a.splits, tid);
    // every store has completed before the workgroup counts itself in
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) s.found = atomicAdd(&hand.done, 1u) + 1u == static_cast<uint32_t>(a.splits);
    __syncthreads();
    if (!s.found) return;
  } else {
    plan = hand.plan;
    // the p cut's bin follows from the k cut
    if (!kPicks && plan.by_k && plan.by_p && !q.few) planned(s, a, row_id, q, bin, tid);
  }
  if (q.few) plan.candidates = load_coherent(&hand.listed);
  if (tid < a.parts) s.part[tid] = load_coherent(&hand.part[tid]);
  if (plan.candidates <= kList) {
    const int n = static_cast<int>(plan.candidates);
#pragma unroll 1
    for (int i = tid; i < n; i += 4 * kThreads) {
      uint32_t k[4];
      int32_t at[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        k[j] = load_coherent(&hand.key[min(i + j * kThreads, n - 1)]);
        at[j] = load_coherent(&hand.index[min(i + j * kThreads, n - 1)]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j * kThreads < n) s.key[i + j * kThreads] = k[j], s.index[i + j * kThreads] = at[j];
    }
  }
  __syncthreads();
  finish(s, a.p, row_id, row, q, plan, bin, a.part, a.parts, tid);
}

// Workgroups a row.
int splits_of(int rows, int vocab) {
  int n = 1;
  while (n < kMaxSplit && 2 * n * rows <= kWorkgroups && vocab / (2 * n) >= kThreads) n *= 2;
  return n;
}

template <typename T>
void launch(SampleArgs p, void* workspace, hipStream_t stream) {
  for (int left = p.rows; left > 0; left -= kMaxRows) {
    p.rows = left < kMaxRows ? left : kMaxRows;
    const int splits = splits_of(p.rows, p.vocab);
    // parts of whole rounds of a wave, a multiple of `splits` in number
    const int vecs = ceil_div(p.vocab, Row<T>::kVec), round = 64;
    const int part = round * ceil_div(vecs, round * kMaxParts);
    const int picks = splits * 2 < kMaxSplit ? splits * 2 : kMaxSplit;
    const int parts = picks * ceil_div(ceil_div(vecs, part), picks);
    const dim3 grid(splits, p.rows), block(kThreads);
    Hand* hand = static_cast<Hand*>(workspace);
    const SplitArgs a{p, hand, reinterpret_cast<Histogram*>(hand + p.rows), splits, part, parts};
    hipLaunchKernelGGL(sample_best_kernel<T>, grid, block, 0, stream, a);
    hipLaunchKernelGGL(sample_scan_kernel<T>, grid, block, 0, stream, a);
    // Few rows gain from one launch less (one row 24 us of kernels against 28); with many, pick's share is faster
    // in a kernel of fewer registers, and idle workgroups in one of fewer launches (256 rows 130 against 147).
    if (splits * p.rows <= kFewWorkgroups) {
      hipLaunchKernelGGL((sample_draw_kernel<T, true>), grid, block, 0, stream, a);
    } else {
      hipLaunchKernelGGL(sample_pick_kernel<T>, dim3(picks, p.rows), block, 0, stream, a);
      hipLaunchKernelGGL((sample_draw_kernel<T, false>), dim3(1, p.rows), block, 0, stream, a);
    }
    p.logits = static_cast<const T*>(p.logits) + kMaxRows * p.stride;
    p.u += kMaxRows, p.temperature += kMaxRows, p.top_p += kMaxRows, p.min_p += kMaxRows, p.top_k += kMaxRows;
    p.tokens += kMaxRows;
    if (p.logprobs) p.logprobs += kMaxRows;
  }
}

}  // namespace
}  // namespace pega

using namespace pega;

PEGA_API long long pega_sample_workspace_bytes(int rows, int vocab) {
  if (rows <= 0 || vocab <= 0) return 0;
  // for any batch up to `rows`: the most rows, and the most histograms
  const long long most = rows < kMaxRows ? rows : kMaxRows;
  const long long hists = most * kMaxSplit < kWorkgroups ? most * kMaxSplit : kWorkgroups;
  return most * static_cast<long long>(sizeof(Hand)) + hists * static_cast<long long>(sizeof(Histogram));
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
  const auto there = [&](const float* v) { return v ? v : uniform; };
  const SampleArgs p{logits, row_stride, rows, vocab, uniform, there(temperature), there(top_p), there(min_p),
                     top_k ? top_k : reinterpret_cast<const int32_t*>(uniform), tokens, logprobs,
                     temperature != nullptr, top_p != nullptr, min_p != nullptr, top_k != nullptr};
  if (logits_bf16) launch<uint16_t>(p, workspace, stream);
  else launch<float>(p, workspace, stream);
  return launch_status("sample_tokens");
}
