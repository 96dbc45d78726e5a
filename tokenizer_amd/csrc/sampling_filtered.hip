// Draws under temperature, top-k, top-p and min-p from given uniform numbers.
//
// The tokens of a row stand in the order of falling logit, lower index first among equals; token i weighs
// w_i = exp((l_i - max) / T).  Kept are the first k of the order (k <= 0: all of them), of those the shortest prefix that reaches
// top_p of their weight (top_p >= 1: all), of those the tokens with w_i >= min_p.  Every cut keeps a prefix of the one order, so what
// is kept is the shortest of the three prefixes, and the draw is the first token of the whole order whose running weight exceeds
// uniform * (weight of what is kept).  A draw is therefore three questions, "where does the running count or the running weight of
// the order reach a number", asked one after the other.
//
// Weights are whole numbers, w_i * 2^44 rounded to nearest (the exponential in 64 bits).  Sums of whole numbers do not depend on their
// order, so a draw is the same however a row is cut over workgroups, and up to 2^19 tokens' sum stays within 63 bits.  A weight is off
// by its rounding, 2^-45 of the row's largest, and by what the exponential was off before it, some 2^-46 of itself: 32-bit weights would
// move the border between two tokens of a flat row of 150,000 by a good part of a token.  Tokens that weigh nothing then (31.2 T below the
// maximum) are never drawn.
//
// No row is sorted whole: the tokens among which the answers lie, some hundreds, are gathered and ordered in LDS.
//   * Where the first k tokens are all that counts, or those that min-p keeps, a logit is known below which nothing does
//     (`fs_cut`): the k-th largest of the maxima of the row's parts, of which at least k tokens are no smaller, or
//     max + T ln(min_p).  What is not below it is the list, where those maxima say that it is short.
//   * Else every token's weight matters.  The tokens fall into FS_BINS ranges of logit, equal parts of what lies between the maximum and the
//     lowest logit that weighs anything, each with its count and weight; the answers then lie in a few ranges (what is not known
//     yet of an earlier answer is at most a range's weight), whose tokens are the list.
// Should there be more than FS_LIST of them (thousands of logits that are equal, or nearly beside the row's whole range), one workgroup goes
// through the row again and again and narrows the answer's range by counting, key by key.
//
// What bounds it, measured with logits of 32 bits in the caches (the operator's own launches, replayed):
//   one row of 151,936 under top-k 40: 14.6 us, a chain of three launches (extents 3.6, the list 6.0, the draw 6.0 with the profiler's
//     share), each a few dependent steps of one workgroup a piece; reading 0.6 MB would take 0.1.  Under top-p alone 22.
//   64 rows of 151,936, each under other limits: 31 us: the extents 8.8, the second reading 11.5 (weights in 64 bits where the bins are
//     needed), ordering the lists 9.2, the gathering and the draws 4.6.
//   256 rows of 152,064 under min-p: 55 us: the extents 25 (156 MB at 6.2 TB/s), the list 16, the draw 9; a row read once at the rate of a
//     large copy would take 31.  Rows of 151,936 flat logits of which min-p keeps thousands or all: 8 rows 37, 256 rows 144 to 171.  Under top-p alone, where every token's weight and bin is worked out, 134.
// A workgroup has 4,096 logits, sixteen a thread, all asked for at once; a single row is then 38 workgroups.
//
// NaN is no token.  A row without a finite maximum, and a row whose temperature is not positive, gets its first maximum (0 if it
// holds no number).
#include "common.h"

#define FS_THREADS 256                  // of a long row's workgroups
#define FS_EACH 16                      // logits a thread holds
#define FS_PIECE (FS_THREADS * FS_EACH)
#define FS_SHORT_THREADS 512            // of a short row's
#define FS_SHORT_EACH 16
#define FS_BINS 256                     // four a lane
#define FS_LIST 8192
#define FS_FEW 128
#define FS_SLOTS 256                    // ranges that a round of narrowing tells apart
// Long rows of up to so many pieces together (a compute unit each) take three launches instead of five.  (Three | five, us on the device alone:
// rows of 151,936, 2 rows under top-p 23.2 | 24.7, under top-k 40 15.9 | 18.6, 6 rows 35.5 | 33.5, 15.9 | 18.4; rows of 32,000, 16 rows
// 22.6 | 24.4, 16.5 | 19.6, 32 rows 26.9 | 24.6, 16.7 | 20.2; and two launches less for the host.)
#define FS_FEW_PIECES 256
#define FS_SPAN 4                       // pieces that a workgroup sees to in the passes behind the first ...
// ... from so many pieces of all rows on.  (One | four pieces a workgroup, us: rows of 151,936 under min-p, 128 rows 34.8 | 33.9, 256 54.3 |
// 47.8, 512 104 | 84; under top-k 40 47.5 | 40.5, 77 | 64, 148 | 120; under top-p 81 | 85, 136 | 137, 267 | 239; rows of 32,000 under
// several limits, 128 rows 35 | 46, 512 86 | 91.)
#define FS_MANY_PIECES 8192
#define FS_MAX_WAVES (FS_SHORT_THREADS / WAVE)
#define FS_UNIT 17592186044416.0        // 2^44
#define FS_REACH 31.3f                  // beyond so many T below the maximum a weight is less than half a unit: nothing

typedef unsigned long long u64;

__device__ __forceinline__ uint32_t fs_key(float v) {      // larger float, larger key; zeros of both signs are one (v is a number)
  const uint32_t b = __float_as_uint(v + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float fs_value(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}

// What a row's logits are measured with.
struct FsRow {
  float top;             // the largest logit
  float per_bin;         // bins a unit of logit
  float reach;           // beyond so far below `top` nothing weighs anything
  double rate;           // log2(e) / T
};

// Whether a row is drawn at all; else it gets its first maximum.
__device__ __forceinline__ bool fs_is_drawn(float t, float top) { return t > 0.f && top > -INFINITY && top < INFINITY; }

__device__ __forceinline__ FsRow fs_row(float t, float top, float low) {
  FsRow r;
  r.top = top;
  r.rate = 1.4426950408889634074 / (double)t;
  r.reach = FS_REACH * t;
  const float span = fminf(top - low, r.reach);
  r.per_bin = span > 0.f ? fminf((float)FS_BINS / span, 3.0e38f) : 0.f;
  return r;
}

// 2^44 exp((v - top) / T) before it is rounded: 2^n of the whole part, and the rest, between -1/2 and 1/2, by the power series of 2^f,
// whose terms from the twelfth on are below 2^-47 together.
__device__ __forceinline__ double fs_share(float v, const FsRow& r) {
  constexpr double L = 0.69314718055994530942, c2 = L * L / 2, c3 = c2 * L / 3, c4 = c3 * L / 4, c5 = c4 * L / 5, c6 = c5 * L / 6,
                   c7 = c6 * L / 7, c8 = c7 * L / 8, c9 = c8 * L / 9, c10 = c9 * L / 10, c11 = c10 * L / 11;
  const double x = fmax(((double)v - (double)r.top) * r.rate, -100.0);
  const double n = rint(x), f = x - n;
  double p = fma(c11, f, c10);
  p = fma(p, f, c9); p = fma(p, f, c8); p = fma(p, f, c7); p = fma(p, f, c6); p = fma(p, f, c5);
  p = fma(p, f, c4); p = fma(p, f, c3); p = fma(p, f, c2); p = fma(p, f, L); p = fma(p, f, 1.0);
  return ldexp(p, (int)n + 44);
}
// Rounded to nearest (2^52 more leaves no bits behind the point).
__device__ __forceinline__ u64 fs_whole(double share) {
  return (u64)__double_as_longlong(share + 4503599627370496.0) & 0xfffffffffffffull;
}
__device__ __forceinline__ u64 fs_weight(float v, const FsRow& r) { return fs_whole(fs_share(v, r)); }
// Falls with the logit, so a bin is a run of the order; `top` is in bin 0.
__device__ __forceinline__ int fs_bin(float v, const FsRow& r) {
  return min(FS_BINS - 1, (int)((r.top - v) * r.per_bin));
}

struct FsAsked { float temperature, top_p, min_p, uniform; int top_k; };

// The weight of what min-p keeps, from that of the tokens whose share reaches it and of the maxima: above one no share reaches it, and the order's
// first token alone is kept (equal maxima weigh 2^44 each).
__device__ __forceinline__ u64 fs_kept_by_floor(const FsAsked& asked, u64 over) { return asked.min_p > 1.f ? 1ull << 44 : over; }

struct FsSmall {
  u64 mass[FS_BINS];                    // the bins, of a piece or of the whole row
  uint32_t count[FS_BINS];
  u64 wave_mass[FS_MAX_WAVES], wave_over[FS_MAX_WAVES];
  uint32_t wave_count[FS_MAX_WAVES];
  float wave_low[FS_MAX_WAVES], wave_high[FS_MAX_WAVES];
  int wave_at[FS_MAX_WAVES];
  int n_listed, listed;
  float cut;
};

struct FsFew { u64 token, w; };

struct FsShared : FsSmall {
  FsFew few[FS_FEW];                    // a short list with its weights, and what its parts add up
  u64 part_mass[FS_SHORT_THREADS];
  uint32_t part_count[FS_SHORT_THREADS];
  union {
    u64 list[FS_LIST];                  // the gathered tokens, key in the upper half, the index's complement in the lower
    struct { u64 mass[FS_SLOTS]; uint32_t count[FS_SLOTS]; } slots;      // a round of narrowing
  };
  u64 spread_mass[256];                 // what lies before the ranges that a list is spread over
  uint32_t spread_count[256], spread_start[256], spread_next[256];
  u64 missing_mass[FS_BINS];            // of bins that were not gathered, in front of this one
  uint32_t missing_count[FS_BINS];
  u64 found_mass, kept, over;
  uint32_t found_count;
  int found;
  uint32_t key_low, key_high;
};

__device__ __forceinline__ u64 fs_up(u64 v, int off, int lane) {          // the value `off` lanes down, 0 where there is none
  const u64 got = __shfl_up(v, off, WAVE);
  return lane >= off ? got : 0;
}

// Sum over the workgroup, to every thread.
template <int THREADS>
__device__ __forceinline__ u64 fs_sum(u64 v, FsSmall& s) {
  for (int off = WAVE / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, WAVE);
  __syncthreads();
  if ((threadIdx.x & (WAVE - 1)) == 0) s.wave_mass[threadIdx.x / WAVE] = v;
  __syncthreads();
  u64 total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / WAVE; ++w) total += s.wave_mass[w];
  return total;
}

// The logits of a piece in registers: thread i has logits i, i + THREADS, ...; NaN where there is none, and in threads that are not `wanted`,
// which ask memory for nothing.
template <int THREADS, int EACH, typename T>
__device__ __forceinline__ void fs_load(const T* __restrict__ row, int begin, int vocab, float (&v)[EACH], bool wanted = true) {
#pragma unroll
  for (int j = 0; j < EACH; ++j) v[j] = __uint_as_float(0x7fc00000u);
  if (wanted) {
#pragma unroll
    for (int j = 0; j < EACH; ++j) v[j] = ld(row + min(begin + j * THREADS + (int)threadIdx.x, vocab - 1));
#pragma unroll
    for (int j = 0; j < EACH; ++j)
      if (begin + j * THREADS + (int)threadIdx.x >= vocab) v[j] = __uint_as_float(0x7fc00000u);
  }
}

// The largest of a piece's logits, its lowest index, and the smallest above -inf, to every thread.  `of_wave`, `of_row`: the
// largest of the wave's, and of those of the thread's sixteen lanes.
template <int THREADS, int EACH>
__device__ __forceinline__ void fs_extent(const float (&v)[EACH], int begin, float& high, int& at, float& low, float& of_wave, float& of_row,
                                          FsSmall& s) {
  high = -INFINITY;
  low = INFINITY;
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    high = fmaxf(high, v[j]);
    low = fminf(low, v[j] > -INFINITY ? v[j] : INFINITY);
  }
  of_row = wave_max_repeated<16>(high);
  high = of_wave = wave_max_across<32>(wave_max_across<16>(of_row));
  low = -wave_max(-low);
  at = 0x7fffffff;
  if (high > -INFINITY) {
#pragma unroll
    for (int j = EACH - 1; j >= 0; --j) {
      const unsigned long long equal = __ballot(v[j] == high);
      if (equal) at = begin + j * THREADS + (int)(threadIdx.x & ~(WAVE - 1)) + __ffsll(equal) - 1;
    }
  }
  const int wave = threadIdx.x / WAVE;
  if ((threadIdx.x & (WAVE - 1)) == 0) { s.wave_high[wave] = high; s.wave_at[wave] = at; s.wave_low[wave] = low; }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / WAVE; ++w) {
    if (s.wave_high[w] > high || (s.wave_high[w] == high && s.wave_at[w] < at)) { high = s.wave_high[w]; at = s.wave_at[w]; }
    low = fminf(low, s.wave_low[w]);
  }
}

// Bins in `s.mass` and (if `counted`) `s.count`.  A thread's logits are added to them, and the weight of those that min-p keeps is returned.
__device__ __forceinline__ void fs_clear_bins(FsSmall& s) {
  if (threadIdx.x < FS_BINS) { s.mass[threadIdx.x] = 0; s.count[threadIdx.x] = 0; }
  __syncthreads();
}
template <int EACH>
__device__ __forceinline__ u64 fs_fill_bins(const float (&v)[EACH], const FsRow& r, const FsAsked& asked, FsSmall& s) {
  const bool counted = asked.top_k > 0, floored = asked.min_p > 0.f;
  const double floor_share = (double)asked.min_p * FS_UNIT;
  u64 over = 0;
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    if (r.top - v[j] <= r.reach) {                         // (false for NaN)
      const double share = fs_share(v[j], r);
      const u64 w = fs_whole(share);
      const int bin = fs_bin(v[j], r);
      atomicAdd(&s.mass[bin], w);
      if (counted) atomicAdd(&s.count[bin], 1u);
      if (!floored || !(share < floor_share) || v[j] == r.top) over += w;
    }
  }
  return over;
}

// A wave's view of the bins: running counts and weights, bins 4 lane .. + 3.
struct FsRunning {
  u64 mass[4];
  uint32_t count[4];
  __device__ __forceinline__ void of(const FsSmall& s) {
    const int lane = threadIdx.x & (WAVE - 1);
    u64 m = 0, c = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m += s.mass[4 * lane + j];
      c += s.count[4 * lane + j];
      mass[j] = m;
      count[j] = (uint32_t)c;
    }
    u64 run_m = m, run_c = c;
    for (int off = 1; off < WAVE; off <<= 1) {
      run_m += fs_up(run_m, off, lane);
      run_c += fs_up(run_c, off, lane);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) { mass[j] += run_m - m; count[j] += (uint32_t)(run_c - c); }
  }
  // How many bins' running numbers are below: that is the bin in which it is reached.
  __device__ __forceinline__ int bin_of_mass(u64 need) const {
    int below = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) below += __popcll(__ballot(mass[j] < need));
    return below;
  }
  __device__ __forceinline__ int bin_of_count(uint32_t need) const {
    int below = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) below += __popcll(__ballot(count[j] < need));
    return below;
  }
  __device__ __forceinline__ u64 mass_to(int bin) const {                 // of bins 0 .. bin
    if (bin < 0) return 0;
    u64 v = mass[0];
#pragma unroll
    for (int j = 1; j < 4; ++j) v = (bin & 3) == j ? mass[j] : v;
    return __shfl(v, bin >> 2, WAVE);
  }
  __device__ __forceinline__ uint32_t count_to(int bin) const {
    if (bin < 0) return 0;
    uint32_t v = count[0];
#pragma unroll
    for (int j = 1; j < 4; ++j) v = (bin & 3) == j ? count[j] : v;
    return (uint32_t)__shfl((int)v, bin >> 2, WAVE);
  }
};

// The running weight at which top-p's prefix ends, given the weight of what top-k keeps; and the one at which the draw lies, given the
// weight of what is kept.  Both rise with what is given.
__device__ __forceinline__ u64 fs_need_of_share(float top_p, u64 kept) {
  const double share = ceil((double)fmaxf(top_p, 0.f) * (double)kept);
  return share < 1.0 ? 1ull : (u64)share;
}
__device__ __forceinline__ u64 fs_need_of_draw(float uniform, u64 kept) {
  const double target = (double)uniform * (double)kept;
  const u64 need = target >= 0.0 ? (target < (double)kept ? (u64)floor(target) + 1 : kept) : 1ull;
  const u64 most = need < kept ? need : kept;
  return most > 0 ? most : 1ull;
}

// The bins in which the three answers lie (first > last: none).
struct FsRanges {
  int k_bin, p_first, p_last, draw_first, draw_last;
  __device__ __forceinline__ bool has(int bin) const {
    return bin == k_bin || (bin >= p_first && bin <= p_last) || (bin >= draw_first && bin <= draw_last);
  }
};
__device__ __forceinline__ FsRanges fs_ranges(const FsRunning& run, const FsAsked& asked, u64 over) {
  FsRanges g;
  const u64 total = run.mass_to(FS_BINS - 1);
  u64 least = total, most = total;
  g.k_bin = -1;
  if (asked.top_k > 0 && run.count_to(FS_BINS - 1) >= (uint32_t)asked.top_k) {
    g.k_bin = run.bin_of_count((uint32_t)asked.top_k);
    least = run.mass_to(g.k_bin - 1);
    most = run.mass_to(g.k_bin);
  }
  g.p_first = 0;
  g.p_last = -1;
  if (asked.top_p < 1.f) {
    const u64 need_least = fs_need_of_share(asked.top_p, least), need_most = fs_need_of_share(asked.top_p, most);
    g.p_first = run.bin_of_mass(need_least);
    g.p_last = run.bin_of_mass(need_most);
    const u64 to_last = run.mass_to(min(g.p_last, FS_BINS - 1));
    least = need_least;
    most = to_last < most ? to_last : most;
  }
  if (over < least) least = over;
  if (over < most) most = over;
  g.draw_first = run.bin_of_mass(fs_need_of_draw(asked.uniform, least));
  g.draw_last = run.bin_of_mass(fs_need_of_draw(asked.uniform, most));
  return g;
}

// ------------------------------------------------------------------------------------------------
// Narrowing, for more tokens than are sorted: the row is read again for every round.

// Where the order of the slots, the last one first unless `forwards`, reaches a number (the running count if `counting`, else the running
// mass).  Returns the slot, and what lies before it in `count` and `mass`; -1 if the whole order does not reach it.
__device__ int fs_reach(FsShared& s, bool forwards, bool counting, u64 need, uint32_t& count, u64& mass) {
  static_assert(FS_SLOTS == 4 * WAVE, "four slots a lane of one wave");
  const int lane = threadIdx.x & (WAVE - 1);
  __syncthreads();
  if (threadIdx.x < WAVE) {
    u64 m[4], c[4], all_m = 0, all_c = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int slot = forwards ? 4 * lane + j : FS_SLOTS - 1 - 4 * lane - j;
      m[j] = s.slots.mass[slot];
      c[j] = s.slots.count[slot];
      all_m += m[j];
      all_c += c[j];
    }
    u64 run_m = all_m, run_c = all_c;
    for (int off = 1; off < WAVE; off <<= 1) {
      run_m += fs_up(run_m, off, lane);
      run_c += fs_up(run_c, off, lane);
    }
    run_m -= all_m;
    run_c -= all_c;
    if (lane == 0) s.found = -1;
    wave_exchange();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const u64 before = counting ? run_c : run_m, here = counting ? c[j] : m[j];
      if (before < need && before + here >= need) {        // one slot of one lane
        s.found = forwards ? 4 * lane + j : FS_SLOTS - 1 - 4 * lane - j;
        s.found_mass = run_m;
        s.found_count = (uint32_t)run_c;
      }
      run_m += m[j];
      run_c += c[j];
    }
  }
  __syncthreads();
  const int at = s.found;
  count = s.found_count;
  mass = s.found_mass;
  __syncthreads();
  return at;
}

__device__ __forceinline__ void fs_clear_slots(FsShared& s) {
  __syncthreads();
  if (threadIdx.x < FS_SLOTS) { s.slots.mass[threadIdx.x] = 0; s.slots.count[threadIdx.x] = 0; }
  __syncthreads();
}

// Calls use(value, index) for every number of the row, a thread every THREADS-th one, sixteen loads asked for at a time.
template <int THREADS, typename T, typename Use>
__device__ __forceinline__ void fs_numbers(const T* __restrict__ row, int vocab, Use use) {
  for (int base = threadIdx.x; base < vocab; base += 16 * THREADS) {
    float v[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = ld(row + min(base + j * THREADS, vocab - 1));
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (base + j * THREADS < vocab && v[j] == v[j]) use(v[j], base + j * THREADS);
  }
}

// The key at which the order reaches a number, what lies before the tokens of that key, and what each of them weighs.
struct FsCrossing {
  uint32_t key, before_count;
  u64 before_mass, each;
};

template <int THREADS, typename T>
__device__ FsCrossing fs_narrow(FsShared& s, const T* row, int vocab, const FsRow& r, int bin, bool counting, u64 need, uint32_t before_count,
                                u64 before_mass) {
  uint32_t low = 0xffffffffu, high = 0;
  fs_numbers<THREADS>(row, vocab, [&](float v, int) {
    if (r.top - v <= r.reach && fs_bin(v, r) == bin) {
      const uint32_t key = fs_key(v);
      low = min(low, key);
      high = max(high, key);
    }
  });
  __syncthreads();
  if (threadIdx.x == 0) { s.key_low = 0xffffffffu; s.key_high = 0; }
  __syncthreads();
  atomicMin(&s.key_low, low);
  atomicMax(&s.key_high, high);
  __syncthreads();
  low = s.key_low;
  high = s.key_high;
  while (low < high) {
    int shift = 0;
    while (((high - low) >> shift) >= FS_SLOTS) ++shift;
    fs_clear_slots(s);
    fs_numbers<THREADS>(row, vocab, [&](float v, int) {
      if (r.top - v <= r.reach && fs_bin(v, r) == bin) {
        const uint32_t key = fs_key(v);
        if (key >= low && key <= high) {
          atomicAdd(&s.slots.count[(key - low) >> shift], 1u);
          atomicAdd(&s.slots.mass[(key - low) >> shift], fs_weight(v, r));
        }
      }
    });
    uint32_t inner_count = 0;
    u64 inner_mass = 0;
    const int slot = fs_reach(s, false, counting, need - (counting ? (u64)before_count : before_mass), inner_count, inner_mass);
    if (slot < 0) break;                                   // (cannot be: the bin reaches it)
    before_count += inner_count;
    before_mass += inner_mass;
    low += (uint32_t)slot << shift;
    high = min(high, low + ((1u << shift) - 1u));
  }
  FsCrossing x;
  x.key = high;
  x.before_count = before_count;
  x.before_mass = before_mass;
  x.each = fs_weight(fs_value(high), r);
  return x;
}

template <int THREADS, typename T>
__device__ int fs_draw_by_narrowing(FsShared& s, const T* row, int vocab, const FsRow& r, const FsAsked& asked) {
  // The bins of the whole row, weights and counts, anew (the row may have come here without any).
  __syncthreads();
  if (threadIdx.x < FS_BINS) { s.mass[threadIdx.x] = 0; s.count[threadIdx.x] = 0; }
  __syncthreads();
  const double floor_share = (double)asked.min_p * FS_UNIT;
  u64 over = 0;
  fs_numbers<THREADS>(row, vocab, [&](float v, int) {
    if (r.top - v <= r.reach) {
      const double share = fs_share(v, r);
      const u64 w = fs_whole(share);
      const int bin = fs_bin(v, r);
      atomicAdd(&s.mass[bin], w);
      atomicAdd(&s.count[bin], 1u);
      if (!(asked.min_p > 0.f) || !(share < floor_share) || v == r.top) over += w;
    }
  });
  over = fs_kept_by_floor(asked, fs_sum<THREADS>(over, s));
  FsRunning run;
  run.of(s);
  auto crossing = [&](int bin, bool counting, u64 need) {
    return fs_narrow<THREADS>(s, row, vocab, r, bin, counting, need, run.count_to(bin - 1), run.mass_to(bin - 1));
  };
  u64 kept = run.mass_to(FS_BINS - 1);
  if (asked.top_k > 0 && run.count_to(FS_BINS - 1) >= (uint32_t)asked.top_k) {
    const FsCrossing x = crossing(run.bin_of_count((uint32_t)asked.top_k), true, (u64)asked.top_k);
    kept = x.before_mass + ((u64)asked.top_k - x.before_count) * x.each;
  }
  if (asked.top_p < 1.f) {
    const u64 need = fs_need_of_share(asked.top_p, kept);
    const FsCrossing x = crossing(run.bin_of_mass(need), false, need);
    if (x.each > 0) {
      const u64 to = x.before_mass + (need - x.before_mass + x.each - 1) / x.each * x.each;
      kept = to < kept ? to : kept;
    }
  }
  kept = over < kept ? over : kept;
  const u64 need = fs_need_of_draw(asked.uniform, kept);
  const FsCrossing x = crossing(run.bin_of_mass(need), false, need);
  const u64 rank = x.each > 0 ? (need - x.before_mass + x.each - 1) / x.each : 1;
  // The rank-th token of the key: which run of indices has it, then which of the run.
  const int per = (vocab + FS_SLOTS - 1) / FS_SLOTS;
  fs_clear_slots(s);
  fs_numbers<THREADS>(row, vocab, [&](float v, int at) {
    if (fs_key(v) == x.key) atomicAdd(&s.slots.count[at / per], 1u);
  });
  uint32_t before = 0;
  u64 unused;
  const int part = fs_reach(s, true, true, rank, before, unused);
  if (threadIdx.x < WAVE) {                                // a wave looks through the run, sixty-four tokens at a time
    const int lane = threadIdx.x;
    const int end = part < 0 ? 0 : min(vocab, (part + 1) * per);
    uint32_t left = (uint32_t)(rank - before);
    int pick = 0;
    for (int i = max(part, 0) * per; i < end; i += WAVE) {
      const float v = ld(row + min(i + lane, vocab - 1));
      const bool is = i + lane < end && v == v && fs_key(v) == x.key;
      const unsigned long long votes = __ballot(is);
      const uint32_t here = (uint32_t)__popcll(votes);
      if (left <= here) {
        const bool mine = is && (uint32_t)__popcll(votes & ((1ull << lane) - 1ull)) + 1 == left;
        pick = i + __ffsll(__ballot(mine)) - 1;
        break;
      }
      left -= here;
    }
    if (lane == 0) s.found = pick;
  }
  __syncthreads();
  return s.found;
}

// ------------------------------------------------------------------------------------------------
// `size` (a power of two, at least 128) numbers of `s.list`, the largest first: runs of `run_of` fall and rise in turn until one is
// left.  Numbers at most 64 apart lie in a stretch of 128 that one wave sees to alone: no barrier between such steps.
template <int THREADS>
__device__ __forceinline__ void fs_sort(FsShared& s, int size) {
  for (int run_of = 2; run_of <= size; run_of <<= 1)
    for (int apart = run_of >> 1; apart > 0; apart >>= 1) {
      for (int i = threadIdx.x; i < size / 2; i += THREADS) {
        const int a = 2 * i - (i & (apart - 1)), b = a + apart;
        const u64 x = s.list[a], y = s.list[b];
        if ((x < y) == ((a & run_of) == 0)) { s.list[a] = y; s.list[b] = x; }
      }
      if (apart > 64 || (apart == 1 && run_of >= 128)) __syncthreads();      // (behind the last step of a run the next is wider than a wave's)
      else wave_exchange();
    }
  __syncthreads();
}

// The three answers.  `each(use)` calls use(token, weight, weight before it on the list, place on the list) for every token of the
// list, each by one thread.  `all`: the weight of the whole row (of the list, if that holds the order's first tokens: `all_listed`);
// `over`: the weight of what min-p keeps, if it is known.
template <typename Each>
__device__ __forceinline__ int fs_answers(FsShared& s, const FsRow& r, const FsAsked& asked, u64 all, bool k_here, u64 over, bool all_listed,
                                          Each each) {
  const double floor_share = (double)asked.min_p * FS_UNIT;
  if (threadIdx.x == 0) {
    s.kept = all;
    s.found = 0;
    s.over = 0;
  }
  __syncthreads();
  auto missing = [&](u64 token) { return all_listed ? 0ull : s.missing_mass[fs_bin(fs_value((uint32_t)(token >> 32)), r)]; };
  u64 above = 0;
  each([&](u64 token, u64 w, u64 before, uint32_t at) {
    const float v = fs_value((uint32_t)(token >> 32));
    before += missing(token);
    if (!all_listed) at += s.missing_count[fs_bin(v, r)];
    else if (!(asked.min_p > 0.f) || !(fs_share(v, r) < floor_share) || v == r.top)
      above = max(above, before + w);                      // (what min-p keeps is in the list, or ends behind it)
    if (k_here && at + 1 == (uint32_t)asked.top_k) s.kept = before + w;
  });
  if (above) atomicMax(&s.over, above);
  __syncthreads();
  u64 kept = s.kept;
  if (all_listed) over = fs_kept_by_floor(asked, s.over);
  if (asked.top_p < 1.f) {
    __syncthreads();
    const u64 need = fs_need_of_share(asked.top_p, kept);
    each([&](u64 token, u64 w, u64 before, uint32_t) {
      before += missing(token);
      if (before < need && before + w >= need) s.kept = before + w;
    });
    __syncthreads();
    kept = s.kept;
  }
  kept = over < kept ? over : kept;
  const u64 need = fs_need_of_draw(asked.uniform, kept);
  each([&](u64 token, u64 w, u64 before, uint32_t) {
    before += missing(token);
    if (before < need && before + w >= need) s.found = (int)~(uint32_t)token;
  });
  __syncthreads();
  return s.found;
}

// Up to FS_FEW tokens: each is held against all others, two to eight threads a token.  (A draw under top-k 40 from 151,936
// logits 14.6 us so, 15.8 by fs_spread; four rows of 1,000 logits 9.0 and 10.2.)
template <int THREADS>
__device__ __forceinline__ int fs_answers_of_few(FsShared& s, const FsRow& r, const FsAsked& asked, u64 all, bool k_here, u64 over, bool all_listed,
                                                 int n) {
  const int size = n <= WAVE ? WAVE : FS_FEW, parts = THREADS / size;
  const int at = threadIdx.x & (size - 1), part = threadIdx.x / size;
  u64 token = at < n ? s.list[at] : 0;
  const u64 w = token ? fs_weight(fs_value((uint32_t)(token >> 32)), r) : 0;
  if (part == 0) s.few[at] = FsFew{token, w};
  __syncthreads();
  u64 before = 0, listed = 0;
  uint32_t place = 0;
  const int of_part = size / parts;
  for (int i = part * of_part; i < (part + 1) * of_part; ++i) {          // (the same for a whole wave)
    const FsFew other = s.few[i];
    const bool first = other.token > token;
    before += first ? other.w : 0;
    place += first ? 1 : 0;
    listed += other.w;
  }
  s.part_mass[threadIdx.x] = before;
  s.part_count[threadIdx.x] = place;
  if (at == 0) s.wave_over[part] = listed;
  __syncthreads();
  before = listed = 0;
  place = 0;
  for (int i = 0; i < parts; ++i) {
    before += s.part_mass[i * size + at];
    place += s.part_count[i * size + at];
    listed += s.wave_over[i];
  }
  const bool goes_on = token && part == 0;                 // (one thread a token)
  return fs_answers(s, r, asked, all_listed ? listed : all, k_here, over, all_listed, [&](auto use) { if (goes_on) use(token, w, before, place); });
}

// More: from the sorted list, of which a thread has `per` neighbours.  (Their weights are worked out again for every answer: keeping
// those of 32 tokens would take the registers of all kernels that come here.)
template <int THREADS>
__device__ __forceinline__ int fs_answers_of_sorted(FsShared& s, const FsRow& r, const FsAsked& asked, u64 all, bool k_here, u64 over,
                                                    bool all_listed, int n, int per) {
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  const int first = threadIdx.x * per, last = min(n, first + per);
  u64 sum = 0;
  for (int i = first; i < last; ++i) sum += fs_weight(fs_value((uint32_t)(s.list[i] >> 32)), r);
  u64 run = sum;
  for (int off = 1; off < WAVE; off <<= 1) run += fs_up(run, off, lane);
  if (lane == WAVE - 1) s.wave_mass[wave] = run;
  run -= sum;
  __syncthreads();
  u64 listed = 0;
#pragma unroll
  for (int i = 0; i < THREADS / WAVE; ++i) {
    if (i < wave) run += s.wave_mass[i];
    listed += s.wave_mass[i];
  }
  return fs_answers(s, r, asked, all_listed ? listed : all, k_here, over, all_listed, [&](auto use) {
    u64 before = run;
    for (int i = first; i < last; ++i) {
      const u64 token = s.list[i], w = fs_weight(fs_value((uint32_t)(token >> 32)), r);
      use(token, w, before, (uint32_t)i);
      before += w;
    }
  });
}

// Up to FS_SPREAD tokens, unless many are (nearly) equal: they are spread over 256 ranges between the list's largest and smallest, whose
// counts and weights are added up in order, and each is held against those of its own range.  s.list: tokens as they came, then in
// order | weight before each | tokens range by range | their weights, FS_SPREAD each.  Returns false with the list as it was if a range has more
// than WAVE tokens.  (With 64 rows of 151,936 the settling pass, slowest row, 14.9 us sorted and 9.2 so; one row that lists 128 tokens or
// fewer takes fs_answers_of_few and pays nothing.)
#define FS_SPREAD (FS_LIST / 4)
template <int THREADS>
__device__ __forceinline__ bool fs_spread(FsShared& s, const FsRow& r, int n, u64& listed) {
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  u64* const before_s = s.list + FS_SPREAD;
  u64* const token_s = s.list + 2 * FS_SPREAD;
  u64* const weight_s = s.list + 3 * FS_SPREAD;
  float low = INFINITY, high = -INFINITY;
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const float v = fs_value((uint32_t)(s.list[i] >> 32));
    low = fminf(low, v);
    high = fmaxf(high, v);
  }
  low = -wave_max(-low);
  high = wave_max(high);
  if (lane == 0) { s.wave_low[wave] = low; s.wave_high[wave] = high; }
  for (int i = threadIdx.x; i < 256; i += THREADS) { s.spread_mass[i] = 0; s.spread_count[i] = 0; }
  if (threadIdx.x == 0) s.found = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / WAVE; ++w) { low = fminf(low, s.wave_low[w]); high = fmaxf(high, s.wave_high[w]); }
  const float per = high > low ? fminf(256.f / (high - low), 3.0e38f) : 0.f;
  auto range_of = [&](u64 token) { return min(255, (int)((high - fs_value((uint32_t)(token >> 32))) * per)); };
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const u64 token = s.list[i];
    const int range = range_of(token);
    if (atomicAdd(&s.spread_count[range], 1u) >= WAVE) s.found = 1;
    atomicAdd(&s.spread_mass[range], fs_weight(fs_value((uint32_t)(token >> 32)), r));
  }
  __syncthreads();
  if (s.found) return false;                               // (the same for the whole workgroup)
  if (wave == 0) {
    u64 m[4], all_m = 0;
    uint32_t c[4], all_c = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[j] = all_m;
      c[j] = all_c;
      all_m += s.spread_mass[4 * lane + j];
      all_c += s.spread_count[4 * lane + j];
    }
    u64 run_m = all_m;
    int run_c = (int)all_c;
    for (int off = 1; off < WAVE; off <<= 1) {
      run_m += fs_up(run_m, off, lane);
      const int got = __shfl_up(run_c, off, WAVE);
      if (lane >= off) run_c += got;
    }
    if (lane == WAVE - 1) s.found_mass = run_m;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      s.spread_mass[4 * lane + j] = m[j] + run_m - all_m;
      s.spread_start[4 * lane + j] = c[j] + (uint32_t)run_c - all_c;
      s.spread_next[4 * lane + j] = c[j] + (uint32_t)run_c - all_c;
    }
  }
  __syncthreads();
  listed = s.found_mass;
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const u64 token = s.list[i];
    const uint32_t to = atomicAdd(&s.spread_next[range_of(token)], 1u);
    token_s[to] = token;
    weight_s[to] = fs_weight(fs_value((uint32_t)(token >> 32)), r);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const u64 token = token_s[i];
    const int range = range_of(token);
    const uint32_t start = s.spread_start[range], end = start + s.spread_count[range];
    u64 before = s.spread_mass[range];
    uint32_t place = start;
    for (uint32_t k = start; k < end; ++k) {
      const bool first = token_s[k] > token;
      before += first ? weight_s[k] : 0;
      place += first ? 1 : 0;
    }
    s.list[place] = token;
    before_s[place] = before;
  }
  __syncthreads();
  return true;
}

// The draw from the `n` tokens in `s.list` (in any order), if they all found room there, else by narrowing.  `ranges`: the list holds
// these bins of the whole row's, which are in `s.mass` and `s.count`; null: it holds the order's first tokens, as many as count.
template <int THREADS, typename T>
__device__ int fs_draw(FsShared& s, const T* row, int vocab, const FsRow& r, const FsAsked& asked, const FsRanges* ranges, u64 over, int n) {
  if (n > FS_LIST) return fs_draw_by_narrowing<THREADS>(s, row, vocab, r, asked);
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  u64 all = 0;
  if (ranges) {
    FsRunning run;
    run.of(s);
    all = run.mass_to(FS_BINS - 1);
    if (wave == 0) {                                       // what lies between the gathered bins
      u64 m[4], c[4], run_m = 0, run_c = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool gathered = ranges->has(4 * lane + j);
        m[j] = run_m;
        c[j] = run_c;
        run_m += gathered ? 0 : s.mass[4 * lane + j];
        run_c += gathered ? 0 : s.count[4 * lane + j];
      }
      const u64 all_m = run_m, all_c = run_c;
      for (int off = 1; off < WAVE; off <<= 1) {
        run_m += fs_up(run_m, off, lane);
        run_c += fs_up(run_c, off, lane);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s.missing_mass[4 * lane + j] = m[j] + run_m - all_m;
        s.missing_count[4 * lane + j] = (uint32_t)(c[j] + run_c - all_c);
      }
    }
  }
  const bool k_here = asked.top_k > 0 && (!ranges || ranges->k_bin >= 0);
  __syncthreads();
  if (n <= FS_FEW) return fs_answers_of_few<THREADS>(s, r, asked, all, k_here, over, ranges == nullptr, n);
  u64 listed;
  if (n <= FS_SPREAD && fs_spread<THREADS>(s, r, n, listed))
    return fs_answers(s, r, asked, ranges ? all : listed, k_here, over, ranges == nullptr, [&](auto use) {
      for (int i = threadIdx.x; i < n; i += THREADS) {
        const u64 before = s.list[FS_SPREAD + i];
        use(s.list[i], (i + 1 < n ? s.list[FS_SPREAD + i + 1] : listed) - before, before, (uint32_t)i);
      }
    });
  int size = 2 * FS_FEW;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += THREADS) s.list[i] = 0;           // (behind every token)
  __syncthreads();
  fs_sort<THREADS>(s, size);
  const int per = max(1, size / THREADS);
  return fs_answers_of_sorted<THREADS>(s, r, asked, all, k_here, over, ranges == nullptr, n, per);
}

struct FsArgs {
  const void* logits;
  int64_t stride;
  const float *temperature, *top_p, *min_p, *uniform;
  const int* top_k;
  int* out;
  int vocab, pieces, shares;            // shares: workgroups of a row behind the first pass, SPAN pieces each
  char* workspace;
  size_t row_bytes;
};

__device__ __forceinline__ FsAsked fs_asked(const FsArgs& a, int row) {
  FsAsked q;
  q.temperature = scalar_float(a.temperature + row);
  q.top_p = scalar_float(a.top_p + row);
  q.min_p = scalar_float(a.min_p + row);
  q.uniform = scalar_float(a.uniform + row);
  q.top_k = scalar_int(a.top_k + row);
  return q;
}

// A row of at most FS_SHORT_THREADS * EACH logits: one workgroup, one launch.
template <typename T, int EACH>
__global__ void __launch_bounds__(FS_SHORT_THREADS)
sample_filtered_short(FsArgs a) {
  constexpr int THREADS = FS_SHORT_THREADS;
  __shared__ FsShared s;
  const int row_at = blockIdx.x;
  const T* row = (const T*)a.logits + (size_t)row_at * a.stride;
  const FsAsked asked = fs_asked(a, row_at);
  float v[EACH], high, low, of_wave, of_row;
  int at;
  fs_load<THREADS>(row, 0, a.vocab, v);
  fs_extent<THREADS>(v, 0, high, at, low, of_wave, of_row, s);
  if (!fs_is_drawn(asked.temperature, high)) {
    if (threadIdx.x == 0) a.out[row_at] = at == 0x7fffffff ? 0 : at;
    return;
  }
  const FsRow r = fs_row(asked.temperature, high, low);
  fs_clear_bins(s);
  const u64 over = fs_kept_by_floor(asked, fs_sum<THREADS>(fs_fill_bins(v, r, asked, s), s));     // (its barriers stand behind the bins, too)
  FsRunning run;
  run.of(s);
  const FsRanges ranges = fs_ranges(run, asked, over);
  if (threadIdx.x == 0) s.n_listed = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < EACH; ++j)
    if (r.top - v[j] <= r.reach && ranges.has(fs_bin(v[j], r))) {
      const int place = atomicAdd(&s.n_listed, 1);
      if (place < FS_LIST) s.list[place] = (u64)fs_key(v[j]) << 32 | (uint32_t)~(uint32_t)(j * THREADS + (int)threadIdx.x);
    }
  __syncthreads();
  const int pick = fs_draw<THREADS>(s, row, a.vocab, r, asked, &ranges, over, s.n_listed);
  if (threadIdx.x == 0) a.out[row_at] = pick;
}

// ------------------------------------------------------------------------------------------------
// A longer row: its pieces' workgroups leave what they found in the workspace, a launch a step.
#define FS_PIECE_WAVES (FS_THREADS / WAVE)
#define FS_PIECE_ROWS (FS_THREADS / 16)
struct FsExtent { float high, low; int at, unused; };
struct FsHead { int n_listed; int ranges[5]; int gathered, listed; u64 over, unused; };   // of a row; `gathered`: pieces that are; `listed`: without bins
struct FsBinned { u64 mass[FS_BINS]; uint32_t count[FS_BINS]; u64 over; u64 unused; };    // of a piece, or of a row
// Per row: its head, its bins, its list, the pieces' extents, the maxima of their waves and of these waves' rows of sixteen lanes, and the
// pieces' bins.
struct FsSpace {
  char* base;
  int pieces, shares;
  __device__ __forceinline__ FsHead* head() const { return (FsHead*)base; }
  __device__ __forceinline__ FsBinned* whole() const { return (FsBinned*)(base + sizeof(FsHead)); }
  __device__ __forceinline__ u64* list() const { return (u64*)(whole() + 1); }
  __device__ __forceinline__ FsExtent* extents() const { return (FsExtent*)(list() + FS_LIST); }
  __device__ __forceinline__ float* of_waves() const { return (float*)(extents() + pieces); }
  __device__ __forceinline__ float* of_rows() const { return of_waves() + pieces * FS_PIECE_WAVES; }
  __device__ __forceinline__ FsBinned* binned() const { return (FsBinned*)(of_rows() + pieces * FS_PIECE_ROWS); }
};
static size_t fs_row_bytes(int pieces) {
  return sizeof(FsHead) + sizeof(FsBinned) + 8 * FS_LIST + (sizeof(FsExtent) + 4 * (FS_PIECE_WAVES + FS_PIECE_ROWS) + sizeof(FsBinned)) * (size_t)pieces;
}
static_assert(sizeof(FsHead) % 16 == 0 && sizeof(FsBinned) % 16 == 0 && sizeof(FsExtent) % 16 == 0 && (FS_PIECE_WAVES + FS_PIECE_ROWS) % 4 == 0, "pieces of sixteen bytes");
__device__ __forceinline__ FsSpace fs_space(const FsArgs& a, int row) { return FsSpace{a.workspace + (size_t)row * a.row_bytes, a.pieces, a.shares}; }

// The row's extent from its pieces' (a lane of every wave looks at one piece of sixty-four), to every thread.
__device__ __forceinline__ void fs_row_extent(const FsSpace& w, float& high, float& low) {
  const int lane = threadIdx.x & (WAVE - 1);
  high = -INFINITY;
  low = INFINITY;
  for (int p = lane; p < w.pieces; p += WAVE) {
    high = fmaxf(high, w.extents()[p].high);
    low = fminf(low, w.extents()[p].low);
  }
  high = wave_max(high);
  low = -wave_max(-low);
}
// The lowest index of the row's largest logit, to every thread; 0 if there is none above -inf.
__device__ __forceinline__ int fs_row_top(const FsSpace& w, float high) {
  const int lane = threadIdx.x & (WAVE - 1);
  int at = 0x7fffffff;
  for (int p = lane; p < w.pieces; p += WAVE)
    if (w.extents()[p].high == high) at = min(at, w.extents()[p].at);
  for (int off = WAVE / 2; off > 0; off >>= 1) at = min(at, __shfl_xor(at, off, WAVE));
  return at == 0x7fffffff ? 0 : at;
}

// How many maxima of rows of sixteen lanes stand for 256 logits each.
__device__ __forceinline__ int fs_full_maxima(int vocab) { return vocab / FS_PIECE * FS_PIECE_ROWS; }
// Whether a row's list may be made without its bins: top-k or min-p says below which logit nothing counts.  (Half as many tokens as maxima
// at most: the list is then about k long; close to their number it would be several times as long.)
__device__ __forceinline__ bool fs_few_wanted(const FsAsked& asked, int vocab) { return asked.top_k > 0 && asked.top_k <= fs_full_maxima(vocab) / 2; }
__device__ __forceinline__ bool fs_floor_alone(const FsAsked& asked) { return !(asked.top_p < 1.f) && asked.min_p > 0.f; }
__device__ __forceinline__ bool fs_may_be_listed(const FsAsked& asked, int vocab) { return fs_few_wanted(asked, vocab) || fs_floor_alone(asked); }

// A logit not below `least` of which at least k of the `count` maxima are no smaller, close to the k-th largest of them; -inf if there are
// not so many.
template <int MOST>
__device__ __forceinline__ float fs_cut_of_maxima(const float* __restrict__ maxima, int count, int k, float least, float most) {
  const int lane = threadIdx.x & (WAVE - 1);
  float m[MOST];                                           // of 64 lanes
#pragma unroll
  for (int j = 0; j < MOST; ++j) {
    m[j] = -INFINITY;
    if (j * WAVE + lane < count) m[j] = maxima[j * WAVE + lane];
  }
  auto no_smaller = [&](float t) {
    int found = 0;
#pragma unroll
    for (int j = 0; j < MOST; ++j)
      if (j * WAVE < count) found += __popcll(__ballot(m[j] >= t));
    return found;
  };
  if (no_smaller(least) < k) return -INFINITY;
  for (int turn = 0; turn < 8; ++turn) {
    const float middle = 0.5f * least + 0.5f * most;
    if (no_smaller(middle) >= k) least = middle; else most = middle;
  }
  return least;
}

// Of how many groups of logits the maximum is no smaller than `cut`, and than `least`.
struct FsAbove { int cut, least; };
template <int MOST>
__device__ __forceinline__ FsAbove fs_above(const float* __restrict__ maxima, int count, float cut, float least) {
  const int lane = threadIdx.x & (WAVE - 1);
  float m[MOST];
#pragma unroll
  for (int j = 0; j < MOST; ++j) {
    m[j] = -INFINITY;
    if (j * WAVE + lane < count) m[j] = maxima[j * WAVE + lane];
  }
  FsAbove above = {0, 0};
#pragma unroll
  for (int j = 0; j < MOST; ++j)
    if (j * WAVE < count) {
      above.cut += __popcll(__ballot(m[j] >= cut));
      above.least += __popcll(__ballot(m[j] >= least));
    }
  return above;
}

// Whether the maxima say that few tokens are no smaller than `cut` (`least`: what lies below weighs nothing): there are no more groups with such a
// token than the list has room for; or one in sixteen of the groups with anything to weigh has none; or the groups with one are hardly more
// than the waves' of four groups.  (Spread evenly over N groups, M tokens leave N e^(-M / N) without any: a sixteenth at 2.8 a group, that is, in a
// row of 151,936 logits, at 420 tokens by the waves' maxima and at 1,650 by those of their rows; and there are one and a half times as many
// groups with a token as waves with one at 200 tokens, where a stretch of neighbours has four times as many.)  The waves' maxima, a quarter as
// many, say it of most rows: 256 rows under min-p of 0.05 52.0 us, by the others alone 52.6.
__device__ __forceinline__ bool fs_is_short(const FsSpace& w, float cut, float least) {
  const int n_waves = w.pieces * FS_PIECE_WAVES, n_rows = w.pieces * FS_PIECE_ROWS;
  const FsAbove waves = fs_above<8>(w.of_waves(), n_waves, cut, least);
  if (waves.cut * (FS_PIECE / FS_PIECE_WAVES) <= FS_LIST || 16 * (waves.least - waves.cut) >= waves.least) return true;
  const FsAbove rows = n_rows <= 12 * WAVE ? fs_above<12>(w.of_rows(), n_rows, cut, least) : fs_above<32>(w.of_rows(), n_rows, cut, least);
  return rows.cut * (FS_PIECE / FS_PIECE_ROWS) <= FS_LIST || 16 * (rows.least - rows.cut) >= rows.least || 2 * rows.cut <= 3 * waves.cut;
}

// A logit so that every token that counts is no smaller, and whether the list of those is known to be short.  (A list of more than FS_LIST tokens is one
// workgroup's, which reads the row again and again: rows of 151,936 flat logits (2.2 N(0, 1)) under min-p of 1e-6 took 359 us, under one of 0.01 at
// T = 1.5 106 to 468; rows of which only 20,000 neighbours are allowed, under top-k 40, 382 to 539.)
//   top-k: at least k of the maxima are no smaller; found by halving between the largest and the smallest logit that weighs
//   anything, and what the halvings leave undecided stays above the cut.  Fewer than k maxima say nothing: the list is then whatever weighs
//   anything.
//   min-p (where top-p cuts nothing): max + T ln(min_p), less what 32 bits may be off by: 4 roundings of each of its parts.
struct FsCut { float cut; bool is_short; };
__device__ __forceinline__ FsCut fs_cut(const FsSpace& w, const FsAsked& asked, const FsRow& r, float low, int vocab) {
  const float high = r.top, least = fmaxf(low, high - r.reach);          // (what lies further below weighs nothing)
  const int maxima = w.pieces * FS_PIECE_ROWS;
  FsCut c = {-INFINITY, false};
  if (fs_few_wanted(asked, vocab)) {
    // Few maxima while k is small beside their number (k = 40 of 152: some 50 tokens are no smaller; 150 of them: 700).
    c.cut = 2 * asked.top_k <= w.pieces * FS_PIECE_WAVES ? fs_cut_of_maxima<8>(w.of_waves(), w.pieces * FS_PIECE_WAVES, asked.top_k, least, high)
            : maxima <= 12 * WAVE                        ? fs_cut_of_maxima<12>(w.of_rows(), maxima, asked.top_k, least, high)
                                                         : fs_cut_of_maxima<32>(w.of_rows(), maxima, asked.top_k, least, high);
    c.is_short = c.cut > -INFINITY || fs_is_short(w, least, least);
  }
  if (fs_floor_alone(asked)) {
    const float down = -asked.temperature * logf(fminf(asked.min_p, 1.f));
    const float floor_cut = high - down - 4.8e-7f * (fabsf(high) + 2.f * down) - 1e-6f * asked.temperature;
    if (!c.is_short) c.is_short = fs_is_short(w, fmaxf(floor_cut, least), least);
    c.cut = fmaxf(c.cut, floor_cut);
  }
  return c;
}

// The tokens of piece `p` that `wanted` names, to the row's list: each thread's, their place among the workgroup's, and the
// workgroup's place in the list.
template <typename Wanted>
__device__ __forceinline__ void fs_append(const FsSpace& w, int p, const float (&v)[FS_EACH], FsSmall& s, Wanted wanted) {
  uint32_t held = 0;
#pragma unroll
  for (int j = 0; j < FS_EACH; ++j)
    if (wanted(v[j])) held |= 1u << j;
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  const int mine = __popc(held);
  int place = mine;
  for (int off = 1; off < WAVE; off <<= 1) {
    const int got = __shfl_up(place, off, WAVE);
    if (lane >= off) place += got;
  }
  if (lane == WAVE - 1) s.wave_count[wave] = (uint32_t)place;
  __syncthreads();
  place -= mine;
  uint32_t all = 0;
#pragma unroll
  for (int i = 0; i < FS_PIECE_WAVES; ++i) {
    if (i < wave) place += (int)s.wave_count[i];
    all += s.wave_count[i];
  }
  if (all == 0) return;                                    // (the same for the whole workgroup)
  if (threadIdx.x == 0) s.n_listed = atomicAdd(&w.head()->n_listed, (int)all);
  __syncthreads();
  place += s.n_listed;
#pragma unroll
  for (int j = 0; j < FS_EACH; ++j)
    if (held >> j & 1) {
      if (place < FS_LIST)
        w.list()[place] = (u64)fs_key(v[j]) << 32 | (uint32_t)~(uint32_t)(p * FS_PIECE + j * FS_THREADS + (int)threadIdx.x);
      ++place;
    }
}

template <typename T>
__global__ void __launch_bounds__(FS_THREADS)
sample_filtered_extents(FsArgs a) {
  __shared__ FsSmall s;
  const FsSpace w = fs_space(a, blockIdx.y);
  float v[FS_EACH], high, low, of_wave, of_row;
  int at;
  fs_load<FS_THREADS>((const T*)a.logits + (size_t)blockIdx.y * a.stride, blockIdx.x * FS_PIECE, a.vocab, v);
  fs_extent<FS_THREADS>(v, blockIdx.x * FS_PIECE, high, at, low, of_wave, of_row, s);
  FsExtent& e = w.extents()[blockIdx.x];
  if ((threadIdx.x & (WAVE - 1)) == 0) w.of_waves()[blockIdx.x * FS_PIECE_WAVES + threadIdx.x / WAVE] = of_wave;
  if ((threadIdx.x & 15) == 0) w.of_rows()[blockIdx.x * FS_PIECE_ROWS + threadIdx.x / 16] = of_row;
  if (threadIdx.x == 0) {
    e.high = high;
    e.low = low;
    e.at = at;
    if (blockIdx.x == 0) { w.head()->n_listed = w.head()->gathered = w.head()->listed = 0; }
  }
}

// The list, where it can be made at once and is short; else the bins of SPAN pieces.
template <typename T, int SPAN>
__global__ void __launch_bounds__(FS_THREADS)
sample_filtered_bins(FsArgs a) {
  __shared__ FsSmall s;
  const FsSpace w = fs_space(a, blockIdx.y);
  const FsAsked asked = fs_asked(a, blockIdx.y);
  const T* row = (const T*)a.logits + (size_t)blockIdx.y * a.stride;
  const int first = blockIdx.x * SPAN;
  float v[FS_EACH], high, low;
  if (fs_may_be_listed(asked, a.vocab)) {
    // (One wave works the cut out: eight halvings among six hundred maxima by every wave of 2,432 workgroups took 14 us of their time.)
    float of_row[SPAN], of_piece[SPAN];
#pragma unroll
    for (int j = 0; j < SPAN; ++j) {
      const int p = min(first + j, a.pieces - 1);
      of_row[j] = w.of_rows()[p * FS_PIECE_ROWS + threadIdx.x / 16];
      of_piece[j] = w.extents()[p].high;
    }
    fs_row_extent(w, high, low);
    if (!fs_is_drawn(asked.temperature, high)) return;
    const FsRow r = fs_row(asked.temperature, high, low);
    if (threadIdx.x < WAVE) {
      const FsCut found = fs_cut(w, asked, r, low, a.vocab);
      if (threadIdx.x == 0) {
        s.cut = found.cut;
        s.listed = found.is_short;
        if (blockIdx.x == 0) w.head()->listed = found.is_short;          // (every workgroup of the row finds the same)
      }
    }
    __syncthreads();
    if (s.listed) {
      const float cut = s.cut;
#pragma unroll
      for (int j = 0; j < SPAN; ++j) {
        const int p = first + j;
        if (p >= a.pieces || of_piece[j] < cut) continue;  // (the same for the whole workgroup)
        // Only lanes whose row of sixteen has something at or above the cut read their logits again: of 256 rows of 152,064 under min-p, 13
        // of 26 us of this pass were the second reading.
        fs_load<FS_THREADS>(row, p * FS_PIECE, a.vocab, v, of_row[j] >= cut);
        fs_append(w, p, v, s, [&](float x) { return x >= cut && r.top - x <= r.reach; });
        if (SPAN > 1) __syncthreads();
      }
      return;
    }
  }
  fs_load<FS_THREADS>(row, first * FS_PIECE, a.vocab, v);
  fs_row_extent(w, high, low);
  if (!fs_is_drawn(asked.temperature, high)) return;
  const FsRow r = fs_row(asked.temperature, high, low);
  fs_clear_bins(s);
  u64 over = 0;
  for (int p = first;;) {
    over += fs_fill_bins(v, r, asked, s);
    if (SPAN == 1 || ++p == min(first + SPAN, a.pieces)) break;
    fs_load<FS_THREADS>(row, p * FS_PIECE, a.vocab, v);
  }
  over = fs_sum<FS_THREADS>(over, s);
  FsBinned& mine = w.binned()[blockIdx.x];
  mine.mass[threadIdx.x] = s.mass[threadIdx.x];
  mine.count[threadIdx.x] = s.count[threadIdx.x];
  if (threadIdx.x == 0) mine.over = over;
}
static_assert(FS_THREADS == FS_BINS, "a thread a bin");

// The row's bins from its pieces', into `s`; the weight of what min-p keeps; and the ranges of bins in which the answers lie.
__device__ __forceinline__ FsRanges fs_settle(const FsSpace& w, const FsAsked& asked, u64& over, FsSmall& s) {
  u64 m = 0;
  uint32_t c = 0;
  over = 0;
  for (int first = 0; first < w.shares; first += 16) {     // (sixteen pieces asked for at a time)
    u64 of_mass[16];
    uint32_t of_count[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const FsBinned& piece = w.binned()[min(first + j, w.shares - 1)];
      of_mass[j] = piece.mass[threadIdx.x];
      of_count[j] = piece.count[threadIdx.x];
    }
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (first + j < w.shares) { m += of_mass[j]; c += of_count[j]; }
  }
  for (int p = threadIdx.x; p < w.shares; p += FS_THREADS) over += w.binned()[p].over;
  s.mass[threadIdx.x] = m;
  s.count[threadIdx.x] = c;
  over = fs_kept_by_floor(asked, fs_sum<FS_THREADS>(over, s));
  FsRunning run;
  run.of(s);
  return fs_ranges(run, asked, over);
}

// The draw from the row's list in the workspace, `n` tokens; `ranges` as in fs_draw.
template <typename T>
__device__ __forceinline__ void fs_draw_listed(const FsArgs& a, const FsSpace& w, const FsAsked& asked, const FsRow& r, int row_at,
                                               const FsRanges* ranges, u64 over, int n, FsShared& s) {
  for (int i = threadIdx.x; i < min(n, FS_LIST); i += FS_THREADS) s.list[i] = w.list()[i];
  __syncthreads();
  const int pick = fs_draw<FS_THREADS>(s, (const T*)a.logits + (size_t)row_at * a.stride, a.vocab, r, asked, ranges, over, n);
  if (threadIdx.x == 0) a.out[row_at] = pick;
}

// The tokens of SPAN pieces in the ranges, to the row's list.
template <int SPAN, typename T>
__device__ __forceinline__ void fs_gather(const FsArgs& a, const FsSpace& w, const T* row, const FsRow& r, const FsRanges& ranges, FsSmall& s) {
  const int last_bin = max(ranges.k_bin, max(ranges.p_last, ranges.draw_last));
#pragma unroll
  for (int j = 0; j < SPAN; ++j) {
    const int p = blockIdx.x * SPAN + j;
    if (SPAN > 1 && p >= a.pieces) break;                  // (the same for the whole workgroup)
    const float of_row = w.of_rows()[p * FS_PIECE_ROWS + threadIdx.x / 16];
    float v[FS_EACH];
    // (A row of sixteen lanes whose maximum lies behind all the ranges has nothing in them.)
    const bool wanted = r.top - of_row <= r.reach && fs_bin(of_row, r) <= last_bin;
    fs_load<FS_THREADS>(row, p * FS_PIECE, a.vocab, v, wanted);
    fs_append(w, p, v, s, [&](float x) { return r.top - x <= r.reach && ranges.has(fs_bin(x, r)); });
    if (SPAN > 1) __syncthreads();
  }
}

// Many rows.  A row whose list is there: its draw.  Another: its bins and ranges, left for its pieces, which gather; and its draw.
template <typename T>
__global__ void __launch_bounds__(FS_THREADS)
sample_filtered_settle(FsArgs a) {
  __shared__ FsShared s;
  const int row_at = blockIdx.x;
  const FsSpace w = fs_space(a, row_at);
  const FsAsked asked = fs_asked(a, row_at);
  const int listed = scalar_int(&w.head()->listed);
  float high, low;
  fs_row_extent(w, high, low);
  if (!fs_is_drawn(asked.temperature, high)) {
    const int at = fs_row_top(w, high);
    if (threadIdx.x == 0) a.out[row_at] = at;
    return;
  }
  if (listed) {
    fs_draw_listed<T>(a, w, asked, fs_row(asked.temperature, high, low), row_at, nullptr, 0, w.head()->n_listed, s);
    return;
  }
  u64 over;
  const FsRanges ranges = fs_settle(w, asked, over, s);
  w.whole()->mass[threadIdx.x] = s.mass[threadIdx.x];
  w.whole()->count[threadIdx.x] = s.count[threadIdx.x];
  if (threadIdx.x == 0) {
    FsHead& head = *w.head();
    head.ranges[0] = ranges.k_bin; head.ranges[1] = ranges.p_first; head.ranges[2] = ranges.p_last;
    head.ranges[3] = ranges.draw_first; head.ranges[4] = ranges.draw_last;
    head.over = over;
  }
}

__device__ __forceinline__ FsRanges fs_kept_ranges(const FsSpace& w) {
  const int* kept = w.head()->ranges;
  return FsRanges{scalar_int(kept), scalar_int(kept + 1), scalar_int(kept + 2), scalar_int(kept + 3), scalar_int(kept + 4)};
}

template <typename T, int SPAN>
__global__ void __launch_bounds__(FS_THREADS)
sample_filtered_gather(FsArgs a) {
  __shared__ FsSmall s;
  const FsSpace w = fs_space(a, blockIdx.y);
  const FsAsked asked = fs_asked(a, blockIdx.y);
  if (scalar_int(&w.head()->listed)) return;
  float high, low;
  fs_row_extent(w, high, low);
  if (!fs_is_drawn(asked.temperature, high)) return;
  fs_gather<SPAN>(a, w, (const T*)a.logits + (size_t)blockIdx.y * a.stride, fs_row(asked.temperature, high, low), fs_kept_ranges(w), s);
}

template <typename T>
__global__ void __launch_bounds__(FS_THREADS)
sample_filtered_draw(FsArgs a) {
  __shared__ FsShared s;
  const FsSpace w = fs_space(a, blockIdx.x);
  const FsAsked asked = fs_asked(a, blockIdx.x);
  if (scalar_int(&w.head()->listed)) return;
  float high, low;
  fs_row_extent(w, high, low);
  if (!fs_is_drawn(asked.temperature, high)) return;
  s.mass[threadIdx.x] = w.whole()->mass[threadIdx.x];
  s.count[threadIdx.x] = w.whole()->count[threadIdx.x];
  const FsRanges ranges = fs_kept_ranges(w);
  fs_draw_listed<T>(a, w, asked, fs_row(asked.temperature, high, low), blockIdx.x, &ranges, w.head()->over, w.head()->n_listed, s);
}

// Few rows, where a launch counts: every piece's workgroup adds the row's bins up for itself, gathers, and the one that comes last in its row
// finds the whole list there and draws.  (Nobody waits: each leaves its tokens, then counts itself in.)  The draw's LDS lets one
// workgroup onto a compute unit.
template <typename T>
__global__ void __launch_bounds__(FS_THREADS)
sample_filtered_finish(FsArgs a) {
  __shared__ FsShared s;
  __shared__ int came;
  const int row_at = blockIdx.y;
  const FsSpace w = fs_space(a, row_at);
  const FsAsked asked = fs_asked(a, row_at);
  const bool listed = scalar_int(&w.head()->listed);
  if (listed && blockIdx.x > 0) return;
  float high, low;
  fs_row_extent(w, high, low);
  if (!fs_is_drawn(asked.temperature, high)) {
    const int at = fs_row_top(w, high);
    if (threadIdx.x == 0 && blockIdx.x == 0) a.out[row_at] = at;
    return;
  }
  const FsRow r = fs_row(asked.temperature, high, low);
  if (listed) {
    fs_draw_listed<T>(a, w, asked, r, row_at, nullptr, 0, w.head()->n_listed, s);
    return;
  }
  u64 over;
  const FsRanges ranges = fs_settle(w, asked, over, s);
  fs_gather<1>(a, w, (const T*)a.logits + (size_t)row_at * a.stride, r, ranges, s);
  // Every wave waits for its own tokens to have come to the chiplet's cache: a barrier does not wait for stores to global memory (its fences are
  // the workgroup's, whose waves see each other's through the compute unit's cache), and one wave's fence waits for that wave's stores.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {                                  // (what is in that cache one thread's fences bring out, and in, for all)
    __threadfence();                                       // the tokens are there for all that see the count
    came = atomicAdd(&w.head()->gathered, 1);
    __threadfence();                                       // and so is what the others left before they counted themselves in
  }
  __syncthreads();
  if (came != w.shares - 1) return;                        // (the same for the whole workgroup)
  const int n = __hip_atomic_load(&w.head()->n_listed, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  fs_draw_listed<T>(a, w, asked, r, row_at, &ranges, over, n, s);
}

#define FS_MAX_VOCAB (1 << 19)
static_assert((FS_MAX_VOCAB / FS_PIECE) * FS_PIECE_WAVES <= 8 * WAVE && (FS_MAX_VOCAB / FS_PIECE) * FS_PIECE_ROWS <= 32 * WAVE,
              "the maxima that fs_cut holds");

static bool fs_is_short(int vocab) { return vocab <= FS_SHORT_THREADS * FS_SHORT_EACH; }
static int fs_pieces(int vocab) { return (vocab + FS_PIECE - 1) / FS_PIECE; }

// Bytes of workspace a row needs (a multiple of 16; none for a short row).
extern "C" int ta_sample_filtered_workspace(int vocab) { return fs_is_short(vocab) ? 0 : (int)fs_row_bytes(fs_pieces(vocab)); }

// The passes of long rows behind the first: so many pieces a workgroup.
template <typename T, int SPAN>
static int launch_long(FsArgs a, int n_rows, hipStream_t stream) {
  a.shares = (a.pieces + SPAN - 1) / SPAN;
  const dim3 grid(a.shares, n_rows);
  sample_filtered_bins<T, SPAN><<<grid, FS_THREADS, 0, stream>>>(a);
  int status = LAUNCH_STATUS();
  if (status) return status;
  if (SPAN == 1 && a.pieces * n_rows <= FS_FEW_PIECES) {
    sample_filtered_finish<T><<<grid, FS_THREADS, 0, stream>>>(a);
    return LAUNCH_STATUS();
  }
  sample_filtered_settle<T><<<n_rows, FS_THREADS, 0, stream>>>(a);
  status = LAUNCH_STATUS();
  if (status) return status;
  sample_filtered_gather<T, SPAN><<<grid, FS_THREADS, 0, stream>>>(a);
  status = LAUNCH_STATUS();
  if (status) return status;
  sample_filtered_draw<T><<<n_rows, FS_THREADS, 0, stream>>>(a);
  return LAUNCH_STATUS();
}

template <typename T>
static int launch_filtered(FsArgs a, int n_rows, hipStream_t stream) {
  if (fs_is_short(a.vocab)) {
    if (a.vocab <= FS_SHORT_THREADS * FS_SHORT_EACH / 4)
      sample_filtered_short<T, FS_SHORT_EACH / 4><<<n_rows, FS_SHORT_THREADS, 0, stream>>>(a);
    else
      sample_filtered_short<T, FS_SHORT_EACH><<<n_rows, FS_SHORT_THREADS, 0, stream>>>(a);
    return LAUNCH_STATUS();
  }
  sample_filtered_extents<T><<<dim3(a.pieces, n_rows), FS_THREADS, 0, stream>>>(a);
  const int status = LAUNCH_STATUS();
  if (status) return status;
  return (int64_t)a.pieces * n_rows >= FS_MANY_PIECES ? launch_long<T, FS_SPAN>(a, n_rows, stream) : launch_long<T, 1>(a, n_rows, stream);
}

// logits [n_rows, vocab] (float or bfloat16), rows `stride` elements apart; the others one number a row; workspace: n_rows *
// ta_sample_filtered_workspace(vocab) bytes at a multiple of 16.
extern "C" int ta_sample_filtered(const void* logits, int64_t stride, const void* temperature, const void* top_k, const void* top_p,
                                  const void* min_p, const void* uniform, void* out, void* workspace, int n_rows, int vocab, int dtype,
                                  hipStream_t stream) {
  if (n_rows <= 0) return 0;
  if (vocab < 1 || vocab > FS_MAX_VOCAB || stride < 0 || n_rows > 65535) return -1;
  if (!logits || !temperature || !top_k || !top_p || !min_p || !uniform || !out || (!workspace && !fs_is_short(vocab))) return -1;
  FsArgs a;
  a.logits = logits; a.stride = stride; a.temperature = (const float*)temperature; a.top_p = (const float*)top_p;
  a.min_p = (const float*)min_p; a.uniform = (const float*)uniform; a.top_k = (const int*)top_k; a.out = (int*)out;
  a.vocab = vocab; a.pieces = fs_pieces(vocab); a.shares = a.pieces; a.workspace = (char*)workspace;
  a.row_bytes = fs_row_bytes(a.pieces);
  return dtype == DT_F32 ? launch_filtered<float>(a, n_rows, stream) : launch_filtered<bf16_t>(a, n_rows, stream);
}
