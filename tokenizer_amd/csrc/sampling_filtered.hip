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
// by 2^-45 of the row's largest at most: 32-bit weights would move the border between two tokens of a flat row of 150,000 by a good
// part of a token.  Tokens that weigh nothing then (31.2 T below the maximum) are never drawn.
//
// No row is sorted whole.  Its tokens fall into FS_BINS ranges of logit, equal parts of what lies between the maximum and the lowest
// logit that weighs anything, each with its count and weight; the three questions then lie in a few ranges (what is not known
// yet of an earlier answer is at most a range's weight), whose tokens, some hundreds, are gathered and sorted in LDS.  Should there
// be more than FS_LIST of them (thousands of equal logits), a range is narrowed by counting instead, key by key.
//
// NaN is no token.  A row without a finite maximum, and a row whose temperature is not positive, gets its first maximum (0 if it
// holds no number).
#include "common.h"

#define FS_THREADS 1024
#define FS_WAVES (FS_THREADS / WAVE)
#define FS_EACH 20                      // logits a thread holds
#define FS_PIECE (FS_THREADS * FS_EACH)
#define FS_BINS 256                     // four a lane
#define FS_LIST 8192
#define FS_SLOTS 1024                   // ranges a round of narrowing tells apart, one a thread
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

struct FsShared {
  union {
    u64 list[FS_LIST];                  // the gathered tokens, key in the upper half, the index's complement in the lower
    struct { u64 mass[FS_SLOTS]; uint32_t count[FS_SLOTS]; } slots;      // a round of narrowing
  };
  u64 mass[FS_BINS];                    // the bins, whole row
  uint32_t count[FS_BINS];
  u64 missing_mass[FS_BINS];            // of bins that were not gathered, in front of this one
  uint32_t missing_count[FS_BINS];
  u64 wave_mass[FS_WAVES];
  uint32_t wave_count[FS_WAVES];
  float wave_low[FS_WAVES], wave_high[FS_WAVES];
  int wave_at[FS_WAVES];
  u64 found_mass, kept;
  uint32_t found_count;
  int found, n_listed;
  uint32_t key_low, key_high;
};

__device__ __forceinline__ u64 fs_up(u64 v, int off, int lane) {          // the value `off` lanes down, 0 where there is none
  const u64 got = __shfl_up(v, off, WAVE);
  return lane >= off ? got : 0;
}

// Sum over the workgroup, to every thread.
__device__ __forceinline__ u64 fs_sum(u64 v, FsShared& s) {
  for (int off = WAVE / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, WAVE);
  __syncthreads();
  if ((threadIdx.x & (WAVE - 1)) == 0) s.wave_mass[threadIdx.x / WAVE] = v;
  __syncthreads();
  u64 total = 0;
  for (int w = 0; w < FS_WAVES; ++w) total += s.wave_mass[w];
  return total;
}

// The logits of a piece in registers: thread i has logits i, i + FS_THREADS, ...; NaN where there is none.
template <typename T>
__device__ __forceinline__ void fs_load(const T* __restrict__ row, int begin, int vocab, float (&v)[FS_EACH]) {
#pragma unroll
  for (int j = 0; j < FS_EACH; ++j) v[j] = ld(row + min(begin + j * FS_THREADS + (int)threadIdx.x, vocab - 1));
#pragma unroll
  for (int j = 0; j < FS_EACH; ++j)
    if (begin + j * FS_THREADS + (int)threadIdx.x >= vocab) v[j] = __uint_as_float(0x7fc00000u);
}

// The largest of a piece's logits, its lowest index, and the smallest above -inf, to every thread.
__device__ __forceinline__ void fs_extent(const float (&v)[FS_EACH], int begin, float& high, int& at, float& low, FsShared& s) {
  high = -INFINITY;
  low = INFINITY;
  at = 0x7fffffff;
#pragma unroll
  for (int j = 0; j < FS_EACH; ++j) {
    if (v[j] > high) { high = v[j]; at = begin + j * FS_THREADS + (int)threadIdx.x; }
    if (v[j] > -INFINITY) low = fminf(low, v[j]);
  }
  for (int off = WAVE / 2; off > 0; off >>= 1) {
    const float other = __shfl_xor(high, off, WAVE);
    const int other_at = __shfl_xor(at, off, WAVE);
    if (other > high || (other == high && other_at < at)) { high = other; at = other_at; }
    low = fminf(low, __shfl_xor(low, off, WAVE));
  }
  const int wave = threadIdx.x / WAVE;
  if ((threadIdx.x & (WAVE - 1)) == 0) { s.wave_high[wave] = high; s.wave_at[wave] = at; s.wave_low[wave] = low; }
  __syncthreads();
  for (int w = 0; w < FS_WAVES; ++w) {
    if (s.wave_high[w] > high || (s.wave_high[w] == high && s.wave_at[w] < at)) { high = s.wave_high[w]; at = s.wave_at[w]; }
    low = fminf(low, s.wave_low[w]);
  }
}

// A piece's bins into `s.mass` and (if `counted`) `s.count`, and the weight of its tokens that min-p keeps, to every thread.
__device__ __forceinline__ u64 fs_fill_bins(const float (&v)[FS_EACH], const FsRow& r, const FsAsked& asked, FsShared& s) {
  const bool counted = asked.top_k > 0, floored = asked.min_p > 0.f;
  const double floor_share = (double)asked.min_p * FS_UNIT;
  if (threadIdx.x < FS_BINS) { s.mass[threadIdx.x] = 0; s.count[threadIdx.x] = 0; }
  __syncthreads();
  u64 over = 0;
#pragma unroll
  for (int j = 0; j < FS_EACH; ++j) {
    if (r.top - v[j] <= r.reach) {                         // (false for NaN)
      const double share = fs_share(v[j], r);
      const u64 w = fs_whole(share);
      const int bin = fs_bin(v[j], r);
      atomicAdd(&s.mass[bin], w);
      if (counted) atomicAdd(&s.count[bin], 1u);
      if (!floored || !(share < floor_share) || v[j] == r.top) over += w;
    }
  }
  return fs_sum(over, s);                                  // (its barriers stand behind the bins, too)
}

// A wave's view of the bins: running counts and weights, bins 4 lane .. + 3.
struct FsRunning {
  u64 mass[4];
  uint32_t count[4];
  __device__ __forceinline__ void of(const FsShared& s) {
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
// Narrowing, for ranges of more tokens than are sorted: the row is read again for every round.

// Where the order of the slots, the last one first, reaches a number (the running count if `counting`, else the running mass).  Returns the
// slot, and what lies before it in `count` and `mass`; -1 if the whole order does not reach it.
__device__ int fs_reach(FsShared& s, bool forwards, bool counting, u64 need, uint32_t& count, u64& mass) {
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  const int slot = forwards ? threadIdx.x : FS_SLOTS - 1 - threadIdx.x;
  const u64 m = s.slots.mass[slot];
  const u64 c = s.slots.count[slot];
  u64 run_m = m, run_c = c;
  for (int off = 1; off < WAVE; off <<= 1) {
    run_m += fs_up(run_m, off, lane);
    run_c += fs_up(run_c, off, lane);
  }
  __syncthreads();
  if (threadIdx.x == 0) s.found = -1;
  if (lane == WAVE - 1) { s.wave_mass[wave] = run_m; s.wave_count[wave] = (uint32_t)run_c; }
  __syncthreads();
  u64 before_m = run_m - m, before_c = run_c - c;
  for (int w = 0; w < wave; ++w) { before_m += s.wave_mass[w]; before_c += s.wave_count[w]; }
  const u64 before = counting ? before_c : before_m, here = counting ? c : m;
  if (before < need && before + here >= need) {            // one thread
    s.found = slot;
    s.found_mass = before_m;
    s.found_count = (uint32_t)before_c;
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
  s.slots.mass[threadIdx.x] = 0;
  s.slots.count[threadIdx.x] = 0;
  __syncthreads();
}

// Calls use(value, index) for every number of the row, a thread every FS_THREADS-th one, eight loads asked for at a time.
template <typename T, typename Use>
__device__ __forceinline__ void fs_numbers(const T* __restrict__ row, int vocab, Use use) {
  for (int base = threadIdx.x; base < vocab; base += 8 * FS_THREADS) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = ld(row + min(base + j * FS_THREADS, vocab - 1));
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (base + j * FS_THREADS < vocab && v[j] == v[j]) use(v[j], base + j * FS_THREADS);
  }
}

// The key at which the order reaches a number, what lies before the tokens of that key, and what each of them weighs.
struct FsCrossing {
  uint32_t key, before_count;
  u64 before_mass, each;
};

template <typename T>
__device__ FsCrossing fs_narrow(FsShared& s, const T* row, int vocab, const FsRow& r, int bin, bool counting, u64 need, uint32_t before_count,
                                u64 before_mass) {
  uint32_t low = 0xffffffffu, high = 0;
  fs_numbers(row, vocab, [&](float v, int) {
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
    fs_numbers(row, vocab, [&](float v, int) {
      if (r.top - v <= r.reach && fs_bin(v, r) == bin) {
        const uint32_t key = fs_key(v);
        if (key >= low && key <= high) {
          atomicAdd(&s.slots.count[(key - low) >> shift], 1u);
          atomicAdd(&s.slots.mass[(key - low) >> shift], fs_weight(v, r));
        }
      }
    });
    __syncthreads();
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

template <typename T>
__device__ int fs_draw_by_narrowing(FsShared& s, const T* row, int vocab, const FsRow& r, const FsAsked& asked, const FsRunning& run, u64 over) {
  auto crossing = [&](int bin, bool counting, u64 need) {
    return fs_narrow(s, row, vocab, r, bin, counting, need, run.count_to(bin - 1), run.mass_to(bin - 1));
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
  fs_numbers(row, vocab, [&](float v, int at) {
    if (fs_key(v) == x.key) atomicAdd(&s.slots.count[at / per], 1u);
  });
  __syncthreads();
  uint32_t before = 0;
  u64 unused;
  const int part = fs_reach(s, true, true, rank, before, unused);
  if (threadIdx.x == 0) {
    int pick = 0;
    u64 left = rank - before;
    for (int i = part < 0 ? vocab : part * per; i < min(vocab, (part + 1) * per); ++i) {
      const float v = ld(row + i);
      if (v == v && fs_key(v) == x.key && --left == 0) { pick = i; break; }
    }
    s.found = pick;
  }
  __syncthreads();
  return s.found;
}

// ------------------------------------------------------------------------------------------------
// The draw, with the bins of the whole row in `s.mass` and `s.count`: from the `n` gathered tokens in `s.list` (in any order) if they all
// found room there, else by narrowing.
template <typename T>
__device__ int fs_draw(FsShared& s, const T* row, int vocab, const FsRow& r, const FsAsked& asked, const FsRunning& run,
                       const FsRanges& ranges, u64 over, int n) {
  if (n > FS_LIST) return fs_draw_by_narrowing(s, row, vocab, r, asked, run, over);
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  if (wave == 0) {                                         // what lies between the gathered bins
    u64 m[4], c[4], run_m = 0, run_c = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool gathered = ranges.has(4 * lane + j);
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
  int size = WAVE;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += FS_THREADS) s.list[i] = 0;        // (behind every token)
  __syncthreads();
  // Sorted by exchanges, the largest first: runs of `run_of` fall and rise in turn until one is left.
  for (int run_of = 2; run_of <= size; run_of <<= 1)
    for (int apart = run_of >> 1; apart > 0; apart >>= 1) {
      for (int i = threadIdx.x; i < size / 2; i += FS_THREADS) {
        const int a = 2 * i - (i & (apart - 1)), b = a + apart;
        const u64 x = s.list[a], y = s.list[b];
        if ((x < y) == ((a & run_of) == 0)) { s.list[a] = y; s.list[b] = x; }
      }
      __syncthreads();
    }
  // Running weights: a thread has `per` neighbours of the list.
  constexpr int MOST = FS_LIST / FS_THREADS;
  const int per = max(1, size / FS_THREADS);
  u64 token[MOST], w[MOST], sum = 0;
#pragma unroll
  for (int j = 0; j < MOST; ++j) {
    const int i = threadIdx.x * per + j;
    token[j] = 0;
    w[j] = 0;
    if (j < per && i < n) {
      token[j] = s.list[i];
      w[j] = fs_weight(fs_value((uint32_t)(token[j] >> 32)), r);
    }
    sum += w[j];
  }
  u64 before = sum;
  for (int off = 1; off < WAVE; off <<= 1) before += fs_up(before, off, lane);
  if (lane == WAVE - 1) s.wave_mass[wave] = before;
  before -= sum;
  const u64 total = run.mass_to(FS_BINS - 1);              // (the whole wave takes part)
  if (threadIdx.x == 0) {
    s.kept = total;
    s.found = (int)~(uint32_t)s.list[0];
  }
  __syncthreads();
  for (int i = 0; i < wave; ++i) before += s.wave_mass[i];
  u64 at_mass[MOST];                                       // what stands before a token in the whole order
#pragma unroll
  for (int j = 0; j < MOST; ++j) {
    at_mass[j] = before;
    before += w[j];
    if (token[j]) {
      const int bin = fs_bin(fs_value((uint32_t)(token[j] >> 32)), r);
      at_mass[j] += s.missing_mass[bin];
      if (ranges.k_bin >= 0 && s.missing_count[bin] + threadIdx.x * per + j + 1 == (uint32_t)asked.top_k) s.kept = at_mass[j] + w[j];
    }
  }
  __syncthreads();
  u64 kept = s.kept;
  if (asked.top_p < 1.f) {
    __syncthreads();
    const u64 need = fs_need_of_share(asked.top_p, kept);
#pragma unroll
    for (int j = 0; j < MOST; ++j)
      if (token[j] && at_mass[j] < need && at_mass[j] + w[j] >= need) s.kept = at_mass[j] + w[j];
    __syncthreads();
    kept = s.kept;
  }
  kept = over < kept ? over : kept;
  const u64 need = fs_need_of_draw(asked.uniform, kept);
#pragma unroll
  for (int j = 0; j < MOST; ++j)
    if (token[j] && at_mass[j] < need && at_mass[j] + w[j] >= need) s.found = (int)~(uint32_t)token[j];
  __syncthreads();
  return s.found;
}

struct FsArgs {
  const void* logits;
  int64_t stride;
  const float *temperature, *top_p, *min_p, *uniform;
  const int* top_k;
  int* out;
  int vocab, pieces;
  char* workspace;
  size_t row_bytes;
};

__device__ __forceinline__ FsAsked fs_asked(const FsArgs& a, int row) {
  FsAsked q;
  q.temperature = a.temperature[row];
  q.top_p = a.top_p[row];
  q.min_p = a.min_p[row];
  q.uniform = a.uniform[row];
  q.top_k = a.top_k[row];
  return q;
}

// A row of at most FS_PIECE logits: one workgroup, one launch.
template <typename T>
__global__ void __launch_bounds__(FS_THREADS)
sample_filtered_short(FsArgs a) {
  __shared__ FsShared s;
  const int row_at = blockIdx.x;
  const T* row = (const T*)a.logits + (size_t)row_at * a.stride;
  const FsAsked asked = fs_asked(a, row_at);
  float v[FS_EACH], high, low;
  int at;
  fs_load(row, 0, a.vocab, v);
  fs_extent(v, 0, high, at, low, s);
  if (!fs_is_drawn(asked.temperature, high)) {
    if (threadIdx.x == 0) a.out[row_at] = at == 0x7fffffff ? 0 : at;
    return;
  }
  const FsRow r = fs_row(asked.temperature, high, low);
  const u64 over = fs_fill_bins(v, r, asked, s);
  FsRunning run;
  run.of(s);
  const FsRanges ranges = fs_ranges(run, asked, over);
  if (threadIdx.x == 0) s.n_listed = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < FS_EACH; ++j)
    if (r.top - v[j] <= r.reach && ranges.has(fs_bin(v[j], r))) {
      const int place = atomicAdd(&s.n_listed, 1);
      if (place < FS_LIST) s.list[place] = (u64)fs_key(v[j]) << 32 | (uint32_t)~(uint32_t)(j * FS_THREADS + (int)threadIdx.x);
    }
  __syncthreads();
  const int pick = fs_draw(s, row, a.vocab, r, asked, run, ranges, over, s.n_listed);
  if (threadIdx.x == 0) a.out[row_at] = pick;
}

// A longer row: its pieces' workgroups leave what they found in the workspace, a launch a step.
struct FsExtent { float high, low; int at, unused; };
__device__ __host__ __forceinline__ size_t fs_bins_at(int pieces) { return 16 + sizeof(FsExtent) * (size_t)pieces; }
__device__ __host__ __forceinline__ size_t fs_whole_at(int pieces) { return fs_bins_at(pieces) + (size_t)pieces * (12 * FS_BINS + 8); }
__device__ __host__ __forceinline__ size_t fs_list_at(int pieces) { return fs_whole_at(pieces) + 12 * FS_BINS + 8; }
// Per row: how many tokens were gathered (and 12 bytes of nothing); the pieces' extents; the pieces' bins (weights, then counts, then the
// weight that min-p keeps); those of the whole row; the gathered tokens.
struct FsSpace {
  char* base;
  int pieces;
  __device__ __forceinline__ int* n_listed() const { return (int*)base; }
  __device__ __forceinline__ FsExtent* extents() const { return (FsExtent*)(base + 16); }
  __device__ __forceinline__ u64* mass(int piece) const { return (u64*)(base + fs_bins_at(pieces) + (size_t)piece * (12 * FS_BINS + 8)); }
  __device__ __forceinline__ u64* whole() const { return (u64*)(base + fs_whole_at(pieces)); }
  __device__ __forceinline__ u64* list() const { return (u64*)(base + fs_list_at(pieces)); }
};
__device__ __forceinline__ FsSpace fs_space(const FsArgs& a, int row) { return FsSpace{a.workspace + (size_t)row * a.row_bytes, a.pieces}; }

__device__ __forceinline__ void fs_row_extent(const FsSpace& w, float& high, int& at, float& low) {
  high = -INFINITY;
  low = INFINITY;
  at = 0x7fffffff;
  for (int p = 0; p < w.pieces; ++p) {
    const FsExtent e = w.extents()[p];
    if (e.high > high) { high = e.high; at = e.at; }       // (pieces in the order of their indices)
    low = fminf(low, e.low);
  }
}

template <typename T>
__global__ void __launch_bounds__(FS_THREADS)
sample_filtered_extents(FsArgs a) {
  __shared__ FsShared s;
  const FsSpace w = fs_space(a, blockIdx.y);
  float v[FS_EACH], high, low;
  int at;
  fs_load((const T*)a.logits + (size_t)blockIdx.y * a.stride, blockIdx.x * FS_PIECE, a.vocab, v);
  fs_extent(v, blockIdx.x * FS_PIECE, high, at, low, s);
  if (threadIdx.x == 0) {
    w.extents()[blockIdx.x] = FsExtent{high, low, at, 0};
    if (blockIdx.x == 0) *w.n_listed() = 0;
  }
}

template <typename T>
__global__ void __launch_bounds__(FS_THREADS)
sample_filtered_bins(FsArgs a) {
  __shared__ FsShared s;
  const FsSpace w = fs_space(a, blockIdx.y);
  const FsAsked asked = fs_asked(a, blockIdx.y);
  float v[FS_EACH], high, low;
  int at;
  fs_load((const T*)a.logits + (size_t)blockIdx.y * a.stride, blockIdx.x * FS_PIECE, a.vocab, v);
  fs_row_extent(w, high, at, low);
  if (!fs_is_drawn(asked.temperature, high)) return;
  const u64 over = fs_fill_bins(v, fs_row(asked.temperature, high, low), asked, s);
  u64* mass = w.mass(blockIdx.x);
  uint32_t* count = (uint32_t*)(mass + FS_BINS + 1);
  if (threadIdx.x < FS_BINS) {
    mass[threadIdx.x] = s.mass[threadIdx.x];
    count[threadIdx.x] = s.count[threadIdx.x];
  }
  if (threadIdx.x == 0) mass[FS_BINS] = over;
}

template <typename T>
__global__ void __launch_bounds__(FS_THREADS)
sample_filtered_gather(FsArgs a) {
  __shared__ FsShared s;
  const FsSpace w = fs_space(a, blockIdx.y);
  const FsAsked asked = fs_asked(a, blockIdx.y);
  float v[FS_EACH], high, low;
  int at;
  fs_load((const T*)a.logits + (size_t)blockIdx.y * a.stride, blockIdx.x * FS_PIECE, a.vocab, v);
  fs_row_extent(w, high, at, low);
  if (!fs_is_drawn(asked.temperature, high)) return;
  const FsRow r = fs_row(asked.temperature, high, low);
  if (threadIdx.x < FS_BINS) {
    u64 m = 0;
    uint32_t c = 0;
    for (int p = 0; p < a.pieces; ++p) {
      m += w.mass(p)[threadIdx.x];
      c += ((const uint32_t*)(w.mass(p) + FS_BINS + 1))[threadIdx.x];
    }
    s.mass[threadIdx.x] = m;
    s.count[threadIdx.x] = c;
    if (blockIdx.x == 0) {
      w.whole()[threadIdx.x] = m;
      ((uint32_t*)(w.whole() + FS_BINS + 1))[threadIdx.x] = c;
    }
  }
  u64 over = 0;
  for (int p = 0; p < a.pieces; ++p) over += w.mass(p)[FS_BINS];
  if (blockIdx.x == 0 && threadIdx.x == 0) w.whole()[FS_BINS] = over;
  __syncthreads();
  FsRunning run;
  run.of(s);
  const FsRanges ranges = fs_ranges(run, asked, over);
  // Each thread's tokens in the ranges, their place in the workgroup's, and the workgroup's place in the row's list.
  uint32_t mine = 0, held = 0;
#pragma unroll
  for (int j = 0; j < FS_EACH; ++j)
    if (r.top - v[j] <= r.reach && ranges.has(fs_bin(v[j], r))) { ++mine; held |= 1u << j; }
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  int place = (int)mine;
  for (int off = 1; off < WAVE; off <<= 1) {
    const int got = __shfl_up(place, off, WAVE);
    if (lane >= off) place += got;
  }
  if (lane == WAVE - 1) s.wave_count[wave] = (uint32_t)place;
  __syncthreads();
  place -= (int)mine;
  uint32_t all = 0;
  for (int i = 0; i < FS_WAVES; ++i) {
    if (i < wave) place += (int)s.wave_count[i];
    all += s.wave_count[i];
  }
  if (threadIdx.x == 0) s.n_listed = all ? atomicAdd(w.n_listed(), (int)all) : 0;
  __syncthreads();
  place += s.n_listed;
#pragma unroll
  for (int j = 0; j < FS_EACH; ++j)
    if (held >> j & 1) {
      if (place < FS_LIST)
        w.list()[place] = (u64)fs_key(v[j]) << 32 | (uint32_t)~(uint32_t)(blockIdx.x * FS_PIECE + j * FS_THREADS + (int)threadIdx.x);
      ++place;
    }
}

template <typename T>
__global__ void __launch_bounds__(FS_THREADS)
sample_filtered_draw(FsArgs a) {
  __shared__ FsShared s;
  const int row_at = blockIdx.x;
  const FsSpace w = fs_space(a, row_at);
  const FsAsked asked = fs_asked(a, row_at);
  float high, low;
  int at;
  fs_row_extent(w, high, at, low);
  if (!fs_is_drawn(asked.temperature, high)) {
    if (threadIdx.x == 0) a.out[row_at] = at == 0x7fffffff ? 0 : at;
    return;
  }
  const int n = *w.n_listed();
  if (threadIdx.x < FS_BINS) {
    s.mass[threadIdx.x] = w.whole()[threadIdx.x];
    s.count[threadIdx.x] = ((const uint32_t*)(w.whole() + FS_BINS + 1))[threadIdx.x];
  }
  for (int i = threadIdx.x; i < min(n, FS_LIST); i += FS_THREADS) s.list[i] = w.list()[i];
  const u64 over = w.whole()[FS_BINS];
  __syncthreads();
  FsRunning run;
  run.of(s);
  const FsRanges ranges = fs_ranges(run, asked, over);
  const int pick = fs_draw(s, (const T*)a.logits + (size_t)row_at * a.stride, a.vocab, fs_row(asked.temperature, high, low), asked, run, ranges,
                           over, n);
  if (threadIdx.x == 0) a.out[row_at] = pick;
}

#define FS_MAX_VOCAB (1 << 19)

static int fs_pieces(int vocab) { return (vocab + FS_PIECE - 1) / FS_PIECE; }

// Bytes of workspace a row needs (a multiple of 16; none up to FS_PIECE logits).
extern "C" int ta_sample_filtered_workspace(int vocab) {
  const int pieces = fs_pieces(vocab);
  return pieces <= 1 ? 0 : (int)((fs_list_at(pieces) + 8 * FS_LIST + 15) / 16 * 16);
}

template <typename T>
static int launch_filtered(FsArgs a, int n_rows, hipStream_t stream) {
  if (a.pieces <= 1) {
    sample_filtered_short<T><<<n_rows, FS_THREADS, 0, stream>>>(a);
    return LAUNCH_STATUS();
  }
  const dim3 grid(a.pieces, n_rows);
  sample_filtered_extents<T><<<grid, FS_THREADS, 0, stream>>>(a);
  int status = LAUNCH_STATUS();
  if (status) return status;
  sample_filtered_bins<T><<<grid, FS_THREADS, 0, stream>>>(a);
  status = LAUNCH_STATUS();
  if (status) return status;
  sample_filtered_gather<T><<<grid, FS_THREADS, 0, stream>>>(a);
  status = LAUNCH_STATUS();
  if (status) return status;
  sample_filtered_draw<T><<<n_rows, FS_THREADS, 0, stream>>>(a);
  return LAUNCH_STATUS();
}

// logits [n_rows, vocab] (float or bfloat16), rows `stride` elements apart; the others one number a row; workspace: n_rows *
// ta_sample_filtered_workspace(vocab) bytes at a multiple of 16.
extern "C" int ta_sample_filtered(const void* logits, int64_t stride, const void* temperature, const void* top_k, const void* top_p,
                                  const void* min_p, const void* uniform, void* out, void* workspace, int n_rows, int vocab, int dtype,
                                  hipStream_t stream) {
  if (n_rows <= 0) return 0;
  if (vocab < 1 || vocab > FS_MAX_VOCAB || stride < 0 || n_rows > 65535) return -1;
  if (!logits || !temperature || !top_k || !top_p || !min_p || !uniform || !out || (!workspace && fs_pieces(vocab) > 1)) return -1;
  FsArgs a;
  a.logits = logits; a.stride = stride; a.temperature = (const float*)temperature; a.top_p = (const float*)top_p;
  a.min_p = (const float*)min_p; a.uniform = (const float*)uniform; a.top_k = (const int*)top_k; a.out = (int*)out;
  a.vocab = vocab; a.pieces = fs_pieces(vocab); a.workspace = (char*)workspace;
  a.row_bytes = (size_t)ta_sample_filtered_workspace(vocab);
  return dtype == DT_F32 ? launch_filtered<float>(a, n_rows, stream) : launch_filtered<bf16_t>(a, n_rows, stream);
}
