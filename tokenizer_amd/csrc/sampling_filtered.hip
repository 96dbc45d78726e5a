// Draws under temperature, top-k, top-p and min-p from given uniform numbers.
//
// The tokens of a row stand in the order of falling logit, lower index first among equals; token i weighs
// w_i = exp((l_i - max) / T).  Kept are the first k of the order (k <= 0: all of them), of those the shortest prefix that reaches
// top_p of their weight (top_p >= 1: all), of those the tokens with w_i >= min_p.  Every cut keeps a prefix of the one order, so what
// is kept is the shortest of the three prefixes, and the draw is the first token of the whole order whose running weight exceeds
// uniform * (weight of what is kept).  A draw is therefore three questions, "where does the running count or the running weight of
// the order reach a number": no row is sorted.
//
// Weights are whole numbers, w_i * 2^44 rounded to nearest (the exponential in 64 bits).  Sums of whole numbers do not depend on their
// order, so a draw is the same however a row is cut over threads, and up to 2^19 tokens' sum stays within 63 bits.  A weight is off by
// 2^-45 of the row's largest at most: 32-bit weights would move the border between two tokens of a flat row of 150,000 by a good
// part of a token.  Tokens that weigh nothing then (31.2 T below the maximum) are never drawn.
//
// NaN is no token.  A row without a finite maximum, and a row whose temperature is not positive, gets its first maximum (0 if it
// holds no number).
#include "common.h"

#define FS_THREADS 1024
#define FS_WAVES (FS_THREADS / WAVE)
#define FS_BINS 2048
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
  double rate;           // 1 / T
};

__device__ __forceinline__ u64 fs_weight(float v, const FsRow& r) {
  const double x = ((double)v - (double)r.top) * r.rate;
  return x < -31.25 ? 0ull : (u64)rint(exp(x) * FS_UNIT);
}
// Falls with the logit, so a bin is a run of the order; `top` is in bin 0.
__device__ __forceinline__ int fs_bin(float v, const FsRow& r) {
  return min(FS_BINS - 1, (int)((r.top - v) * r.per_bin));
}

struct FsShared {
  u64 mass[FS_BINS];
  uint32_t count[FS_BINS];
  u64 wave_mass[FS_WAVES];
  uint32_t wave_count[FS_WAVES];
  u64 found_mass;
  uint32_t found_count;
  int found;
  uint32_t key_low, key_high;
  float wave_low[FS_WAVES], wave_high[FS_WAVES];
  u64 below;
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

// Where an order of 2 * FS_THREADS slots reaches a number.  The slots' counts and masses are in `s.count` and `s.mass` ([0, n_slots),
// slot `n_slots - 1 - i` first if `backwards`); `need`: the running count (`counting`) or mass to reach.  Returns the slot, and what lies
// before it in `count` and `mass`; -1 if the whole order does not reach it (`count` and `mass` are its sums then).
__device__ int fs_reach(FsShared& s, int n_slots, bool backwards, bool counting, u64 need, uint32_t& count, u64& mass) {
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  u64 m[2];
  uint32_t c[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int place = 2 * threadIdx.x + j;
    const int slot = backwards ? n_slots - 1 - place : place;
    m[j] = place < n_slots ? s.mass[slot] : 0;
    c[j] = place < n_slots ? s.count[slot] : 0;
  }
  u64 run_m = m[0] + m[1];
  u64 run_c = c[0] + c[1];
  for (int off = 1; off < WAVE; off <<= 1) {
    run_m += fs_up(run_m, off, lane);
    run_c += fs_up(run_c, off, lane);
  }
  __syncthreads();
  if (threadIdx.x == 0) s.found = -1;
  if (lane == WAVE - 1) { s.wave_mass[wave] = run_m; s.wave_count[wave] = (uint32_t)run_c; }
  __syncthreads();
  u64 before_m = 0, all_m = 0;
  uint32_t before_c = 0, all_c = 0;
  for (int w = 0; w < FS_WAVES; ++w) {
    if (w < wave) { before_m += s.wave_mass[w]; before_c += s.wave_count[w]; }
    all_m += s.wave_mass[w];
    all_c += s.wave_count[w];
  }
  u64 at_m = before_m + run_m - m[0] - m[1];
  uint32_t at_c = before_c + (uint32_t)run_c - c[0] - c[1];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const u64 before = counting ? (u64)at_c : at_m;
    const u64 here = counting ? (u64)c[j] : m[j];
    if (before < need && before + here >= need) {          // one slot of one thread
      s.found = 2 * threadIdx.x + j;
      s.found_mass = at_m;
      s.found_count = at_c;
    }
    at_m += m[j];
    at_c += c[j];
  }
  __syncthreads();
  const int place = s.found;
  count = place >= 0 ? s.found_count : all_c;
  mass = place >= 0 ? s.found_mass : all_m;
  __syncthreads();
  return place < 0 ? -1 : backwards ? n_slots - 1 - place : place;
}

// The token at which the order reaches a number: its key, and what lies before the tokens of that key.
struct FsCrossing {
  uint32_t key;
  uint32_t before_count;
  u64 before_mass;
  u64 each;              // what a token of the key weighs
};

// Inside one bin of the order: the keys of its members are narrowed, some thousand ranges a round, until one key is left.
// `members(use)` calls use(value) for every member, spread over the workgroup.  `before_*`: what lies before the bin.
template <typename Members>
__device__ FsCrossing fs_inside(FsShared& s, const FsRow& r, bool counting, u64 need, uint32_t before_count, u64 before_mass, Members members) {
  uint32_t low = 0xffffffffu, high = 0;
  members([&](float v) {
    const uint32_t key = fs_key(v);
    low = min(low, key);
    high = max(high, key);
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
    while (((high - low) >> shift) >= FS_BINS) ++shift;
    __syncthreads();
    for (int i = threadIdx.x; i < FS_BINS; i += FS_THREADS) { s.mass[i] = 0; s.count[i] = 0; }
    __syncthreads();
    members([&](float v) {
      const uint32_t key = fs_key(v);
      if (key >= low && key <= high) {
        atomicAdd(&s.count[(key - low) >> shift], 1u);
        atomicAdd(&s.mass[(key - low) >> shift], fs_weight(v, r));
      }
    });
    __syncthreads();
    uint32_t inner_count;
    u64 inner_mass;
    const u64 past = counting ? (u64)before_count : before_mass;
    const int slot = fs_reach(s, FS_BINS, true, counting, need - past, inner_count, inner_mass);
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

// One workgroup a row.
template <typename T>
__global__ void __launch_bounds__(FS_THREADS)
sample_filtered_rows(const T* __restrict__ logits, int64_t stride, const float* __restrict__ temperature, const int* __restrict__ top_k,
                     const float* __restrict__ top_p, const float* __restrict__ min_p, const float* __restrict__ uniform,
                     int* __restrict__ out, int vocab) {
  __shared__ FsShared s;
  const T* row = logits + (size_t)blockIdx.x * stride;
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  const float t = temperature[blockIdx.x];
  // The largest logit and the smallest above -inf.
  float high = -INFINITY, low = INFINITY;
  fs_numbers(row, vocab, [&](float v, int) {
    high = fmaxf(high, v);
    if (v > -INFINITY) low = fminf(low, v);
  });
  for (int off = WAVE / 2; off > 0; off >>= 1) {
    high = fmaxf(high, __shfl_xor(high, off, WAVE));
    low = fminf(low, __shfl_xor(low, off, WAVE));
  }
  if (lane == 0) { s.wave_high[wave] = high; s.wave_low[wave] = low; }
  __syncthreads();
  for (int w = 0; w < FS_WAVES; ++w) { high = fmaxf(high, s.wave_high[w]); low = fminf(low, s.wave_low[w]); }
  uint32_t key = 0;
  u64 rank = 1;                                            // the draw is the rank-th token of its key, by index
  if (!(t > 0.f) || !(high > -INFINITY) || !(high < INFINITY)) {
    if (!(high > -INFINITY)) {                             // nothing above -inf
      if (threadIdx.x == 0) out[blockIdx.x] = 0;
      return;
    }
    key = fs_key(high);
  } else {
    FsRow r;
    r.top = high;
    r.rate = 1.0 / (double)t;
    r.reach = FS_REACH * t;
    const float span = fminf(high - low, r.reach);
    r.per_bin = span > 0.f ? fminf((float)FS_BINS / span, 3.0e38f) : 0.f;
    const double floor_p = (double)min_p[blockIdx.x];
    for (int i = threadIdx.x; i < FS_BINS; i += FS_THREADS) { s.mass[i] = 0; s.count[i] = 0; }
    __syncthreads();
    u64 over = 0;                                          // weight of the tokens that min-p keeps
    fs_numbers(row, vocab, [&](float v, int) {
      if (r.top - v <= r.reach) {
        const u64 w = fs_weight(v, r);
        const int bin = fs_bin(v, r);
        atomicAdd(&s.count[bin], 1u);
        atomicAdd(&s.mass[bin], w);
        if (!(exp(((double)v - (double)r.top) * r.rate) < floor_p) || v == r.top) over += w;
      }
    });
    over = fs_sum(over, s);
    // (The bins are used again inside one of them: they are kept in registers meanwhile.)
    u64 kept_mass[2];
    uint32_t kept_count[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) { kept_mass[j] = s.mass[threadIdx.x + j * FS_THREADS]; kept_count[j] = s.count[threadIdx.x + j * FS_THREADS]; }
    auto crossing = [&](bool counting, u64 need, FsCrossing& x) -> bool {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 2; ++j) { s.mass[threadIdx.x + j * FS_THREADS] = kept_mass[j]; s.count[threadIdx.x + j * FS_THREADS] = kept_count[j]; }
      __syncthreads();
      const int bin = fs_reach(s, FS_BINS, false, counting, need, x.before_count, x.before_mass);
      if (bin < 0) return false;
      x = fs_inside(s, r, counting, need, x.before_count, x.before_mass, [&](auto use) {
        fs_numbers(row, vocab, [&](float v, int) { if (r.top - v <= r.reach && fs_bin(v, r) == bin) use(v); });
      });
      return true;
    };
    FsCrossing x;
    // What top-k keeps weighs ...
    u64 kept;
    const int k = top_k[blockIdx.x];
    if (k > 0 && crossing(true, (u64)k, x)) kept = x.before_mass + ((u64)k - x.before_count) * x.each;
    else {
      u64 all = kept_mass[0] + kept_mass[1];
      kept = fs_sum(all, s);
    }
    // ... of that top-p keeps the shortest prefix that reaches its share ...
    const float p = top_p[blockIdx.x];
    if (p < 1.f) {
      const double share = ceil((double)fmaxf(p, 0.f) * (double)kept);
      const u64 need = share < 1.0 ? 1 : (u64)share;
      if (crossing(false, need, x) && x.each > 0) {
        const u64 tokens = (need - x.before_mass + x.each - 1) / x.each;
        kept = min(kept, x.before_mass + tokens * x.each);
      }
    }
    // ... and min-p what it keeps of all.
    kept = min(kept, over);
    const double target = (double)uniform[blockIdx.x] * (double)kept;
    u64 need = target >= 0.0 ? (target < (double)kept ? (u64)floor(target) + 1 : kept) : 1;
    need = min(need, kept);
    key = fs_key(high);
    if (crossing(false, need, x) && x.each > 0) {
      key = x.key;
      rank = (need - x.before_mass + x.each - 1) / x.each;
    }
  }
  // The rank-th token of the key: which run of indices has it, then which of the run.
  const int per = (vocab + FS_BINS - 1) / FS_BINS;
  __syncthreads();
  for (int i = threadIdx.x; i < FS_BINS; i += FS_THREADS) { s.mass[i] = 0; s.count[i] = 0; }
  __syncthreads();
  fs_numbers(row, vocab, [&](float v, int at) {
    if (fs_key(v) == key) atomicAdd(&s.count[at / per], 1u);
  });
  __syncthreads();
  uint32_t before;
  u64 unused;
  const int run = fs_reach(s, FS_BINS, false, true, rank, before, unused);
  if (threadIdx.x == 0) {
    int pick = 0;
    u64 left = rank - before;
    for (int i = run < 0 ? vocab : run * per; i < min(vocab, (run + 1) * per); ++i) {
      const float v = ld(row + i);
      if (v == v && fs_key(v) == key && --left == 0) { pick = i; break; }
    }
    out[blockIdx.x] = pick;
  }
}

#define FS_MAX_VOCAB (1 << 19)

// logits [n_rows, vocab] (float or bfloat16), rows `stride` elements apart; the others one number a row.
extern "C" int ta_sample_filtered(const void* logits, int64_t stride, const void* temperature, const void* top_k, const void* top_p,
                                  const void* min_p, const void* uniform, void* out, int n_rows, int vocab, int dtype,
                                  hipStream_t stream) {
  if (n_rows <= 0) return 0;
  if (vocab < 1 || vocab > FS_MAX_VOCAB || stride < 0) return -1;
  if (!logits || !temperature || !top_k || !top_p || !min_p || !uniform || !out) return -1;
  if (dtype == DT_F32)
    sample_filtered_rows<float><<<n_rows, FS_THREADS, 0, stream>>>((const float*)logits, stride, (const float*)temperature,
                                                                   (const int*)top_k, (const float*)top_p, (const float*)min_p,
                                                                   (const float*)uniform, (int*)out, vocab);
  else
    sample_filtered_rows<bf16_t><<<n_rows, FS_THREADS, 0, stream>>>((const bf16_t*)logits, stride, (const float*)temperature,
                                                                    (const int*)top_k, (const float*)top_p, (const float*)min_p,
                                                                    (const float*)uniform, (int*)out, vocab);
  return LAUNCH_STATUS();
}
