// Attention of a batch of single query tokens whose requests share leading pages of the cache.
//
// A softmax over a set of keys falls apart over disjoint runs of them: a run leaves, for every query, the largest score m, the sum
// l of exp(score - m) and the values weighed with exp(score - m), and runs are joined as
//   o = sum_i exp(m_i - m) o_i / sum_i exp(m_i - m) l_i,   m = max_i m_i.
// So the keys that several requests share are gone through once, for the queries of all of them (a column of the products each, all
// query heads of a kv head side by side), and each request's own keys behind them on their own; a second kernel joins a query's runs.
//
// Both products are computed transposed, S^T = K Q^T and O^T = V^T P^T: a lane then holds one column of scores and outputs alike, and
// rescaling takes nothing from other lanes.  The rows of the first product are taken in the order in which the second wants its
// keys, so the weights go from the one to the other in registers, and what a lane contracts over is contiguous in a page of V^T.
//
// Three kernels share the work, by how many columns go through a run of keys:
//   * few (a request's own keys; all columns where there is little work; up to 48 left of a run's): sixteen columns a workgroup, whose
//     waves share the keys out;
//   * more, in bfloat16 at head sizes 64 and 128: 128 columns a workgroup, 32 a wave, keys and values through LDS;
//   * more, of other types and sizes: 32 columns a workgroup, whose waves share the keys out.
// What bounds them, measured with keys and values of 16 bits in the caches, head size 128, 4 kv heads of 7 query heads:
//   256 requests behind 32,000 keys: 146 us, 9 of them the join; the products are 118 GFLOP, 0.8 PFLOP/s.  The matrix instructions share the
//     SIMD's issue with an exponential a score and its weight's rounding.
//   64 requests behind 4,096 keys, in eight families of 512 more, with 20 to 700 of their own: 25 us, 4.4 GFLOP and 43 MB: four blocks of
//     keys a workgroup, some 7 us around them (a chain of loads to the first block, the partial results), and the join, 5.
//   4 requests behind 512 keys (head size 64): 7 us, two launches of a few dependent loads each.
// In 32 bits, 21 requests behind 1,040 keys of head size 64: 12.5 us.
// Fragments of the 32x32 instructions: row r of a block of 32 keys is key 16 (r / 16) + 8 (r / 4 % 2) + 4 (r / 8 % 2) + r % 4, and lane
// half h then holds keys 16 s + 8 h .. + 7 of step s of the second product.  Of the 16x16 ones: row r of the first product's
// instruction t is key 8 (r / 4) + 4 t + r % 4, and lane group g then holds keys 8 g .. 8 g + 7.
#include "common.h"

typedef __bf16 sp_bf16x8 __attribute__((ext_vector_type(8)));
typedef float sp_floatx4 __attribute__((ext_vector_type(4)));
typedef float sp_floatx16 __attribute__((ext_vector_type(16)));

#define SP_WAVES 4
#define SP_BLOCK 32                    // keys of a step of a wave
#define SP_WIDE_COLUMNS 128
#define SP_WIDE_BLOCK 64               // keys of a step of a workgroup that shares them through LDS
#define LOG2E 1.4426950408889634f

// A run of shared keys and some of the queries that read them, as the host lists them.
struct SharedItem {
  int rows_at;                         // where in `order` the requests of the run start
  int columns;                         // query columns of the run: its requests times the query heads of a kv head
  int first_column;                    // of this item
  int key_begin, key_end;              // positions; key_end - 1 is the last
  int slot;                            // which of a query's partial results this one is
  int table_row;                       // a request whose block table names the run's pages
  int kv_head;
};
struct SharedOwn {                     // a part of a request's own keys (row -1: an item that only fills the list up)
  int row, begin, slot;                // where it begins, and which of a query's partial results it is
  int left;                            // of the request's parts, this one included; the last has all keys that come behind it
};

struct SharedArgs {
  const void *q, *k_pages, *vt_pages;
  float *part_o, *part_ml;             // [rows, n_q, slots, D], [rows, n_q, slots, 2]
  const SharedItem* items;             // those of few columns first, then those of many
  const int* order;                    // the requests, those of a run side by side
  const SharedOwn *own, *own_of_row;   // all parts, and by request the first
  const int* own_keys;                 // keys of a part (one number; beside the lists, so that a captured launch can be given others)
  const int *positions, *block_table;
  const float* sinks;
  int q_stride, table_stride, n_narrow, n_many, n_own, n_rows, n_q, n_kv, page_size, n_pages, slots;
  int page_shift;                      // page_size as a power of two, -1 if it is none
  float scale, softcap;
};

// Which page of a table holds a key, and where in it (for a whole wave; the scalar unit has no division).
__device__ __forceinline__ void sp_page_of(const SharedArgs& a, int key, int& index, int& slot) {
  if (a.page_shift >= 0) {
    index = key >> a.page_shift;
    slot = key & (a.page_size - 1);
  } else {
    index = key / a.page_size;
    slot = key - index * a.page_size;
  }
}

// A cap on a score: cap tanh(x), x = `inner` / (2 log2(e)) times the raw one.  1 - 2 / (1 + e^2x) is off by some roundings of one, that is of the
// cap: for bfloat16 nothing beside the weights' rounding, in 32 bits more than all else (1.4e-6 of a result's norm instead of 6e-7), so there
// tanh itself is called.
template <typename T>
__device__ __forceinline__ float sp_capped(float raw, float inner, float cap) {
  if constexpr (sizeof(T) == 4) return cap * tanhf(raw * (inner * (0.5f / LOG2E)));
  return cap * (1.f - 2.f * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(inner * raw)));
}

// The fragments of one type: how a block of 32 keys, the queries and the weights lie in registers, and the products.
template <typename T, int D> struct Frag;

template <int D>
struct Frag<bf16_t, D> {
  static constexpr int STEPS = D / 16, ROWS = (D + 31) / 32;
  sp_bf16x8 k[STEPS];
  sp_bf16x8 v[ROWS][2];
  struct Query { sp_bf16x8 f[STEPS]; };
  static __device__ __forceinline__ void load_query(Query& q, const bf16_t* row, bool there, int half) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
#pragma unroll
      for (int i = 0; i < 8; ++i) q.f[s][i] = (__bf16)0.f;
      if (there) q.f[s] = *reinterpret_cast<const sp_bf16x8*>(row + 16 * s + 8 * half);
    }
  }
  __device__ __forceinline__ void load_keys(const bf16_t* row, int half) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) k[s] = *reinterpret_cast<const sp_bf16x8*>(row + 16 * s + 8 * half);
  }
  // `first`, `second`: where the sixteen keys of the two steps start in the pages of V^T (coordinate 0).
  __device__ __forceinline__ void load_values(const bf16_t* first, const bf16_t* second, int page_size, int col, int half) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int d = min(32 * r + col, D - 1);
      v[r][0] = *reinterpret_cast<const sp_bf16x8*>(first + (size_t)d * page_size + 8 * half);
      v[r][1] = *reinterpret_cast<const sp_bf16x8*>(second + (size_t)d * page_size + 8 * half);
    }
  }
  // Slots that nobody wrote hold anything, and a weight of zero times that need not be zero: the values of keys from `there` on
  // (counted from the block's first) are set to zero.
  __device__ __forceinline__ void cut_values(int there, int half) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (16 * s + 8 * half + i >= there) v[r][s][i] = (__bf16)0.f;
  }
  __device__ __forceinline__ sp_floatx16 scores(const Query& q) const {
    sp_floatx16 s = {};
#pragma unroll
    for (int i = 0; i < STEPS; ++i) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[i], q.f[i], s, 0, 0, 0);
    return s;
  }
  // The weights meet the values in bfloat16, as in the other kernels of this type: each is off by 2^-8 of itself at most, and their sum
  // is taken of the weights before they are rounded.
  __device__ __forceinline__ void add_values(const sp_floatx16& p, sp_floatx16 (&o)[ROWS]) const {
    sp_bf16x8 w[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i >> 3][i & 7] = (__bf16)p[i];
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int s = 0; s < 2; ++s) o[r] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[r][s], w[s], o[r], 0, 0, 0);
  }
};

// In 32 bits a step of a product takes two coordinates or two keys, one a lane half: half h has coordinates 8 t + 4 h .. + 3 of every
// eight, and keys 16 s + 8 h .. + 7 as above.
template <int D>
struct Frag<float, D> {
  static constexpr int EIGHTS = D / 8, ROWS = (D + 31) / 32;
  sp_floatx4 k[EIGHTS];
  sp_floatx4 v[ROWS][4];
  struct Query { sp_floatx4 f[EIGHTS]; };
  static __device__ __forceinline__ void load_query(Query& q, const float* row, bool there, int half) {
#pragma unroll
    for (int e = 0; e < EIGHTS; ++e) {
      q.f[e] = (sp_floatx4){0.f, 0.f, 0.f, 0.f};
      if (there) q.f[e] = *reinterpret_cast<const sp_floatx4*>(row + 8 * e + 4 * half);
    }
  }
  __device__ __forceinline__ void load_keys(const float* row, int half) {
#pragma unroll
    for (int e = 0; e < EIGHTS; ++e) k[e] = *reinterpret_cast<const sp_floatx4*>(row + 8 * e + 4 * half);
  }
  __device__ __forceinline__ void load_values(const float* first, const float* second, int page_size, int col, int half) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int d = min(32 * r + col, D - 1);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        v[r][j] = *reinterpret_cast<const sp_floatx4*>(first + (size_t)d * page_size + 8 * half + 4 * j);
        v[r][2 + j] = *reinterpret_cast<const sp_floatx4*>(second + (size_t)d * page_size + 8 * half + 4 * j);
      }
    }
  }
  __device__ __forceinline__ void cut_values(int there, int half) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (16 * (i >> 3) + 8 * half + (i & 7) >= there) v[r][i >> 2][i & 3] = 0.f;
  }
  __device__ __forceinline__ sp_floatx16 scores(const Query& q) const {
    // (Sums of half of the coordinates each, as with few columns; a quarter, where the registers of the one wave a SIMD leave room.)
    constexpr int SUMS = D >= 112 && D <= 160 ? 4 : 2;
    sp_floatx16 s[SUMS] = {};
#pragma unroll
    for (int e = 0; e < EIGHTS; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i % SUMS] = __builtin_amdgcn_mfma_f32_32x32x2f32(k[e][i], q.f[e][i], s[i % SUMS], 0, 0, 0);
    if constexpr (SUMS == 4) return (s[0] + s[1]) + (s[2] + s[3]);
    return s[0] + s[1];
  }
  __device__ __forceinline__ void add_values(const sp_floatx16& p, sp_floatx16 (&o)[ROWS]) const {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[r] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[r][i >> 2][i & 3], p[i], o[r], 0, 0, 0);
  }
};

// A step of the softmax: `s` holds 32 scores a column (a lane half's sixteen each), of which the first `there` keys count;
// they become weights.  m: the largest score so far, in units of 1 / log2(e) (a weight is then one instruction of the exponent's),
// l: this lane's sum of weights, o: the weighed values, all brought to the new maximum where it has grown for any of the wave's columns.
//   The maximum is a reference alone: a weight may be up to 2^SP_SLACK as long as no rescaling has been due (rescaling at every new maximum
//   of any of 32 columns came up in nearly every block: 64 of 220 vector instructions of a block of 64 keys at head size 128).
#define SP_SLACK 8.f
template <typename T, int ROWS>
__device__ __forceinline__ void sp_softmax(const SharedArgs& a, sp_floatx16& s, int there, int half, float& m, float& l, sp_floatx16 (&o)[ROWS]) {
  float scale = a.scale * LOG2E;
  if (a.softcap > 0.f) {
    const float inner = 2.f * LOG2E * a.scale / a.softcap;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = sp_capped<T>(s[i], inner, a.softcap);
    scale = LOG2E;
  }
  if (there < SP_BLOCK) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (16 * (i >> 3) + 8 * half + (i & 7) >= there) s[i] = -INFINITY;
  }
  float high = s[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) high = fmaxf(high, s[i]);
  high = wave_max_across<32>(high) * scale;                // (the scale is positive)
  if (__any(high > m + SP_SLACK)) {
    const float m_new = high > m + SP_SLACK ? high : m;       // (each column for itself: what stands beside it changes nothing)
    const float corr = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
    m = m_new;
    l *= corr;
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[r][i] *= corr;
  }
  const float from = m == -INFINITY ? 0.f : m;             // (no key yet: weights of exp(-inf))
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], scale, -from));
    sum += s[i];
  }
  l += sum;
}

// ------------------------------------------------------------------------------------------------
// Many columns: a wave has 32 of the workgroup's SP_WIDE_COLUMNS, and all of them go through the same keys, which the workgroup brings into
// LDS in blocks of 64 ahead of their use.  Loads write LDS in the order of their lanes, so the lanes ask for pieces of sixteen bytes in
// the order in which the reads find them in different banks: a unit of sixteen keys lies key by key, piece p of key k at place p ^ (k, or
// k / 2 where a key is half as long as the banks are wide); its values lie coordinate by coordinate, the two pieces of a coordinate d
// changing places with d / 8.
//
// The work is a pipeline over steps of 32 keys.  In step k the weights of step k - 1 meet their values while the maximum of step k's scores
// is looked for, and the scores of step k + 1 are made while those of step k become weights: the matrix instructions of a step wait
// for no vector instruction of the same step, and the other way round.  (One after the other, a block of 64 keys took a wave alone
// on its SIMD 1.6 us at head size 128; its 32 instructions of 32x32x16 take 0.43.)  So in iteration b, steps 2 b + 1 and 2 b + 2, the keys
// of block b + 1 and the values of block b are read, and the keys of block b + 2 and the values of block b + 1 come in.
template <int D>
struct Wide {
  static constexpr int PIECES = D / 8, KEY = 2 * D, UNIT = 16 * KEY, TILE = 4 * UNIT;      // pieces of a key; bytes of keys (values alike)
  static constexpr int ROUNDS = TILE / 4096, STEPS = D / 16, ROWS = D / 32;   // (as many pieces of keys as of values: 2 ROWS = STEPS)
  static_assert(D == 64 || D == 128, "the order of the pieces is made for keys of 128 and of 256 bytes");
  typedef const char __attribute__((address_space(1)))* from_t;
  typedef char __attribute__((address_space(3)))* lds_t;

  static __device__ __forceinline__ int turn(int key) { return D == 128 ? key & 15 : (key >> 1) & 7; }
  // Which of the block's four units of sixteen keys a wave brings in round j.
  static __device__ __forceinline__ int unit_of(int j, int wave) { return D == 128 ? j : 2 * j + (wave >> 1); }

  // Bytes from a unit's start in its page to what this thread brings, for keys and for values.
  static __device__ __forceinline__ uint32_t key_place(int thread) {
    const int key = thread / PIECES % 16, place = thread % PIECES;
    return key * KEY + 16 * (place ^ turn(key));
  }
  static __device__ __forceinline__ uint32_t value_place(int thread, int page_size) {
    const int d = thread / 2 % D;
    return d * page_size * 2 + 16 * ((thread & 1) ^ ((d >> 3) & 1));
  }
  // Where piece `half` of a key (of the block's first half) lies; its piece 2 i + half is at that place with the bits of 32 i turned over.
  static __device__ __forceinline__ int key_at(int key, int half) { return key * KEY + 16 * (half ^ turn(key & 15)); }
  static __device__ __forceinline__ sp_bf16x8 key_piece(const char* keys, int part, int at, int i) {
    return *reinterpret_cast<const sp_bf16x8*>(keys + SP_BLOCK * KEY * part + (at ^ (32 * i)));
  }
  static __device__ __forceinline__ sp_bf16x8 value_piece(const char* values, int unit, int d, int half) {
    return *reinterpret_cast<const sp_bf16x8*>(values + unit * UNIT + d * 32 + 16 * (half ^ ((d >> 3) & 1)));
  }
};

template <int D, bool CAPPED>
__device__ __forceinline__ void sp_wide(const SharedArgs& a, char* keys0, char* keys1, char* values0, char* values1) {
  typedef Wide<D> W;
  typedef Frag<bf16_t, D> F;
  constexpr int ROWS = W::ROWS;
  const int* item = reinterpret_cast<const int*>(a.items + a.n_narrow + blockIdx.x);
  const int rows_at = scalar_int(item), columns = scalar_int(item + 1), first_column = scalar_int(item + 2);
  const int begin = scalar_int(item + 3), end = scalar_int(item + 4), slot = scalar_int(item + 5);
  const int* table = a.block_table + (size_t)scalar_int(item + 6) * a.table_stride;
  const int kvh = scalar_int(item + 7), group = a.n_q / a.n_kv;
  if (columns <= 0) return;                                // an item that only fills the list up
  const int lane = threadIdx.x & 63, wave = wave_index(), col = lane & 31, half = lane >> 5;
  // (At head size 128 worked out anew wherever it is used: kept, such numbers are what no register is left for.  With nine of them in
  // memory 40 requests behind 32,000 keys took 49 us instead of 44; at 64, kept, 256 requests 62 instead of 64.)
  auto thread_now = [&] {
    int of_wave = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    if (D == 128) asm volatile("" : "+v"(of_wave));
    return wave * WAVE + of_wave;
  };
  // (A layer's keys are fewer than 2^31 elements: places in bytes fit 32 bits.)
  const uint32_t page_bytes = (uint32_t)a.page_size * D * 2, all_heads = page_bytes * a.n_kv, of_head = page_bytes * kvh;
  const typename W::from_t k_from = (typename W::from_t)a.k_pages, v_from = (typename W::from_t)a.vt_pages;
  // Where this wave's units of a block lie in the pages (the run's last unit stands in for one behind it, of which nothing counts).
  struct Units { int page[W::ROUNDS], at[W::ROUNDS]; };
  auto look_up = [&](int block) {
    Units u;
#pragma unroll
    for (int j = 0; j < W::ROUNDS; ++j) {
      int index;
      sp_page_of(a, min(begin + SP_WIDE_BLOCK * block + 16 * W::unit_of(j, wave), end - 16), index, u.at[j]);
      u.page[j] = scalar_int(table + index);
    }
    return u;
  };
  auto start = [&](const Units& u, int j) { return (uint32_t)min(max(u.page[j], 0), a.n_pages - 1) * all_heads + of_head; };
  auto fetch_keys = [&](const Units& u, char* to) {
    const uint32_t key_place = W::key_place(thread_now());
#pragma unroll
    for (int j = 0; j < W::ROUNDS; ++j)
      __builtin_amdgcn_global_load_lds(k_from + (start(u, j) + (uint32_t)u.at[j] * W::KEY + key_place),
                                       (typename W::lds_t)(to + j * 4096 + wave * 1024), 16, 0, 0);
  };
  auto fetch_values = [&](const Units& u, char* to) {
    const uint32_t value_place = W::value_place(thread_now(), a.page_size);
#pragma unroll
    for (int j = 0; j < W::ROUNDS; ++j)
      __builtin_amdgcn_global_load_lds(v_from + (start(u, j) + (uint32_t)u.at[j] * 2 + value_place),
                                       (typename W::lds_t)(to + j * 4096 + wave * 1024), 16, 0, 0);
  };
  const int blocks = (end - begin + SP_WIDE_BLOCK - 1) / SP_WIDE_BLOCK;
  Units before = look_up(0), next = look_up(1);
  // (The queries are asked for ahead of the keys: which request a column belongs to is looked up while the pages are, and a wait for that would
  // wait for keys under way as well.)
  const bool wave_there = first_column + 32 * wave < columns;
  typename F::Query q;
  {
    // (Behind the last column that one stands in: nothing of it is stored.)
    const int column = min(first_column + 32 * wave + col, columns - 1);
    const int row = a.order[rows_at + column / group], head = kvh * group + column % group;
    __builtin_amdgcn_sched_barrier(0);                     // (the pages and the request are asked for by here)
    F::load_query(q, (const bf16_t*)a.q + (size_t)row * a.q_stride + (size_t)head * D, true, half);
  }
  fetch_keys(before, keys0);
  fetch_values(before, values0);
  fetch_keys(next, keys1);
  before = next;                                           // (block b + 1's, whose values come in iteration b; `next`: block b + 2's)
  next = look_up(2);

  sp_floatx16 o[ROWS];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) o[r] = (sp_floatx16){};
  const int keys_at = W::key_at(16 * (col >> 4) + 8 * ((col >> 2) & 1) + 4 * ((col >> 3) & 1) + (col & 3), half);
  const float scale = CAPPED ? LOG2E : a.scale * LOG2E;
  const float inner = CAPPED ? 2.f * LOG2E * a.scale / a.softcap : 0.f;

  // Pieces of the keys, and of the values, of one half (32 keys) of a block: all asked for before the first is used, ahead of other work (left to itself
  // the compiler asks for two, waits, and asks for the next two).
  struct Pieces { sp_bf16x8 p[W::STEPS]; };
  auto read_keys = [&](const char* keys, int part) {
    Pieces f;
    int at = keys_at;
    if (D == 128) asm volatile("" : "+v"(at));             // (the pieces' places anew as well)
#pragma unroll
    for (int i = 0; i < W::STEPS; ++i) f.p[i] = W::key_piece(keys, part, at, i);
    return f;
  };
  auto read_values = [&](const char* values, int part) {
    Pieces f;
#pragma unroll
    for (int i = 0; i < 2 * ROWS; ++i) f.p[i] = W::value_piece(values, 2 * part + (i & 1), 32 * (i >> 1) + col, half);
    return f;
  };
  auto scores = [&](const Pieces& f) {
    sp_floatx16 s = {};
#pragma unroll
    for (int i = 0; i < W::STEPS; ++i) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.p[i], q.f[i], s, 0, 0, 0);
    return s;
  };
  auto add_values = [&](const Pieces& f, const sp_bf16x8 (&w)[2]) {
#pragma unroll
    for (int i = 0; i < 2 * ROWS; ++i) o[i >> 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.p[i], w[i & 1], o[i >> 1], 0, 0, 0);
  };
  // The reference brought up where a weight would pass 2^SP_SLACK (see `sp_softmax`); `here`: keys of the step that count.
  auto settle = [&](sp_floatx16& s, int here) {
    if (CAPPED) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = sp_capped<bf16_t>(s[i], inner, a.softcap);
    }
    if (here < SP_BLOCK) {
      asm volatile("");                                    // (a branch: worked out for every step the cuts are 48 instructions of it)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (16 * (i >> 3) + 8 * half + (i & 7) >= here) s[i] = -INFINITY;
    }
    float high = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) high = fmaxf(high, s[i]);
    high = wave_max_across<32>(high) * scale;
    if (__any(high > m + SP_SLACK)) {
      const float m_new = high > m + SP_SLACK ? high : m;
      const float corr = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      l *= corr;
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[r][i] *= corr;
    }
  };
  auto weigh = [&](const sp_floatx16& s, sp_bf16x8 (&w)[2]) {
    const float from = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float p = __builtin_amdgcn_exp2f(fmaf(s[i], scale, -from));
      l += p;
      w[i >> 3][i & 7] = (__bf16)p;
    }
  };
  sp_floatx16 even, odd;                                   // scores of the steps in turn
  sp_bf16x8 w[2];
  // Iteration b: `keys` of block b + 1, `values` of block b; the two buffers that the iteration before has freed are filled.
  auto iteration = [&](int b, const char* keys, const char* values, char* keys_to, char* values_to) {
    __builtin_amdgcn_s_waitcnt(0x0F70);                    // all that this wave fetched has arrived (vmcnt 0)
    __syncthreads();
    if (b + 2 < blocks) fetch_keys(next, keys_to);
    if (b + 1 < blocks) fetch_values(before, values_to);
    before = next;
    next = look_up(b + 3);
    if (wave_there) {
      const int here = end - begin - SP_WIDE_BLOCK * b;    // keys from block b on
      const Pieces v0 = read_values(values, 0), k0 = read_keys(keys, 0);
      __builtin_amdgcn_sched_barrier(0);
      add_values(v0, w);
      settle(odd, here - SP_BLOCK);
      const Pieces v1 = read_values(values, 1);
      __builtin_amdgcn_sched_barrier(0);
      even = scores(k0);
      weigh(odd, w);
      const Pieces k1 = read_keys(keys, 1);
      __builtin_amdgcn_sched_barrier(0);
      add_values(v1, w);
      settle(even, here - 2 * SP_BLOCK);
      odd = scores(k1);
      weigh(even, w);
    }
  };
  __builtin_amdgcn_s_waitcnt(0x0F70);
  __syncthreads();
  if (wave_there) {
    even = scores(read_keys(keys0, 0));
    odd = scores(read_keys(keys0, 1));
    settle(even, end - begin);
    weigh(even, w);
  }
  for (int b = 0; b < blocks; b += 2) {
    iteration(b, keys1, values0, keys0, values1);
    if (b + 1 >= blocks) break;                            // (the same for the whole workgroup)
    iteration(b + 1, keys0, values1, keys1, values0);
  }
  // A column's results lie 16 bytes a lane: they go through LDS, so that a store takes whole columns side by side.  Piece p of column c lies at
  // place p ^ c.
  l = wave_add_across<32>(l);
  const int column = first_column + 32 * wave + col, here = columns - first_column - 32 * wave;
  int query = 0;
  if (column < columns) query = a.order[rows_at + column / group] * a.n_q + kvh * group + column % group;
  if (half == 0 && column < columns)
    st_through(reinterpret_cast<uint2*>(a.part_ml) + (size_t)query * a.slots + slot, make_uint2(__float_as_uint(m), __float_as_uint(l)));
  __syncthreads();                                         // the last block has been read
  char* mine = wave < 2 ? (wave == 0 ? keys0 : keys1) : (wave == 2 ? values0 : values1);
  constexpr int LANES = D / 2, AT_ONCE = WAVE / LANES;     // of a column; columns a store
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<sp_floatx4*>(mine + col * 4 * D + 16 * ((8 * r + 2 * j + half) ^ (col & (D / 4 - 1)))) =
          (sp_floatx4){o[r][4 * j], o[r][4 * j + 1], o[r][4 * j + 2], o[r][4 * j + 3]};
  wave_exchange();
  const int in_column = lane % LANES;
#pragma unroll 8
  for (int c = lane / LANES; c < 32; c += AT_ONCE) {
    const int to = __shfl(query, c, WAVE);
    const uint2 v = *reinterpret_cast<const uint2*>(mine + c * 4 * D + 16 * ((in_column >> 1) ^ (c & (D / 4 - 1))) + 8 * (in_column & 1));
    if (c < here) st_through(reinterpret_cast<uint2*>(a.part_o + ((size_t)to * a.slots + slot) * D) + in_column, v);
  }
}

// ------------------------------------------------------------------------------------------------
// One workgroup: 32 columns of one kv head and a run of keys, which its waves share out block by block.
template <typename T, int D>
__global__ void __launch_bounds__(SP_WAVES * WAVE)
shared_prefix_kernel(SharedArgs a) {
  typedef Frag<T, D> F;
  constexpr int ROWS = F::ROWS;
  __shared__ float o_s[SP_WAVES / 2][ROWS * 32][33];
  __shared__ float m_s[SP_WAVES][32], l_s[SP_WAVES][32];
  const int lane = threadIdx.x & 63, wave = wave_index();
  const int col = lane & 31, half = lane >> 5;
  const int group = a.n_q / a.n_kv;
  const int* item = reinterpret_cast<const int*>(a.items + a.n_narrow + blockIdx.x);
  const int rows_at = scalar_int(item), columns = scalar_int(item + 1), first_column = scalar_int(item + 2);
  const int begin = scalar_int(item + 3), end = scalar_int(item + 4), slot = scalar_int(item + 5);
  const int kvh = scalar_int(item + 7);
  if (columns <= 0) return;                                // an item that only fills the list up
  // This lane's column: request (row of the batch) and query head.
  const int column = first_column + col;
  const int row = column < columns ? a.order[rows_at + column / group] : -1;
  const int head = kvh * group + column % group;
  typename F::Query q;
  F::load_query(q, (const T*)a.q + (size_t)max(row, 0) * a.q_stride + (size_t)head * D, row >= 0, half);
  const int* table = a.block_table + (size_t)scalar_int(item + 6) * a.table_stride;
  sp_floatx16 o[ROWS];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) o[r] = (sp_floatx16){};
  const size_t page_elems = (size_t)a.page_size * D;
  const T *k_pages = (const T*)a.k_pages, *vt_pages = (const T*)a.vt_pages;
  // Which key of a block this lane's row of the first product is.
  const int my_key = 16 * (col >> 4) + 8 * ((col >> 2) & 1) + 4 * ((col >> 3) & 1) + (col & 3);
  for (int kb = begin + SP_BLOCK * wave; kb < end; kb += SP_BLOCK * SP_WAVES) {
    // Runs of shared keys begin and end with pages, whose sizes are multiples of sixteen: a half of a block lies in one page.  The second
    // half may have no key: the first one's page stands in for it, and nothing that is read there counts.
    const int second = kb + 16 < end ? kb + 16 : kb;
    int index0, index1, slot0, slot1;
    sp_page_of(a, kb, index0, slot0);
    sp_page_of(a, second, index1, slot1);
    const int page0 = min(max(scalar_int(table + index0), 0), a.n_pages - 1);
    const int page1 = min(max(scalar_int(table + index1), 0), a.n_pages - 1);
    const size_t at0 = ((size_t)page0 * a.n_kv + kvh) * page_elems, at1 = ((size_t)page1 * a.n_kv + kvh) * page_elems;
    F f;
    f.load_keys(k_pages + (my_key < 16 ? at0 + (size_t)(slot0 + my_key) * D : at1 + (size_t)(slot1 + my_key - 16) * D), half);
    f.load_values(vt_pages + at0 + slot0, vt_pages + at1 + slot1, a.page_size, col, half);
    const int there = end - kb;                            // keys of the block that count
    if (there < SP_BLOCK) f.cut_values(there, half);
    sp_floatx16 s = f.scores(q);
    sp_softmax<T, ROWS>(a, s, there, half, m, l, o);
    f.add_values(s, o);
  }
  // The waves' results brought together: two halves of the waves, then one wave takes what the other left.
  l = wave_add_across<32>(l);
  if (half == 0) { m_s[wave][col] = m; l_s[wave][col] = l; }
  __syncthreads();
  float all_m = -INFINITY, all_l = 0.f;
  for (int w = 0; w < SP_WAVES; ++w) all_m = fmaxf(all_m, m_s[w][col]);
  for (int w = 0; w < SP_WAVES; ++w) all_l += all_m == -INFINITY ? 0.f : l_s[w][col] * __builtin_amdgcn_exp2f(m_s[w][col] - all_m);
  const float mine = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - all_m);
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[r][i] *= mine;
#pragma unroll
  for (int step = SP_WAVES / 2; step >= 1; step >>= 1) {
    if (wave >= step && wave < 2 * step) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int i = 0; i < 16; ++i) o_s[wave - step][32 * r + 8 * (i >> 2) + 4 * half + (i & 3)][col] = o[r][i];
    }
    __syncthreads();
    if (wave < step) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[r][i] += o_s[wave][32 * r + 8 * (i >> 2) + 4 * half + (i & 3)][col];
    }
    __syncthreads();
  }
  if (wave != 0 || row < 0) return;
  const size_t at = ((size_t)row * a.n_q + head) * a.slots + slot;
  if (half == 0) { a.part_ml[2 * at] = all_m; a.part_ml[2 * at + 1] = all_l; }
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = 32 * r + 8 * j + 4 * half;
      if (D % 32 == 0 || d < D)
        *reinterpret_cast<sp_floatx4*>(a.part_o + at * D + d) = (sp_floatx4){o[r][4 * j], o[r][4 * j + 1], o[r][4 * j + 2], o[r][4 * j + 3]};
    }
}

// ------------------------------------------------------------------------------------------------
// Few columns: sixteen, the waves share out the keys.  The workgroups from `n_narrow` on take the requests' own keys.
template <typename T, int D> struct Frag16;

template <int D>
struct Frag16<bf16_t, D> {
  static constexpr int STEPS = (D + 31) / 32, ROWS = D / 16;
  sp_bf16x8 k[2][STEPS];
  sp_bf16x8 v[ROWS];
  struct Query { sp_bf16x8 f[STEPS]; };
  static __device__ __forceinline__ sp_bf16x8 none() {
    sp_bf16x8 z;
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = (__bf16)0.f;
    return z;
  }
  static __device__ __forceinline__ void load_query(Query& q, const bf16_t* row, bool there, int g) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      q.f[s] = none();
      if (there && (D % 32 == 0 || 32 * s + 8 * g < D)) q.f[s] = *reinterpret_cast<const sp_bf16x8*>(row + 32 * s + 8 * g);
    }
  }
  __device__ __forceinline__ void load_keys(int t, const bf16_t* row, int g) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      if (D % 32) k[t][s] = none();
      if (D % 32 == 0 || 32 * s + 8 * g < D) k[t][s] = *reinterpret_cast<const sp_bf16x8*>(row + 32 * s + 8 * g);
    }
  }
  __device__ __forceinline__ void load_values(const bf16_t* from, int page_size, int col) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) v[r] = *reinterpret_cast<const sp_bf16x8*>(from + (16 * r + col) * page_size);
  }
  __device__ __forceinline__ void cut_values(int there) {  // as above; `there` counted from the lane's first key
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i >= there) v[r][i] = (__bf16)0.f;
  }
  __device__ __forceinline__ sp_floatx4 scores(int t, const Query& q) const {
    sp_floatx4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < STEPS; ++i) s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[t][i], q.f[i], s, 0, 0, 0);
    return s;
  }
  __device__ __forceinline__ void add_values(const float (&p)[8], sp_floatx4 (&o)[ROWS]) const {
    sp_bf16x8 w;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = (__bf16)p[i];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) o[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[r], w, o[r], 0, 0, 0);
  }
};

// In 32 bits a step takes four coordinates or four keys, one a lane group: group g has coordinates 16 e + 4 g .. + 3 of every sixteen.
template <int D>
struct Frag16<float, D> {
  static constexpr int STEPS = D / 16, ROWS = D / 16;
  sp_floatx4 k[2][STEPS];
  sp_floatx4 v[ROWS][2];
  struct Query { sp_floatx4 f[STEPS]; };
  static __device__ __forceinline__ void load_query(Query& q, const float* row, bool there, int g) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      q.f[s] = (sp_floatx4){0.f, 0.f, 0.f, 0.f};
      if (there) q.f[s] = *reinterpret_cast<const sp_floatx4*>(row + 16 * s + 4 * g);
    }
  }
  __device__ __forceinline__ void load_keys(int t, const float* row, int g) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) k[t][s] = *reinterpret_cast<const sp_floatx4*>(row + 16 * s + 4 * g);
  }
  __device__ __forceinline__ void load_values(const float* from, int page_size, int col) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int i = 0; i < 2; ++i) v[r][i] = *reinterpret_cast<const sp_floatx4*>(from + (16 * r + col) * page_size + 4 * i);
  }
  __device__ __forceinline__ void cut_values(int there) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i >= there) v[r][i >> 2][i & 3] = 0.f;
  }
  __device__ __forceinline__ sp_floatx4 scores(int t, const Query& q) const {
    // (Four sums of a quarter of the coordinates each: a sum's roundings grow with its length, and no instruction waits for the one before.)
    sp_floatx4 s[4] = {};
#pragma unroll
    for (int e = 0; e < STEPS; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t][e][i], q.f[e][i], s[i], 0, 0, 0);
    return (s[0] + s[1]) + (s[2] + s[3]);
  }
  __device__ __forceinline__ void add_values(const float (&p)[8], sp_floatx4 (&o)[ROWS]) const {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int i = 0; i < 8; ++i) o[r] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[r][i >> 2][i & 3], p[i], o[r], 0, 0, 0);
  }
};

#define SP_FEW_COLUMNS 16

struct FewSums {                         // what the waves leave for each other, beside their outputs
  float m[SP_WAVES][SP_FEW_COLUMNS], l[SP_WAVES][SP_FEW_COLUMNS];
  int row[SP_FEW_COLUMNS], head[SP_FEW_COLUMNS];
};
template <int D> constexpr int few_outputs() { return SP_FEW_COLUMNS * (D + 4); }      // floats of a wave's outputs, column by column

// `block`: which of the workgroups for few columns; o0 .. o3: LDS for the waves' outputs.
template <typename T, int D>
__device__ __forceinline__ void sp_few(const SharedArgs& a, int block, float* o0, float* o1, float* o2, float* o3, FewSums& sums) {
  typedef Frag16<T, D> F;
  constexpr int ROWS = F::ROWS, COLUMN = D + 4;
  const int lane = threadIdx.x & 63, wave = wave_index(), col = lane & 15, g = lane >> 4;
  const int group = a.n_q / a.n_kv;
  int columns, first_column, begin, end, slot, table_row, kvh, row = -1;
  const bool own = block >= a.n_narrow;
  const int* table;
  // Which pages the two halves of the wave's next block of keys lie in, asked for a block ahead.  The second half may have no key: the first
  // one's page stands in for it, and nothing that is read there counts.  (The first block of a request's own keys is looked up beside its
  // position: an entry of the table past its pages may hold anything, and is not used.)
  struct Pages { int page0, page1, slot0, slot1; };
  auto look_up = [&](int kb, int last) {
    Pages p;
    int index0, index1;
    sp_page_of(a, kb, index0, p.slot0);
    sp_page_of(a, kb + 16 <= last ? kb + 16 : kb, index1, p.slot1);
    p.page0 = scalar_int(table + min(index0, a.table_stride - 1));
    p.page1 = scalar_int(table + min(index1, a.table_stride - 1));
    return p;
  };
  Pages next;
  if (!own) {
    const int* item = reinterpret_cast<const int*>(a.items + block);
    const int rows_at = scalar_int(item);
    columns = scalar_int(item + 1); first_column = scalar_int(item + 2);
    begin = scalar_int(item + 3); end = scalar_int(item + 4); slot = scalar_int(item + 5);
    table_row = scalar_int(item + 6); kvh = scalar_int(item + 7);
    if (columns <= 0) return;                              // an item that only fills the list up
    table = a.block_table + (size_t)table_row * a.table_stride;
    next = look_up(begin + SP_BLOCK * wave, end - 1);
    if (first_column + col < columns) row = a.order[rows_at + (first_column + col) / group];
  } else {
    const int tiles = (group + SP_FEW_COLUMNS - 1) / SP_FEW_COLUMNS;
    int at = block - a.n_narrow;
    kvh = at % a.n_kv;
    at /= a.n_kv;
    const int tile = at % tiles;
    const int* of = reinterpret_cast<const int*>(a.own + at / tiles);
    table_row = scalar_int(of);
    begin = scalar_int(of + 1);
    slot = scalar_int(of + 2);
    const int left = scalar_int(of + 3), own_keys = scalar_int(a.own_keys);
    if (table_row < 0) return;
    columns = group;
    first_column = tile * SP_FEW_COLUMNS;
    table = a.block_table + (size_t)table_row * a.table_stride;
    end = min(scalar_int(a.positions + table_row), a.table_stride * a.page_size - 1) + 1;
    next = look_up(begin + SP_BLOCK * wave, begin + SP_BLOCK * wave + 16);
    if (begin >= end) return;                              // a short request: its last parts are empty, and not asked for
    if (left > 1) end = min(end, begin + own_keys);
    if (begin + SP_BLOCK * wave + 16 >= end) { next.page1 = next.page0; next.slot1 = next.slot0; }
    if (first_column + col < columns) row = table_row;
  }
  const int column = first_column + col, head = kvh * group + column % group;
  typename F::Query q;
  F::load_query(q, (const T*)a.q + (size_t)max(row, 0) * a.q_stride + (size_t)head * D, row >= 0, g);
  sp_floatx4 o[ROWS];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) o[r] = (sp_floatx4){0.f, 0.f, 0.f, 0.f};
  const uint32_t page_elems = (uint32_t)a.page_size * D;
  const T *k_pages = (const T*)a.k_pages, *vt_pages = (const T*)a.vt_pages;
  const float scale = a.softcap > 0.f ? LOG2E : a.scale * LOG2E;
  const float inner = a.softcap > 0.f ? 2.f * LOG2E * a.scale / a.softcap : 0.f;
  constexpr int STRIDE = SP_BLOCK * SP_WAVES;
  auto load = [&](F& f, int kb) {
    const uint32_t page0 = min(max(next.page0, 0), a.n_pages - 1), page1 = min(max(next.page1, 0), a.n_pages - 1);
    const uint32_t at = ((col >> 3 ? page1 : page0) * a.n_kv + kvh) * page_elems +
                        ((col >> 3 ? next.slot1 : next.slot0) + 8 * ((col >> 2) & 1) + (col & 3)) * D;
#pragma unroll
    for (int t = 0; t < 2; ++t) f.load_keys(t, k_pages + at + 4 * t * D, g);
    f.load_values(vt_pages + ((g >> 1 ? page1 : page0) * a.n_kv + kvh) * page_elems + (g >> 1 ? next.slot1 : next.slot0) + 8 * (g & 1),
                  a.page_size, col);
    if (kb + STRIDE < end) next = look_up(kb + STRIDE, end - 1);
  };
  auto attend = [&](F& f, int kb) {
    const int here = end - kb;                             // keys of the block that count
    if (here < SP_BLOCK) f.cut_values(here - 8 * g);
    float s[8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const sp_floatx4 st = f.scores(t, q);
#pragma unroll
      for (int r = 0; r < 4; ++r) s[4 * t + r] = st[r];
    }
    if (a.softcap > 0.f) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = sp_capped<T>(s[i], inner, a.softcap);
    }
    if (here < SP_BLOCK) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (8 * g + i >= here) s[i] = -INFINITY;
    }
    float high = s[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) high = fmaxf(high, s[i]);
    high = wave_max_across<32>(wave_max_across<16>(high)) * scale;
    if (__any(high > m + SP_SLACK)) {
      const float m_new = high > m + SP_SLACK ? high : m;
      const float corr = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      l *= corr;
#pragma unroll
      for (int r = 0; r < ROWS; ++r) o[r] *= corr;
    }
    const float from = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], scale, -from));
      l += s[i];
    }
    f.add_values(s, o);
  };
  // Two blocks in turn, where their registers leave two waves a SIMD: the next one's keys and values are on their way meanwhile.
  constexpr bool AHEAD = sizeof(T) == 2 ? D <= 128 : D <= 64;
  int kb = begin + SP_BLOCK * wave;
  if constexpr (AHEAD) {
    if (kb < end) {
      F one, two;
      load(one, kb);
      while (true) {
        if (kb + STRIDE < end) load(two, kb + STRIDE);
        attend(one, kb);
        kb += STRIDE;
        if (kb >= end) break;
        if (kb + STRIDE < end) load(one, kb + STRIDE);
        attend(two, kb);
        kb += STRIDE;
        if (kb >= end) break;
      }
    }
  } else {
    for (; kb < end; kb += STRIDE) {
      F one;
      load(one, kb);
      attend(one, kb);
    }
  }
  // The waves' sums brought together through LDS, column by column.
  l = wave_add_across<32>(wave_add_across<16>(l));
  float* mine = wave < 2 ? (wave == 0 ? o0 : o1) : (wave == 2 ? o2 : o3);
#pragma unroll
  for (int r = 0; r < ROWS; ++r) *reinterpret_cast<sp_floatx4*>(mine + col * COLUMN + 16 * r + 4 * g) = o[r];
  if (g == 0) { sums.m[wave][col] = m; sums.l[wave][col] = l; }
  if (wave == 0 && g == 0) { sums.row[col] = row; sums.head[col] = head; }
  __syncthreads();
  const int heads_here = min(SP_FEW_COLUMNS, columns - first_column);
  for (int c = wave; c < heads_here; c += SP_WAVES) {
    float top = sums.m[0][c];
#pragma unroll
    for (int w = 1; w < SP_WAVES; ++w) top = fmaxf(top, sums.m[w][c]);
    float factor[SP_WAVES], below = 0.f;
#pragma unroll
    for (int w = 0; w < SP_WAVES; ++w) {
      factor[w] = sums.m[w][c] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sums.m[w][c] - top);
      below += sums.l[w][c] * factor[w];
    }
    const size_t to = ((size_t)sums.row[c] * a.n_q + sums.head[c]) * a.slots + slot;
    if (lane == 0) st_through(reinterpret_cast<uint2*>(a.part_ml + 2 * to), make_uint2(__float_as_uint(top), __float_as_uint(below)));
#pragma unroll
    for (int j = 0; j < (D + WAVE - 1) / WAVE; ++j) {
      const int d = lane + j * WAVE;
      if (d < D) {
        float sum = 0.f;
        sum += o0[c * COLUMN + d] * factor[0];
        sum += o1[c * COLUMN + d] * factor[1];
        sum += o2[c * COLUMN + d] * factor[2];
        sum += o3[c * COLUMN + d] * factor[3];
        st_through(a.part_o + to * D + d, sum);
      }
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(SP_WAVES * WAVE)
shared_prefix_few(SharedArgs a) {
  __shared__ float o_s[SP_WAVES][few_outputs<D>()];
  __shared__ FewSums sums;
  static_assert(SP_WAVES == 4, "outputs of four waves");
  sp_few<T, D>(a, blockIdx.x, o_s[0], o_s[1], o_s[2], o_s[3], sums);
}

// Both in one launch: the workgroups for many columns first.  (Neither leaves more than two waves a SIMD room at head size 128, and each
// alone leaves much of the device idle at its end.)
template <int D, bool CAPPED>
__global__ void __launch_bounds__(SP_WAVES * WAVE, 2)      // (two waves a SIMD: half its registers each)
shared_prefix_both(SharedArgs a) {
  // (The buffers are arrays of their own, each named where it is used: a read of one then waits for no load into another.)
  __shared__ __attribute__((aligned(1024))) char keys0[Wide<D>::TILE];
  __shared__ __attribute__((aligned(1024))) char keys1[Wide<D>::TILE];
  __shared__ __attribute__((aligned(1024))) char values0[Wide<D>::TILE];
  __shared__ __attribute__((aligned(1024))) char values1[Wide<D>::TILE];
  __shared__ FewSums sums;
  static_assert(few_outputs<D>() * 4 <= Wide<D>::TILE, "a wave's outputs in a buffer");
  if ((int)blockIdx.x < a.n_many) {
    sp_wide<D, CAPPED>(a, keys0, keys1, values0, values1);
  } else {
    sp_few<bf16_t, D>(a, blockIdx.x - a.n_many, (float*)keys0, (float*)keys1, (float*)values0, (float*)values1, sums);
  }
}

// A wave joins the runs of one query: those of shared keys, then its own.  A lane has one run's maximum and sum (of sixty-four at a
// time), and the runs' values are asked for eight at a time.
template <typename T, int D>
__global__ void __launch_bounds__(SP_WAVES * WAVE)
shared_prefix_join(SharedArgs a, T* __restrict__ out) {
  const int lane = threadIdx.x & 63, wave = wave_index();
  const int at = blockIdx.x * SP_WAVES + wave;
  if (at >= a.n_rows * a.n_q) return;
  const int row = at / a.n_q, head = at - row * a.n_q;
  const int* mine = reinterpret_cast<const int*>(a.own_of_row + row);
  const int begin = scalar_int(mine + 1), shared = scalar_int(mine + 2), own_parts = scalar_int(mine + 3), own_keys = scalar_int(a.own_keys);
  const int own = min(scalar_int(a.positions + row), a.table_stride * a.page_size - 1) + 1 - begin;
  const int parts = shared + (own > 0 ? min((own - 1) / own_keys + 1, own_parts) : 0);                    // (a.slots at most)
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + (size_t)at * a.slots;
  const float* part = a.part_o + (size_t)at * a.slots * D;
  const float sink = a.sinks ? a.sinks[head] * LOG2E : -INFINITY;
  float m = sink;
  for (int p = lane; p < parts; p += WAVE) m = fmaxf(m, ml[p].x);
  m = wave_max(m);
  float below = 0.f;
  constexpr int PER = (D + WAVE - 1) / WAVE, DEEP = 8;
  float o[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) o[j] = 0.f;
  for (int first = 0; first < parts; first += WAVE) {
    const float2 of = first + lane < parts ? ml[first + lane] : make_float2(-INFINITY, 0.f);
    const float weight = of.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(of.x - m);
    below += weight * of.y;
    const int here = min(WAVE, parts - first);
    for (int p = 0; p < here; p += DEEP) {
      float got[DEEP][PER];
#pragma unroll
      for (int i = 0; i < DEEP; ++i)
#pragma unroll
        for (int j = 0; j < PER; ++j)
          got[i][j] = part[(size_t)(first + min(p + i, here - 1)) * D + min(lane + j * WAVE, D - 1)];
#pragma unroll
      for (int i = 0; i < DEEP; ++i) {
        const float w = p + i < here ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(weight), min(p + i, WAVE - 1))) : 0.f;
        if (p + i < here) {
#pragma unroll
          for (int j = 0; j < PER; ++j) o[j] += w * got[i][j];
        }
      }
    }
  }
  below = wave_sum(below);
  if (sink > -INFINITY) below += __builtin_amdgcn_exp2f(sink - m);
  // (A query that sees no key gets zeros.)
  const float share = below > 0.f ? 1.f / below : 0.f;
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (lane + j * WAVE < D) st(out + (size_t)at * D + lane + j * WAVE, o[j] * share);
}

// Whether many columns of this type and head size go through LDS, 128 a workgroup (else 32 a workgroup).
template <typename T, int D>
constexpr bool sp_is_wide() { return sizeof(T) == 2 && (D == 64 || D == 128); }

template <typename T, int D>
static int launch_shared(const SharedArgs& a, void* out, hipStream_t stream) {
  const int group = a.n_q / a.n_kv, tiles = (group + SP_FEW_COLUMNS - 1) / SP_FEW_COLUMNS;
  const unsigned few = (unsigned)a.n_narrow + (unsigned)a.n_own * tiles * a.n_kv;
  int status = 0;
  if constexpr (sp_is_wide<T, D>()) {
    if (a.n_many == 0) shared_prefix_few<T, D><<<few, SP_WAVES * WAVE, 0, stream>>>(a);
    else if (a.softcap > 0.f) shared_prefix_both<D, true><<<a.n_many + few, SP_WAVES * WAVE, 0, stream>>>(a);
    else shared_prefix_both<D, false><<<a.n_many + few, SP_WAVES * WAVE, 0, stream>>>(a);
    status = LAUNCH_STATUS();
  } else {
    if (a.n_many > 0) {
      shared_prefix_kernel<T, D><<<a.n_many, SP_WAVES * WAVE, 0, stream>>>(a);
      status = LAUNCH_STATUS();
      if (status) return status;
    }
    shared_prefix_few<T, D><<<few, SP_WAVES * WAVE, 0, stream>>>(a);
    status = LAUNCH_STATUS();
  }
  if (status) return status;
  const int queries = a.n_rows * a.n_q;
  shared_prefix_join<T, D><<<(queries + SP_WAVES - 1) / SP_WAVES, SP_WAVES * WAVE, 0, stream>>>(a, (T*)out);
  return LAUNCH_STATUS();
}

// q: the query heads of every row at its start, rows q_stride elements apart; pages as in the other attention kernels; items int32
// [n_narrow + n_many, 8] (`SharedItem`; sixteen columns each, then 128 or 32); order int32 [n_rows]: the rows, those of a run of shared keys
// side by side; own int32 [n_own, 4] (`SharedOwn`): the parts of all rows' own keys; own_of_row int32 [n_rows, 4]: the rows' first parts, whose
// `slot` is how many partial results their shared keys leave; own_keys int32 [1]: keys of a part; positions int32 [n_rows]; block_table int32
// [n_rows, table_stride].  part_o float [n_rows, n_q, slots, head_dim], part_ml float [n_rows, n_q, slots, 2].  -2: a head size without an
// instance.
extern "C" int ta_shared_prefix_attention(const void* q, int q_stride, void* out, const void* k_pages, const void* vt_pages,
                                          const void* items, int n_narrow, int n_many, const void* order, const void* own, int n_own,
                                          const void* own_of_row, const void* own_keys, const void* positions, const void* block_table,
                                          int table_stride, const void* sinks, void* part_o, void* part_ml, int slots, int n_rows, int n_q,
                                          int n_kv, int head_dim, int page_size, int n_pages, float scale, float softcap, int dtype,
                                          hipStream_t stream) {
  if (n_rows <= 0) return 0;
  if (!q || !out || !k_pages || !vt_pages || !order || !own || !own_of_row || !own_keys || !positions || !block_table || !part_o || !part_ml)
    return -1;
  if (n_narrow < 0 || n_many < 0 || (n_narrow + n_many && !items) || n_own < n_rows || n_kv < 1 || n_kv > 65535 || n_q < n_kv || n_q % n_kv ||
      page_size < 16 || page_size % 16 || n_pages < 1 || slots < 1 || table_stride < 1) return -1;
  SharedArgs a = {};
  a.q = q; a.k_pages = k_pages; a.vt_pages = vt_pages; a.part_o = (float*)part_o; a.part_ml = (float*)part_ml;
  a.items = (const SharedItem*)items; a.order = (const int*)order; a.own = (const SharedOwn*)own;
  a.own_of_row = (const SharedOwn*)own_of_row; a.own_keys = (const int*)own_keys; a.positions = (const int*)positions;
  a.block_table = (const int*)block_table; a.sinks = (const float*)sinks; a.q_stride = q_stride; a.table_stride = table_stride;
  a.n_narrow = n_narrow; a.n_many = n_many; a.n_own = n_own; a.n_rows = n_rows; a.n_q = n_q; a.n_kv = n_kv; a.page_size = page_size;
  a.n_pages = n_pages; a.slots = slots;
  a.page_shift = page_size & (page_size - 1) ? -1 : __builtin_ctz(page_size);
  a.scale = scale; a.softcap = softcap;
#define SHARED_CASE(D) \
  case D: return dtype == DT_F32 ? launch_shared<float, D>(a, out, stream) : launch_shared<bf16_t, D>(a, out, stream);
  switch (head_dim) {
    SHARED_CASE(16) SHARED_CASE(32) SHARED_CASE(48) SHARED_CASE(64) SHARED_CASE(80) SHARED_CASE(96) SHARED_CASE(112)
    SHARED_CASE(128) SHARED_CASE(160) SHARED_CASE(192) SHARED_CASE(224) SHARED_CASE(256)
    default: return -2;
  }
}
