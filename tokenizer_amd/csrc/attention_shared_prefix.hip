// Attention of a batch of single query tokens whose requests share leading pages of the cache.
//
// A softmax over a set of keys falls apart over disjoint runs of them: a run leaves, for every query, the largest score m, the sum
// l of exp(score - m) and the values weighed with exp(score - m), and runs are joined as
//   o = sum_i exp(m_i - m) o_i / sum_i exp(m_i - m) l_i,   m = max_i m_i.
// So the keys that several requests share are gone through once, for the queries of all of them (a column of the products each, all
// query heads of a kv head side by side), and each request's own keys behind them on their own; a second kernel joins a query's runs.
//
// Both products are computed transposed, S^T = K Q^T and O^T = V^T P^T, on the 32x32 matrix instructions: a lane then holds one
// column of scores and outputs alike (column lane % 32), and rescaling takes nothing from other lanes.  The rows of the
// first product are taken in the order in which the second wants its keys, so the weights go from the one to the other in
// registers: row r of a block of 32 keys is key 16 (r / 16) + 8 (r / 4 % 2) + 4 (r / 8 % 2) + r % 4, and lane half h then holds
// keys 16 s + 8 h .. + 7 of step s of the second product, which are sixteen contiguous bytes of a page of V^T.
#include "common.h"

typedef __bf16 sp_bf16x8 __attribute__((ext_vector_type(8)));
typedef float sp_floatx4 __attribute__((ext_vector_type(4)));
typedef float sp_floatx16 __attribute__((ext_vector_type(16)));

#define SP_WAVES 4
#define SP_BLOCK 32                    // keys of a step of a wave

// A run of shared keys and some of the queries that read them, as the host lists them.
struct SharedItem {
  int rows_at;                         // where in `order` the requests of the run start
  int columns;                         // query columns of the run: its requests times the query heads of a kv head
  int first_column;                    // of this item
  int key_begin, key_end;              // positions; key_end - 1 is the last
  int slot;                            // which of a query's partial results this one is
  int unused0, unused1;
};

struct SharedArgs {
  const void *q, *k_pages, *vt_pages;
  float *part_o, *part_ml;             // [rows, n_q, slots, D], [rows, n_q, slots, 2]
  const SharedItem* items;
  const int *order, *own_begin, *shared_parts, *positions, *block_table;
  const float* sinks;
  int q_stride, table_stride, n_items, n_rows, n_q, n_kv, page_size, n_pages, slots, own_splits, own_keys;
  float scale, softcap;
};

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
    sp_floatx16 s = {};
#pragma unroll
    for (int e = 0; e < EIGHTS; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) s = __builtin_amdgcn_mfma_f32_32x32x2f32(k[e][i], q.f[e][i], s, 0, 0, 0);
    return s;
  }
  __device__ __forceinline__ void add_values(const sp_floatx16& p, sp_floatx16 (&o)[ROWS]) const {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[r] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[r][i >> 2][i & 3], p[i], o[r], 0, 0, 0);
  }
};

// One workgroup: some columns (COLS blocks of 32) of one kv head and a run of keys, which its waves share out block by block.  The
// workgroups from `n_items` on take the requests' own keys.
template <typename T, int D, int COLS>
__global__ void __launch_bounds__(SP_WAVES * WAVE)
shared_prefix_kernel(SharedArgs a) {
  typedef Frag<T, D> F;
  constexpr int ROWS = F::ROWS;
  __shared__ float o_s[SP_WAVES / 2][COLS][ROWS * 32][33];
  __shared__ float m_s[SP_WAVES][COLS * 32], l_s[SP_WAVES][COLS * 32];
  const int lane = threadIdx.x & 63, wave = wave_index();
  const int col = lane & 31, half = lane >> 5;
  const int kvh = blockIdx.y, group = a.n_q / a.n_kv;
  int rows_at, columns, first_column, begin, end, slot;
  if ((int)blockIdx.x < a.n_items) {
    const int* item = reinterpret_cast<const int*>(a.items + blockIdx.x);
    rows_at = scalar_int(item); columns = scalar_int(item + 1); first_column = scalar_int(item + 2);
    begin = scalar_int(item + 3); end = scalar_int(item + 4); slot = scalar_int(item + 5);
    if (columns <= 0) return;                              // an item that only fills the list up
  } else {
    const int tiles = (group + COLS * 32 - 1) / (COLS * 32);
    const int at = blockIdx.x - a.n_items, split = at % a.own_splits, tile = at / a.own_splits % tiles;
    rows_at = at / a.own_splits / tiles;
    const int row = scalar_int(a.order + rows_at);
    columns = group;
    first_column = tile * COLS * 32;
    begin = scalar_int(a.own_begin + row) + split * a.own_keys;
    end = min(scalar_int(a.positions + row), a.table_stride * a.page_size - 1) + 1;
    if (begin >= end) return;                              // a short request: its last parts are empty, and not asked for
    end = min(end, begin + a.own_keys);
    slot = scalar_int(a.shared_parts + row) + split;
  }
  // This lane's columns: request (row of the batch) and query head of each.
  int row_of[COLS], head_of[COLS];
  typename F::Query q[COLS];
#pragma unroll
  for (int c = 0; c < COLS; ++c) {
    const int column = first_column + 32 * c + col;
    const bool there = column < columns;
    row_of[c] = there ? a.order[rows_at + column / group] : -1;
    head_of[c] = kvh * group + column % group;
    F::load_query(q[c], (const T*)a.q + (size_t)max(row_of[c], 0) * a.q_stride + (size_t)head_of[c] * D, there, half);
  }
  const int* table = a.block_table + (size_t)scalar_int(a.order + rows_at) * a.table_stride;
  sp_floatx16 o[COLS][ROWS];
  float m[COLS], l[COLS];
#pragma unroll
  for (int c = 0; c < COLS; ++c) {
    m[c] = -INFINITY;
    l[c] = 0.f;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) o[c][r] = (sp_floatx16){};
  }
  const size_t page_elems = (size_t)a.page_size * D;
  const T *k_pages = (const T*)a.k_pages, *vt_pages = (const T*)a.vt_pages;
  // Which key of a block this lane's row of the first product is.
  const int my_key = 16 * (col >> 4) + 8 * ((col >> 2) & 1) + 4 * ((col >> 3) & 1) + (col & 3);
  for (int kb = begin + SP_BLOCK * wave; kb < end; kb += SP_BLOCK * SP_WAVES) {
    // Runs of shared keys begin and end with pages, whose sizes are multiples of sixteen: a half of a block lies in one page.  The second
    // half may have no key: the first one's page stands in for it, and nothing that is read there counts.
    const int second = kb + 16 < end ? kb + 16 : kb;
    const int page0 = min(max(scalar_int(table + kb / a.page_size), 0), a.n_pages - 1);
    const int page1 = min(max(scalar_int(table + second / a.page_size), 0), a.n_pages - 1);
    const size_t at0 = ((size_t)page0 * a.n_kv + kvh) * page_elems, at1 = ((size_t)page1 * a.n_kv + kvh) * page_elems;
    const int slot0 = kb % a.page_size, slot1 = second % a.page_size;
    F f;
    f.load_keys(k_pages + (my_key < 16 ? at0 + (size_t)(slot0 + my_key) * D : at1 + (size_t)(slot1 + my_key - 16) * D), half);
    f.load_values(vt_pages + at0 + slot0, vt_pages + at1 + slot1, a.page_size, col, half);
    const int there = end - kb;                            // keys of the block that count
    if (there < SP_BLOCK) f.cut_values(there, half);
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
      sp_floatx16 s = f.scores(q[c]);
      float high = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] *= a.scale;
        if (a.softcap > 0.f) s[i] = a.softcap * (1.f - 2.f / (1.f + __expf(2.f * s[i] / a.softcap)));
        if (there < SP_BLOCK && 16 * (i >> 3) + 8 * half + (i & 7) >= there) s[i] = -INFINITY;
        high = fmaxf(high, s[i]);
      }
      high = wave_max_across<32>(high);
      const float m_new = fmaxf(m[c], high);
      const float corr = m_new == -INFINITY ? 1.f : __expf(m[c] - m_new);
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = m_new == -INFINITY ? 0.f : __expf(s[i] - m_new);
        sum += s[i];
      }
      l[c] = l[c] * corr + sum;
      m[c] = m_new;
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[c][r][i] *= corr;
      f.add_values(s, o[c]);
    }
  }
  // The waves' results brought together: two halves of the waves, then one wave takes what the other left.
#pragma unroll
  for (int c = 0; c < COLS; ++c) {
    l[c] = wave_add_across<32>(l[c]);
    if (half == 0) { m_s[wave][32 * c + col] = m[c]; l_s[wave][32 * c + col] = l[c]; }
  }
  __syncthreads();
  float all_m[COLS], all_l[COLS];
#pragma unroll
  for (int c = 0; c < COLS; ++c) {
    all_m[c] = -INFINITY;
    all_l[c] = 0.f;
    for (int w = 0; w < SP_WAVES; ++w) all_m[c] = fmaxf(all_m[c], m_s[w][32 * c + col]);
    for (int w = 0; w < SP_WAVES; ++w)
      all_l[c] += all_m[c] == -INFINITY ? 0.f : l_s[w][32 * c + col] * __expf(m_s[w][32 * c + col] - all_m[c]);
    const float mine = m[c] == -INFINITY ? 0.f : __expf(m[c] - all_m[c]);
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[c][r][i] *= mine;
  }
#pragma unroll
  for (int step = SP_WAVES / 2; step >= 1; step >>= 1) {
    if (wave >= step && wave < 2 * step) {
#pragma unroll
      for (int c = 0; c < COLS; ++c)
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
          for (int i = 0; i < 16; ++i) o_s[wave - step][c][32 * r + 8 * (i >> 2) + 4 * half + (i & 3)][col] = o[c][r][i];
    }
    __syncthreads();
    if (wave < step) {
#pragma unroll
      for (int c = 0; c < COLS; ++c)
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[c][r][i] += o_s[wave][c][32 * r + 8 * (i >> 2) + 4 * half + (i & 3)][col];
    }
    __syncthreads();
  }
  if (wave != 0) return;
#pragma unroll
  for (int c = 0; c < COLS; ++c) {
    if (row_of[c] < 0) continue;
    const size_t at = ((size_t)row_of[c] * a.n_q + head_of[c]) * a.slots + slot;
    if (half == 0) { a.part_ml[2 * at] = all_m[c]; a.part_ml[2 * at + 1] = all_l[c]; }
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int d = 32 * r + 8 * j + 4 * half;
        if (D % 32 == 0 || d < D)
          *reinterpret_cast<sp_floatx4*>(a.part_o + at * D + d) =
              (sp_floatx4){o[c][r][4 * j], o[c][r][4 * j + 1], o[c][r][4 * j + 2], o[c][r][4 * j + 3]};
      }
  }
}

// A wave joins the runs of one query: `parts` of shared keys, then its own.
template <typename T, int D>
__global__ void __launch_bounds__(SP_WAVES * WAVE)
shared_prefix_join(SharedArgs a, T* __restrict__ out) {
  const int lane = threadIdx.x & 63, wave = wave_index();
  const int at = blockIdx.x * SP_WAVES + wave;
  if (at >= a.n_rows * a.n_q) return;
  const int row = at / a.n_q, head = at % a.n_q;
  const int own = min(scalar_int(a.positions + row), a.table_stride * a.page_size - 1) + 1 - scalar_int(a.own_begin + row);
  const int parts = min(a.slots, scalar_int(a.shared_parts + row) + (own > 0 ? (own + a.own_keys - 1) / a.own_keys : 0));
  const float* ml = a.part_ml + (size_t)at * a.slots * 2;
  const float* part = a.part_o + (size_t)at * a.slots * D;
  float m = a.sinks ? a.sinks[head] : -INFINITY;
  const float sink = m;
  for (int p = 0; p < parts; ++p) m = fmaxf(m, ml[2 * p]);
  float below = a.sinks && m > -INFINITY ? __expf(sink - m) : 0.f;
  constexpr int PER = (D + WAVE - 1) / WAVE;
  float o[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) o[j] = 0.f;
  for (int p = 0; p < parts; ++p) {
    const float w = ml[2 * p] == -INFINITY ? 0.f : __expf(ml[2 * p] - m);
    below += w * ml[2 * p + 1];
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (lane + j * WAVE < D) o[j] += w * part[(size_t)p * D + lane + j * WAVE];
  }
  // (A query that sees no key gets zeros.)
  const float share = below > 0.f ? 1.f / below : 0.f;
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (lane + j * WAVE < D) st(out + (size_t)at * D + lane + j * WAVE, o[j] * share);
}

template <typename T, int D>
static int launch_shared(const SharedArgs& a, void* out, int columns, hipStream_t stream) {
  const int group = a.n_q / a.n_kv, tiles = (group + columns - 1) / columns;
  const dim3 grid((unsigned)a.n_items + (unsigned)a.n_rows * tiles * a.own_splits, a.n_kv);
  if (columns == 32) shared_prefix_kernel<T, D, 1><<<grid, SP_WAVES * WAVE, 0, stream>>>(a);
  else return -2;
  const int status = LAUNCH_STATUS();
  if (status) return status;
  const int queries = a.n_rows * a.n_q;
  shared_prefix_join<T, D><<<(queries + SP_WAVES - 1) / SP_WAVES, SP_WAVES * WAVE, 0, stream>>>(a, (T*)out);
  return LAUNCH_STATUS();
}

// q: the query heads of every row at its start, rows q_stride elements apart; pages as in the other attention kernels; items int32
// [n_items, 8] (`SharedItem`); order int32 [n_rows]: the rows, those of a run of shared keys side by side; own_begin,
// shared_parts int32 [n_rows]: where a request's own keys begin, and how many partial results its shared keys leave; positions
// int32 [n_rows]; block_table int32 [n_rows, table_stride].  part_o float [n_rows, n_q, slots, head_dim], part_ml float
// [n_rows, n_q, slots, 2].  -2: a head size without an instance.
extern "C" int ta_shared_prefix_attention(const void* q, int q_stride, void* out, const void* k_pages, const void* vt_pages,
                                          const void* items, int n_items, const void* order, const void* own_begin,
                                          const void* shared_parts, const void* positions, const void* block_table,
                                          int table_stride, const void* sinks, void* part_o, void* part_ml, int slots,
                                          int own_splits, int own_keys, int columns, int n_rows, int n_q, int n_kv, int head_dim,
                                          int page_size, int n_pages, float scale, float softcap, int dtype, hipStream_t stream) {
  if (n_rows <= 0) return 0;
  if (!q || !out || !k_pages || !vt_pages || !order || !own_begin || !shared_parts || !positions || !block_table || !part_o || !part_ml)
    return -1;
  if (n_items < 0 || (n_items && !items) || n_kv < 1 || n_kv > 65535 || n_q < n_kv || n_q % n_kv || page_size < 16 || page_size % 16 || n_pages < 1 ||
      slots < 1 || own_splits < 1 || own_keys < SP_BLOCK || own_keys % SP_BLOCK || table_stride < 1) return -1;
  SharedArgs a = {};
  a.q = q; a.k_pages = k_pages; a.vt_pages = vt_pages; a.part_o = (float*)part_o; a.part_ml = (float*)part_ml;
  a.items = (const SharedItem*)items; a.order = (const int*)order; a.own_begin = (const int*)own_begin;
  a.shared_parts = (const int*)shared_parts; a.positions = (const int*)positions; a.block_table = (const int*)block_table;
  a.sinks = (const float*)sinks; a.q_stride = q_stride; a.table_stride = table_stride; a.n_items = n_items; a.n_rows = n_rows;
  a.n_q = n_q; a.n_kv = n_kv; a.page_size = page_size; a.n_pages = n_pages; a.slots = slots; a.own_splits = own_splits;
  a.own_keys = own_keys; a.scale = scale; a.softcap = softcap;
#define SHARED_CASE(D) \
  case D: return dtype == DT_F32 ? launch_shared<float, D>(a, out, columns, stream) : launch_shared<bf16_t, D>(a, out, columns, stream);
  switch (head_dim) {
    SHARED_CASE(16) SHARED_CASE(32) SHARED_CASE(48) SHARED_CASE(64) SHARED_CASE(80) SHARED_CASE(96) SHARED_CASE(112)
    SHARED_CASE(128) SHARED_CASE(160) SHARED_CASE(192) SHARED_CASE(224) SHARED_CASE(256)
    default: return -2;
  }
}
