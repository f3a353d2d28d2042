// Operators around a paged key-value cache (gfx950 / CDNA4 only): the step's plan, rotary rows stored to the cache, and
// attention of single rows over it.  The cache holds pages of page_size tokens, [pages][kv_heads][page_size][dim], so a
// head's tokens of one page are one contiguous run.
#include "paged.h"
#include "../../include/vits_amd.h"

#include <type_traits>

namespace vits {
namespace {

constexpr int WAVE = 64;

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// ---------------------------------------------------------------------------------------------------------
// page plan.  With a = max(grow, 0), held = ceil(length / page), fresh = ceil((length + a) / page) - held and back =
// held of a request that ends, three prefix sums over the requests say which rows, which free pages and which ring
// places are whose.  Every block takes those sums over all requests itself (two passes over 8 bytes a request, from
// L2) and then serves its own tile of rows and its own share of the requests: one launch, no second pass over memory,
// and every block comes to the same verdict on whether the step fits before anything is written.
// A fresh page p of a request begins at position p * page >= length, so the row at that position is the one that
// writes the table entry.  Pages are taken at the ring's head and returned at its tail; head .. tail never holds more
// pages than the ring, so no place is read by one block and written by another.
// Bound by latency, not by its bytes: a launch, one dependent load, a scan and a barrier for the sums, the same again for the
// rows, one table entry.  One block would do for the sums, but its rows would then wait for a second launch.  48 requests, a row
// each: 4.8 us; 700 requests, 62 k rows (1.06 MB): 7.5 us; 256 prompts, 254 k rows (4.2 MB): 6.6 us (0.6 TB/s).  Every block reads every
// request, and a block serves 32 of them at most, so many requests cost their square: 4096 take 17 us, 16384 120 us, 65535 1.9 ms.
// ---------------------------------------------------------------------------------------------------------
constexpr int PLAN_THREADS = 256;
constexpr int PLAN_ROWS = 1024;              // rows of a block: four consecutive ones a thread, 16-byte stores
constexpr int PLAN_SHARE = 32;               // requests whose lengths and returned pages a block writes, at most: its four waves
                                             // return pages a request at a time

// Sums that stop at 2^31 - 1: beyond any number of rows or pages that a call may have, so a step that is too large is found
// out without a second word for each sum.
struct PlanSums {
  unsigned rows, fresh, back;
};
__device__ __forceinline__ unsigned plan_add(unsigned a, unsigned b) { return min(a + b, 0x7fffffffu); }
// a request's share of them, and the pages it holds before and after
struct PlanOf {
  unsigned rows, held, after;
  __device__ __forceinline__ unsigned fresh() const { return after - held; }
  __device__ __forceinline__ unsigned back(int grow) const { return grow < 0 ? held : 0u; }
};
__device__ __forceinline__ PlanOf plan_of(int len, int grow, unsigned page) {      // len >= 0, len + grow < 2^31
  const unsigned a = grow < 0 ? 0u : (unsigned)grow, l = (unsigned)len;
  return PlanOf{a, (l + page - 1) / page, (l + a + page - 1) / page};              // page <= 65536: below 2^32
}

__global__ __launch_bounds__(PLAN_THREADS) void page_plan_kernel(PagePlanArgs a) {
  __shared__ PlanSums wave_sum[PLAN_THREADS / WAVE];
  __shared__ int wave_bad[PLAN_THREADS / WAVE], wave_mark[PLAN_THREADS / WAVE];
  __shared__ int mark[PLAN_ROWS], m_base[PLAN_ROWS], m_held[PLAN_ROWS], m_fresh[PLAN_ROWS];
  __shared__ int gone[PLAN_SHARE], gone_held[PLAN_SHARE], gone_at[PLAN_SHARE], n_gone;
  const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
  const unsigned page = (unsigned)a.page_size;
  const int each = (a.requests + PLAN_THREADS - 1) / PLAN_THREADS;
  const int s0 = min(tid * each, a.requests), s1 = min(s0 + each, a.requests);

  const long long head = a.cursor[0], tail = a.cursor[1], free_pages = tail - head;

  // pass 1: this thread's requests
  PlanSums mine = {0, 0, 0};
  int bad = 0;
  for (int s = s0; s < s1; ++s) {
    const int len = a.lengths[s], g = a.grow[s];
    if (len < 0 || g < -1 || (g > 0 && len > 0x7fffffff - g)) { bad |= VITS_PLAN_BAD_LENGTH; continue; }
    const PlanOf p = plan_of(len, g, page);
    if (p.after > (unsigned)a.width) bad |= VITS_PLAN_TABLE_FULL;
    mine = PlanSums{plan_add(mine.rows, p.rows), plan_add(mine.fresh, p.fresh()), plan_add(mine.back, p.back(g))};
  }
  PlanSums upto = mine;                      // inclusive over the wave
#pragma unroll
  for (int d = 1; d < WAVE; d <<= 1) {
    const unsigned r = __shfl_up(upto.rows, d, WAVE), f = __shfl_up(upto.fresh, d, WAVE), b = __shfl_up(upto.back, d, WAVE);
    if (lane >= d) upto = PlanSums{plan_add(upto.rows, r), plan_add(upto.fresh, f), plan_add(upto.back, b)};
    bad |= __shfl_xor(bad, d, WAVE);
  }
  if (lane == WAVE - 1) { wave_sum[wave] = upto; wave_bad[wave] = bad; }
  for (int i = tid; i < PLAN_ROWS; i += PLAN_THREADS) mark[i] = -1;
  if (tid == 0) n_gone = 0;
  __syncthreads();
  PlanSums total = {0, 0, 0}, before = {upto.rows - mine.rows, upto.fresh - mine.fresh, upto.back - mine.back};   // of use if none stopped
  bad = 0;
#pragma unroll
  for (int w = 0; w < PLAN_THREADS / WAVE; ++w) {
    const PlanSums x = wave_sum[w];
    if (w < wave) before = PlanSums{before.rows + x.rows, before.fresh + x.fresh, before.back + x.back};
    total = PlanSums{plan_add(total.rows, x.rows), plan_add(total.fresh, x.fresh), plan_add(total.back, x.back)};
    bad |= wave_bad[w];
  }
  if (head < 0 || free_pages < 0 || free_pages > a.pages || free_pages + total.back > a.pages) bad |= VITS_PLAN_BAD_RING;
  if (total.rows > (unsigned)a.rows) bad |= VITS_PLAN_ROWS_FULL;
  if (total.fresh > free_pages) bad |= VITS_PLAN_NO_PAGES;
  // (a counter of less than 2^32 pages is divided in 32 bits: 64 take a long routine)
  auto place_of = [&](long long c) { return bad ? 0 : c >> 32 ? (int)(c % a.pages) : (int)((unsigned)c % (unsigned)a.pages); };
  const int ring0 = place_of(head), ring1 = place_of(tail);

  // pass 2: mark where requests begin in this block's rows; write what belongs to this block's share of the requests
  const unsigned row0 = blockIdx.x * PLAN_ROWS;           // below 2^30 + PLAN_ROWS
  const int share = (a.requests + gridDim.x - 1) / gridDim.x, own0 = blockIdx.x * share, own1 = own0 + share;   // at most PLAN_SHARE
  for (int s = s0; s < s1; ++s) {
    const int len = a.lengths[s], g = a.grow[s];
    const bool own = s >= own0 && s < own1;
    if (bad) {
      if (own) { a.lengths_out[s] = len; a.row_start[s] = 0; }
      continue;
    }
    const PlanOf p = plan_of(len, g, page);
    if (own) {
      a.lengths_out[s] = g < 0 ? 0 : len + g;
      a.row_start[s] = (int)before.rows;
      if (p.back(g) > 0) {
        const int n = atomicAdd(&n_gone, 1);           // the order in this list does not reach the results
        gone[n] = s; gone_held[n] = (int)p.held; gone_at[n] = (int)before.back;
      }
    }
    if (p.rows > 0 && before.rows < row0 + PLAN_ROWS && before.rows + p.rows > row0) {
      const int at = before.rows > row0 ? (int)(before.rows - row0) : 0;
      mark[at] = s;
      m_base[at] = len - (int)before.rows;
      m_held[at] = (int)p.held;
      m_fresh[at] = (int)before.fresh;
    }
    before = PlanSums{before.rows + p.rows, before.fresh + p.fresh(), before.back + p.back(g)};
  }
  if (blockIdx.x == 0 && tid == 0) {
    a.row_start[a.requests] = bad ? 0 : (int)total.rows;
    a.cursor_out[0] = bad ? head : head + total.fresh;
    a.cursor_out[1] = bad ? tail : tail + total.back;
    a.status[0] = bad;
  }
  __syncthreads();

  // rows: the last mark at or before a row names its request
  const int r0 = tid * 4;
  int at[4], last = -1;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (mark[r0 + i] >= 0) last = r0 + i;
    at[i] = last;
  }
  int scan = last;
#pragma unroll
  for (int d = 1; d < WAVE; d <<= 1) {
    const int v = __shfl_up(scan, d, WAVE);
    if (lane >= d) scan = max(scan, v);
  }
  if (lane == WAVE - 1) wave_mark[wave] = scan;
  __syncthreads();
  int prev = __shfl_up(scan, 1, WAVE);
  if (lane == 0) prev = -1;
  for (int w = 0; w < wave; ++w) prev = max(prev, wave_mark[w]);
  int req[4], pos[4];
  int64_t slot[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long row = (long long)row0 + r0 + i;
    const int m = max(at[i], prev);
    req[i] = pos[i] = -1;
    slot[i] = -1;
    if (!bad && m >= 0 && row < total.rows) {
      req[i] = mark[m];
      pos[i] = (int)row + m_base[m];
      const unsigned p = (unsigned)pos[i] / page, off = (unsigned)pos[i] % page;
      int* entry = a.table + req[i] * a.table_stride + p;
      int id;
      if ((int)p >= m_held[m]) {
        int place = ring0 + m_fresh[m] + ((int)p - m_held[m]) - a.pages;   // both terms are below a.pages
        if (place < 0) place += a.pages;
        id = a.ring[place];
        if (off == 0) *entry = id;
      } else {
        id = *entry;
      }
      slot[i] = (int64_t)id * page + off;
    }
  }
  const long long first = (long long)row0 + r0;
  if (first + 4 <= a.rows && ((reinterpret_cast<uintptr_t>(a.row_request) | reinterpret_cast<uintptr_t>(a.row_position) |
                               reinterpret_cast<uintptr_t>(a.row_slot)) & 15) == 0) {
    *reinterpret_cast<int4*>(a.row_request + first) = make_int4(req[0], req[1], req[2], req[3]);
    *reinterpret_cast<int4*>(a.row_position + first) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    *reinterpret_cast<longlong2*>(a.row_slot + first) = make_longlong2(slot[0], slot[1]);
    *reinterpret_cast<longlong2*>(a.row_slot + first + 2) = make_longlong2(slot[2], slot[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (first + i < a.rows) {
        a.row_request[first + i] = req[i];
        a.row_position[first + i] = pos[i];
        a.row_slot[first + i] = slot[i];
      }
  }

  // pages of requests that end, a wave per request
  const int ends = n_gone;
  for (int n = wave; n < ends; n += PLAN_THREADS / WAVE) {
    const int* from = a.table + gone[n] * a.table_stride;
    for (int j = lane; j < gone_held[n]; j += WAVE) {
      int place = ring1 + gone_at[n] + j - a.pages;
      if (place < 0) place += a.pages;
      a.ring[place] = from[j];
    }
  }
}

// ---------------------------------------------------------------------------------------------------------
// rotary rows, stored to the cache.  A pair of channels (a, b) turns to (a cos - b sin, b cos + a sin); every value is read and
// written once, so a prompt is bound by memory: 8192 rows of 32 + 8 + 8 heads of 128 in bf16, 201 MB, take 43.8 us, 4.6 TB/s
// (a plain copy: 4.9).  A block computes the angles of its rows once, in LDS, for all their heads: a transcendental a pair and
// row instead of one a value.  Few rows are bound by the chain launch - position - angle - barrier - slot - values: one row 2.4
// us, 192 rows of 48 heads of 128 (4.45 MB) 4.0 us; loading the values before the angles was no faster there (the longer code
// costs as much as it hides) and slower on prompts (51 us).
// ---------------------------------------------------------------------------------------------------------
template <typename T> struct Conv;
template <> struct Conv<float> {
  static __device__ __forceinline__ float to(float x) { return x; }
  static __device__ __forceinline__ float from(float x) { return x; }
};
template <> struct Conv<_Float16> {
  static __device__ __forceinline__ float to(_Float16 x) { return (float)x; }
  static __device__ __forceinline__ _Float16 from(float x) { return (_Float16)x; }
};
template <> struct Conv<__bf16> {
  static __device__ __forceinline__ float to(__bf16 x) { return (float)x; }
  static __device__ __forceinline__ __bf16 from(float x) { return (__bf16)x; }
};

template <typename T, int N> struct alignas(sizeof(T) * N) Pack { T v[N]; };

// cos and sin of position * freq, times scale.  A far position leaves fp32 no bits for the angle within its turn
// (position 10^6: half a radian), so the product and the reduction to an eighth of a turn are in 64 bits; what is left
// is rounded to fp32 once, where its error is 2^-24 of at most pi / 4.
__device__ __forceinline__ void rotary_angle(int position, double freq, float scale, f32x2& cs) {
  const double turns = (double)position * freq * 0.15915494309189533577;      // 1 / (2 pi)
  const double whole = rint(turns);
  const double part = turns - whole;                     // -1/2 .. 1/2
  const double quarter = rint(part * 4.0);
  float s0, c0;
  sincospif((float)((part - quarter * 0.25) * 2.0), &s0, &c0);
  const int k = (int)quarter & 3;
  cs.x = scale * (k == 0 ? c0 : k == 1 ? -s0 : k == 2 ? -c0 : s0);
  cs.y = scale * (k == 0 ? s0 : k == 1 ? c0 : k == 2 ? -s0 : -c0);
}

// written as products and sums of its own choice, so that every variant below gives the same bits
__device__ __forceinline__ void rotary_turn(float& u, float& w, float c, float s) {
  const float x = fmaf(u, c, -(w * s)), y = fmaf(w, c, u * s);
  u = x;
  w = y;
}

constexpr int ROT_THREADS = 256;

// 16 bytes at the alignment of their values: global memory takes them at any address
template <int ALIGN> struct AnyAt;
template <> struct AnyAt<2> { typedef unsigned x4 __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct AnyAt<4> { typedef unsigned x4 __attribute__((ext_vector_type(4), aligned(4))); };

// An item is 16 bytes of a head: N channels of both halves (half layout) or N / 2 pairs (interleaved) that turn, N channels
// that pass through, N channels of a value.  RAGGED: not all of these are whole items; what is left of each goes one by one
// (with single channels throughout, 862 rows of 40 heads of 192 of which 182 turn took 19 us, now 8.1).
struct RotaryPart {
  int wide, all;                                         // whole items, and with the single ones
  __host__ __device__ RotaryPart(int channels, int n, int unit) : wide(channels / n), all(channels / n + channels % n / unit) {}
};

// A block takes rows_per_block rows, or a slice of one row's items.
template <typename T, bool INTER, bool RAGGED>
__global__ __launch_bounds__(ROT_THREADS) void rotary_store_kernel(RotaryArgs a, int rows_per_block, int slice) {
  constexpr int N = 16 / sizeof(T), TWO = INTER ? 2 : 1;
  using At = AnyAt<sizeof(T)>;
  extern __shared__ f32x2 cs[];                          // [rows_per_block][pairs]: cos and sin, and what a single item reads beyond
  const int tid = threadIdx.x;
  const int row0 = blockIdx.x * rows_per_block, rows = min(rows_per_block, a.rows - row0);
  for (int i = tid; i < rows * a.pairs; i += ROT_THREADS) {
    const int r = i / a.pairs, p = i % a.pairs;
    rotary_angle(a.position[row0 + r], a.freq[p], a.scale, cs[i]);
  }
  __syncthreads();
  const RotaryPart turn(TWO * a.pairs, N, TWO), pass(a.dim - 2 * a.pairs, N, 1), whole(a.dim, N, 1);
  const int n_turn = RAGGED ? turn.all : turn.wide, n_whole = RAGGED ? whole.all : whole.wide, per_head = n_turn + (RAGGED ? pass.all : pass.wide);
  const int n_q = a.heads * per_head, n_k = a.kv_heads * per_head, per_row = n_q + n_k + a.kv_heads * n_whole;
  const int first = blockIdx.y * slice, last = min(rows * per_row, first + slice);
  const int64_t slots = (int64_t)a.pages * a.page_size;

  auto load = [](const T* src, bool one) {
    u32x4 x = {0, 0, 0, 0};
    if (!RAGGED || !one) x = *(const typename At::x4*)src;
    else if constexpr (sizeof(T) == 4) x[0] = *(const unsigned*)src;
    else x[0] = *(const unsigned short*)src;
    return x;
  };
  auto store = [](T* dst, const u32x4& x, bool one) {
    if (!RAGGED || !one) *(typename At::x4*)dst = x;
    else if constexpr (sizeof(T) == 4) *(unsigned*)dst = x[0];
    else *(unsigned short*)dst = (unsigned short)x[0];
  };
  for (int i = first + tid; i < last; i += ROT_THREADS) {
    const int r = i / per_row, row = row0 + r;
    int j = i - r * per_row;
    int64_t slot = a.slot ? a.slot[row] : 0;
    if (slot < 0) continue;
    if (a.slot && a.k && slot >= slots) {
      if (a.err_flag && j == 0) atomicOr(a.err_flag, 1);
      continue;
    }
    const int64_t pg = a.k ? slot / a.page_size : 0;
    const int64_t cell = pg * a.page_stride + (slot - pg * a.page_size) * a.dim;
    // channel of item j of a part, and whether it is a single one
    auto channel = [](int j, int wide, int unit) { return RAGGED && j >= wide ? wide * N + (j - wide) * unit : j * N; };
    if (j >= n_q + n_k) {
      j -= n_q + n_k;
      const int h = j / n_whole;
      j -= h * n_whole;
      const int c = channel(j, whole.wide, 1);
      const bool one = j >= whole.wide;
      store((T*)a.v_cache + cell + (int64_t)h * a.page_size * a.dim + c, load((const T*)a.v + row * a.v_row + h * a.v_head + c, one), one);
      continue;
    }
    const T* src;
    T* dst;
    int h;
    if (j < n_q) {
      h = j / per_head;
      src = (const T*)a.q + row * a.q_row + h * a.q_head;
      dst = (T*)a.out + row * a.out_row + h * a.out_head;
    } else {
      j -= n_q;
      h = j / per_head;
      src = (const T*)a.k + row * a.k_row + h * a.k_head;
      dst = (T*)a.k_cache + cell + (int64_t)h * a.page_size * a.dim;
    }
    j -= h * per_head;
    if (j >= n_turn) {
      j -= n_turn;
      const int c = 2 * a.pairs + channel(j, pass.wide, 1);
      const bool one = j >= pass.wide;
      store(dst + c, load(src + c, one), one);
      continue;
    }
    const int c = channel(j, turn.wide, TWO);
    const bool one = j >= turn.wide;
    const f32x2* ang = cs + r * a.pairs + c / TWO;
    struct Values { T v[N]; };
    Values x = __builtin_bit_cast(Values, load(src + c, one)), y = x;
    if constexpr (!INTER) y = __builtin_bit_cast(Values, load(src + a.pairs + c, one));
    else if (RAGGED && one) x.v[1] = src[c + 1];
#pragma unroll
    for (int e = 0; e < N / TWO; ++e) {
      T &lo = x.v[TWO * e], &hi = INTER ? x.v[TWO * e + 1] : y.v[e];
      float u = Conv<T>::to(lo), w = Conv<T>::to(hi);
      rotary_turn(u, w, ang[e].x, ang[e].y);
      lo = Conv<T>::from(u);
      hi = Conv<T>::from(w);
    }
    store(dst + c, __builtin_bit_cast(u32x4, x), one);
    if constexpr (!INTER) store(dst + a.pairs + c, __builtin_bit_cast(u32x4, y), one);
    else if (RAGGED && one) dst[c + 1] = x.v[1];
  }
}

template <typename T, bool INTER, bool RAGGED>
hipError_t start_rotary(const RotaryArgs& a, hipStream_t s) {
  constexpr int N = 16 / sizeof(T);
  const RotaryPart turn(INTER ? 2 * a.pairs : a.pairs, N, INTER ? 2 : 1), pass(a.dim - 2 * a.pairs, N, 1), whole(a.dim, N, 1);
  const int per_row = (a.heads + a.kv_heads) * (turn.all + pass.all) + a.kv_heads * whole.all;
  // Up to 2^21 items one a thread, beyond about four, for which the angles serve then.  (862 rows of 40 ragged heads of 192,
  // 7e5 items: 8.1 us with one, 11.5 with four; 8192 rows of 40 heads of 128, 3.7e6 items: 50 us with one, 44 with four.)
  const bool few = (long long)a.rows * per_row <= 1 << 21;
  int rpb = min(min(16, a.rows), few ? max(1, ROT_THREADS / per_row) : (1024 + per_row - 1) / per_row);
  while (rpb > 1 && (a.rows + rpb - 1) / rpb < 256) rpb = (rpb + 1) / 2;   // few rows: spread them over the CUs
  const int slices = few && rpb == 1 ? (per_row + ROT_THREADS - 1) / ROT_THREADS : 1;
  const int slice = rpb == 1 ? (per_row + slices - 1) / slices : rpb * per_row;
  const size_t lds = ((size_t)rpb * a.pairs * 2 + 2 * N) * sizeof(float);          // at most 16 KiB and a little
  hipLaunchKernelGGL((rotary_store_kernel<T, INTER, RAGGED>), dim3((a.rows + rpb - 1) / rpb, slices), dim3(ROT_THREADS), lds, s, a, rpb, slice);
  return hipGetLastError();
}

template <typename T>
hipError_t start_rotary_t(RotaryArgs a, hipStream_t s) {
  constexpr int N = 16 / sizeof(T);
  if (!a.k) a.kv_heads = 0;
  if (!a.q) a.heads = 0;
  const bool ragged = a.dim % N || (a.interleaved ? 2 * a.pairs : a.pairs) % N || (a.dim - 2 * a.pairs) % N;
  if (a.interleaved) return ragged ? start_rotary<T, true, true>(a, s) : start_rotary<T, true, false>(a, s);
  return ragged ? start_rotary<T, false, true>(a, s) : start_rotary<T, false, false>(a, s);
}

// ---------------------------------------------------------------------------------------------------------
// attention of single rows over the cache
//
// Per key-value head the query heads of its group, for up to 16 / group rows of one request that stand beside each other (a
// single new token, drafted tokens, a prompt's rows), are the 16 columns of a matrix product: S^T = K Q^T with 16 keys as
// rows, then O^T = V^T P^T.  In both the result's column is lane & 15, so a column's maximum, sum and rescaling factor
// stay in the lanes that hold its scores and its output.  The contraction of the second product runs over the keys in
// the order the first one leaves them in the lanes (lane group g = lane / 16 holds keys 4g .. 4g + 3 of each 16), so the
// weights go from one to the other without leaving their lane; V's rows are loaded to match: lane group g loads those
// same rows, lane n of it the channels n * DIM / 16 and on, whole rows in one instruction.  Nothing of the cache passes
// through LDS, and no wave waits for another inside the loop over the keys.
// 16-bit types: v_mfma_f32_16x16x32, 32 keys a step; v_perm pairs the rows' channels to operands.  fp32: v_mfma_f32_16x16x4,
// 16 keys a step.  16-bit weights go in as two terms (w = h + l: 2^-17 relative in bf16, 2^-22 in fp16), so that the result carries
// one rounding only, its own: the products' matrix time is a small part of the load time (without the second terms fp16 was off by
// 2.6e-4 of the result, now 2.1e-4, which is the rounding of the result itself, in the same time).
//
// What bounds it: the cache is read once for all rows and heads of a unit, so long and many rows are bound by memory (64 rows of up
// to 4096 tokens, 8 heads of 128 in bf16, 603 MB: 121 us, 5.0 TB/s; one row over 131 k tokens, 537 MB: 107 us, 5.0; 512 rows of up to
// 1500, fp16, 841 MB: 150 us, 5.6, part of it from the last-level cache).  Short ones are bound by latency: a wave takes 1.3 us for a
// step of 32 keys by itself, so a row alone is spread over the waves of a block.  fp32 rows alone are bound by the matrix rate of
// the few CUs that they reach (16x16x4: 1536 cycles for 16 keys of 96 channels, of whose 16 columns one row of a head of its
// own fills one): one row of 500 tokens, 2 heads of 96: 14.6 us.
// ---------------------------------------------------------------------------------------------------------
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x3a __attribute__((ext_vector_type(3), aligned(4)));
typedef unsigned u32x2a __attribute__((ext_vector_type(2), aligned(4)));
typedef unsigned u32x4a __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr int ATT_WAVES = 4;
constexpr int ATT_THREADS = ATT_WAVES * WAVE;
constexpr int ATT_COLS = 16;                 // columns of the products: (row of a run, query head)
constexpr int ATT_PIECES = 2048;             // the most pieces a call's work is cut into: two waves a SIMD
constexpr int ATT_MIN_STEPS = 2;             // the least a piece holds
constexpr int ATT_FEW = 32;                  // units up to which a join takes a block a column
constexpr int ATT_BLOCK_WAVES = 8;           // waves that take a unit by themselves

// max and sum over the four lanes of a column (lane, lane ^ 16, lane ^ 32, lane ^ 48)
__device__ __forceinline__ float col_max(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float col_sum(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Work is laid out on one line, in steps of STEP keys: run after run (a run: rows of one request, up to rows_per_run of
// them beside each other), for each run its units (key-value head, 16 query heads of its group) one after the other, for
// each unit the run's keys.  A run that sees no key has one step, in which everything is masked.
struct AttPlan {
  int group;               // query heads of a key-value head
  int per_page;            // 16-key parts of a page
  int run_shift;           // rows_per_run = 1 << run_shift: a power of two, at most 16 / group (and at least 1)
  int tiles;               // 16-column tiles of a group
  int units;               // kv_heads * tiles
  int pieces;              // waves that the line is cut for (split form), a multiple of ATT_WAVES
  int wide_out;            // outputs lie on 16-byte addresses
};

struct Run {
  int row, n, req;
  int begin, end;          // keys that any of its rows sees: begin a multiple of 16
  int from;                // where its first row's keys begin
};

// a row's keys [begin, end); true if its position lies outside the table
__device__ __forceinline__ bool att_row_keys(const PagedAttArgs& a, int row, int& begin, int& end) {
  const long long cap = (long long)a.width * a.page_size, stop = (long long)a.row_position[row] + 1;
  const long long first = a.window > 0 && stop > a.window ? stop - a.window : 0;
  end = (int)(stop < 0 ? 0 : stop < cap ? stop : cap);
  begin = (int)(first < end ? first : end);
  return stop > cap;
}

// Whether one of the pages of a request's keys [from, to) is one of the cache's.  Asked where a row's weights sum up to 0: if there is
// one, all its scores are -inf and softmax has no value (0 / 0); if there is none, the row sees nothing.
__device__ __forceinline__ bool att_any_page(const PagedAttArgs& a, int req, int from, int to) {
  const int* table = a.table + (long long)req * a.table_stride;
  bool any = false;
  for (int p = from / a.page_size, last = (to - 1) / a.page_size; p <= last && !any; ++p) any = table[p] >= 0 && table[p] < a.pages;
  return any;
}

// whether a run begins at `row`, and what it is
__device__ __forceinline__ bool att_run(const PagedAttArgs& a, const AttPlan& p, int row, Run& r) {
  const int req = a.row_request[row], before = a.row_request[row > 0 ? row - 1 : 0];
  int end;
  att_row_keys(a, row, r.from, end);                     // loaded beside the requests, not after them
  if (req < 0 || req >= a.requests) return false;
  const int in = row & ((1 << p.run_shift) - 1);
  if (in > 0 && before == req) return false;
  r.row = row;
  r.req = req;
  r.begin = r.from < end ? r.from : 0x7fffffff;
  r.end = end;
  const int most = min((1 << p.run_shift) - in, a.rows - row);
  int n = 1;
  for (; n < most && a.row_request[row + n] == req; ++n) {
    int b, e;
    att_row_keys(a, row + n, b, e);
    if (b < e) r.begin = min(r.begin, b);
    r.end = max(r.end, e);
  }
  r.n = n;
  r.begin = r.begin >= r.end ? 0 : r.begin & ~15;
  return true;
}

// the same for a wave whose lanes all ask about the same row: the run's rows are looked at side by side
__device__ __forceinline__ bool att_run_wave(const PagedAttArgs& a, const AttPlan& p, int row, Run& r) {
  const int lane = threadIdx.x & (WAVE - 1), here = min(row + min(lane, ATT_COLS - 1), a.rows - 1);
  const int req = a.row_request[here], before = a.row_request[row > 0 ? row - 1 : 0];
  int from, to;
  att_row_keys(a, here, from, to);
  auto same = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  const int mine = same(req), in = row & ((1 << p.run_shift) - 1);
  if (mine < 0 || mine >= a.requests || (in > 0 && same(before) == mine)) return false;
  const int most = min((1 << p.run_shift) - in, a.rows - row);
  const unsigned long long other = __ballot(lane >= most || req != mine);          // lane 0 is not among them
  r.n = __builtin_ctzll(other);
  r.row = row;
  r.req = mine;
  r.from = same(from);
  int low = lane < r.n && from < to ? from : 0x7fffffff, high = lane < r.n ? to : 0;
#pragma unroll
  for (int d = 1; d < ATT_COLS; d <<= 1) {
    low = min(low, __shfl_xor(low, d, WAVE));
    high = max(high, __shfl_xor(high, d, WAVE));
  }
  r.end = same(high);
  r.begin = same(low) >= r.end ? 0 : same(low) & ~15;
  return true;
}

// x / y of numbers that are not negative: 64-bit division is a long routine, and these are seldom that large
__device__ __forceinline__ long long att_div(long long x, long long y) {
  return (x | y) >> 32 ? x / y : (long long)((unsigned)x / (unsigned)y);
}

template <int STEP>
__device__ __forceinline__ int att_run_steps(const Run& r) {
  return max(1, (r.end - r.begin + STEP - 1) / STEP);
}

// what a block's pieces leave of a unit that they do not hold whole: [0] for the one the block begins in the middle of, [1]
// for the one it ends in the middle of; joined by paged_join_kernel
__host__ __device__ __forceinline__ float* att_slot(float* ws, int block, int which, int dim) {
  return ws + ((long long)block * 2 + which) * ATT_COLS * (dim + 4);
}
struct AttJoin {           // a unit that begins in a block and ends in a later one
  int row, n, unit, parts; // parts: the blocks behind this one that hold some of it; 0: there is none
};

// Column m of a unit: its row (of the run's n) and head, false if there is none
__device__ __forceinline__ bool att_column(int m, int n, int group, int tile, int& row, int& head) {
  if (group <= ATT_COLS) {
    row = m / group;
    head = m - row * group;
    return row < n;
  }
  row = 0;
  head = tile * ATT_COLS + m;
  return head < group;
}

__device__ __forceinline__ float att_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// keys of a step
__host__ __device__ constexpr int att_step(int size, int dim) { return size == 2 && dim <= 192 ? 32 : 16; }

// A result of a matrix instruction is bound to a wait here, in the block that computes it: read in another block, behind a
// taken branch, the compiler (ROCm 7.2) has been seen to leave it too short (needed: up to 11 issue slots).
#define ATT_SETTLE(x) asm volatile("s_nop 15" : "+v"(x))

template <typename T, int DIM>
struct AttTile {
  static constexpr bool HALF = sizeof(T) == 2;
  // Registers: Q, K, V and O of a step have to fit 256 (two waves a SIMD) with room for the rest.  So wide heads take 16
  // keys a step, and fp32 ones load K and V in two or four passes, each when the one before has been used.
  static constexpr int STEP = att_step(sizeof(T), DIM);
  static constexpr int SUB = STEP / 16;                  // 16-key parts of a step
  static constexpr int PASSES = HALF || DIM <= 160 ? 1 : DIM < 256 ? 2 : 4;
  static constexpr int KL = DIM * (int)sizeof(T) / 64;   // 16-byte loads of a lane for 16 keys
  static constexpr int KP = KL / PASSES;
  static constexpr int CH = DIM / 16;                   // channels of a lane in V and in the output
  static constexpr int VW = CH * (int)sizeof(T) / 4;     // dwords of a lane for one row of V
  static constexpr int VP = VW / PASSES;
  static constexpr int ROW = DIM + 4;                   // floats of a column in LDS and in the workspace, padded
  // The running maximum follows once it is exceeded by 2^SLACK.  fp16 holds nothing below 2^-24, and a long context may have most of its
  // sum in weights below that: there the maximum stands for a weight of 2^LIFT (the largest, 2^15, is still one), so the smallest
  // that counts is 2^-35 of it.
  static constexpr bool F16 = __is_same(T, _Float16);
  static constexpr float SLACK = F16 ? 4.f : 8.f, LIFT = F16 ? 11.f : 0.f;
  static_assert(KL % PASSES == 0 && VW % PASSES == 0);

  u32x4 q[KL], k[SUB][KP];
  unsigned v[SUB][4][VP];
  f32x4 o[CH];
  float top, sum;                                       // of this lane's column: running maximum (base 2), and this lane's part of the sum

  __device__ __forceinline__ void load_k(int s, const T* page, int lane, int pass) {
    const char* p = (const char*)page + (lane & 15) * (DIM * sizeof(T)) + (lane >> 4) * 16 + pass * (KP * 64);
#pragma unroll
    for (int i = 0; i < KP; ++i) k[s][i] = *(const u32x4*)(p + 64 * i);
  }
  __device__ __forceinline__ void load_v(int s, const T* page, int lane, int pass) {
    const char* p = (const char*)page + (lane >> 4) * (4 * DIM * sizeof(T)) + (lane & 15) * (VW * 4) + pass * (VP * 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const char* r = p + j * (DIM * sizeof(T));
      int w = 0;
#pragma unroll
      for (; w + 4 <= VP; w += 4) {
        const u32x4a x = *(const u32x4a*)(r + 4 * w);
        v[s][j][w] = x[0]; v[s][j][w + 1] = x[1]; v[s][j][w + 2] = x[2]; v[s][j][w + 3] = x[3];
      }
      if constexpr (VP % 4 == 3) {
        const u32x3a x = *(const u32x3a*)(r + 4 * w);
        v[s][j][w] = x[0]; v[s][j][w + 1] = x[1]; v[s][j][w + 2] = x[2];
      } else if constexpr (VP % 4 == 2) {
        const u32x2a x = *(const u32x2a*)(r + 4 * w);
        v[s][j][w] = x[0]; v[s][j][w + 1] = x[1];
      } else if constexpr (VP % 4 == 1) {
        v[s][j][w] = *(const unsigned*)(r + 4 * w);
      }
    }
  }

  // s += K^T Q over the channels of a pass
  __device__ __forceinline__ void scores(f32x4 (&s)[SUB], int pass) const {
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      f32x4 c = s[u];
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        const u32x4 y = q[pass * KP + i];
        if constexpr (!HALF) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[u][i][e]), __uint_as_float(y[e]), c, 0, 0, 0);
        } else if constexpr (__is_same(T, __bf16)) {
          c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k[u][i]), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
        } else {
          c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, k[u][i]), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
        }
      }
      s[u] = c;
    }
#pragma unroll
    for (int u = 0; u < SUB; ++u) ATT_SETTLE(s[u]);
  }

  // the weights of a step as operands
  struct Weights {
    f32x4 f;                                            // fp32
    unsigned hi[2 * SUB], lo[2 * SUB];                  // 16 bits: two keys each; lo is what 16 bits leave of a weight
  };
  // lifted: no second term is 0 or negative where the first is not 0 (see att_part); the weight then holds one bit less
  static __device__ __forceinline__ Weights weights(const f32x4 (&p)[SUB], bool lifted) {
    Weights w;
    w.f = p[0];
    if constexpr (HALF) {
#pragma unroll
      for (int i = 0; i < 2 * SUB; ++i) {
        const f32x2 x = {p[i / 2][i % 2 * 2], p[i / 2][i % 2 * 2 + 1]};
        using Two = std::conditional_t<__is_same(T, __bf16), bf16x2, f16x2>;
        const Two h = __builtin_convertvector(x, Two);
        w.hi[i] = __builtin_bit_cast(unsigned, h);
        w.lo[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(x - __builtin_convertvector(h, f32x2), Two));
        if (lifted) {                                    // the number before it as the first term
          const Two l = __builtin_bit_cast(Two, w.lo[i]);
          if (!((float)l[0] > 0.f) && (w.hi[i] & 0xffffu)) w.hi[i] -= 1;
          if (!((float)l[1] > 0.f) && (w.hi[i] >> 16)) w.hi[i] -= 0x10000u;
          w.lo[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(x - __builtin_convertvector(__builtin_bit_cast(Two, w.hi[i]), f32x2), Two));
        }
      }
    }
    return w;
  }
  static __device__ __forceinline__ f32x4 product(const unsigned (&x)[2 * SUB], const unsigned (&y)[2 * SUB], f32x4 c) {
    if constexpr (SUB == 2) {
      const u32x4 a = {x[0], x[1], x[2], x[3]}, b = {y[0], y[1], y[2], y[3]};
      if constexpr (__is_same(T, __bf16))
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
      else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    } else {
      const u32x2 a = {x[0], x[1]}, b = {y[0], y[1]};
      if constexpr (__is_same(T, __bf16))
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
      else
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
    }
  }

  // leaves the keys out of V that `see` has no bit for (one a key of this lane: 4 * part + row)
  __device__ __forceinline__ void mask_v(unsigned see) {
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool seen = see >> (4 * u + j) & 1;
#pragma unroll
        for (int w = 0; w < VP; ++w) v[u][j][w] = seen ? v[u][j][w] : 0u;
      }
  }

  // c[0 .. PER) += V^T P^T for the channels of dword w of a pass: one channel in fp32, two in 16 bits
  static constexpr int PER = HALF ? 2 : 1;
  __device__ __forceinline__ void weigh(f32x4* c, int w, const Weights& p) const {
    if constexpr (!HALF) {
#pragma unroll
      for (int j = 0; j < 4; ++j) c[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[0][j][w]), p.f[j], c[0], 0, 0, 0);
    } else {
      unsigned even[2 * SUB], odd[2 * SUB];
#pragma unroll
      for (int i = 0; i < 2 * SUB; ++i) {
        const unsigned x = v[i / 2][i % 2 * 2][w], y = v[i / 2][i % 2 * 2 + 1][w];
        even[i] = __builtin_amdgcn_perm(y, x, 0x05040100);
        odd[i] = __builtin_amdgcn_perm(y, x, 0x07060302);
      }
      c[0] = product(even, p.lo, c[0]);
      c[1] = product(odd, p.lo, c[1]);
      c[0] = product(even, p.hi, c[0]);
      c[1] = product(odd, p.hi, c[1]);
    }
  }

  // the running softmax over one step's scores (base 2, -inf where masked); s becomes the weights
  __device__ __forceinline__ void soften(f32x4 (&s)[SUB]) {
    float t = s[0][0];
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) t = fmaxf(t, s[u][e]);
    t = col_max(t);
    const bool above = t > top + SLACK;
    if (__ballot(above)) {                              // seldom after the first steps
      const float next = above ? t : top;               // a column goes by its own scores alone
      const float keep = above ? att_exp2(top - next) : 1.f;
      sum *= keep;
#pragma unroll
      for (int c = 0; c < CH; ++c) o[c] *= keep;
      top = next;
    }
    // (of an infinite score nothing is taken away, so that it is the sum that becomes infinite, not a NaN)
    const float base = fabsf(top) == INFINITY ? 0.f : top - LIFT;
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[u][e] = att_exp2(s[u][e] - base);
        sum += s[u][e];
      }
  }
};

// x / sum as the result of a column's quad of channels
template <typename T>
__device__ __forceinline__ void att_write(const PagedAttArgs& a, bool wide, int row, int head, int c, f32x4 x, float sum, bool none) {
  T* to = (T*)a.out + (long long)row * a.out_row + (long long)head * a.out_head + c;
  Pack<T, 4> y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y.v[e] = Conv<T>::from(none ? 0.f : x[e] / sum);
  if (!wide) {
#pragma unroll
    for (int e = 0; e < 4; ++e) to[e] = y.v[e];
  } else if constexpr (sizeof(T) == 4) {
    *(u32x4*)to = __builtin_bit_cast(u32x4, y);
  } else {
    *(u32x2*)to = __builtin_bit_cast(u32x2, y);
  }
}
__device__ __forceinline__ void att_write_lse(const PagedAttArgs& a, int row, int head, float top, float sum, bool none) {
  const float base = top == -INFINITY ? 0.f : top;
  a.lse[(long long)row * a.heads + head] = none ? -INFINITY : (base + log2f(sum)) * 0.6931471805599453f;
}

// A wave's result for its column, or its part of it.  The lane's DIM / 4 channels lie beside each other: 4 lg * CH and on.
template <typename T, int DIM>
__device__ __forceinline__ void att_leave(const PagedAttArgs& a, const AttPlan& p, const AttTile<T, DIM>& w, int col, int lg, int row, int head,
                                          bool none, bool whole, float* slot) {
  constexpr int CH = AttTile<T, DIM>::CH;
  float* to = slot + col * AttTile<T, DIM>::ROW;
#pragma unroll
  for (int c = 0; c < 4 * CH; c += 4) {
    f32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = w.o[(c + e) % CH][(c + e) / CH];
    if (whole) att_write<T>(a, p.wide_out, row, head, 4 * lg * CH + c, x, w.sum, none);
    else *(f32x4*)(to + 4 * lg * CH + c) = x;
  }
  if (lg != 0) return;
  if (!whole) {
    to[DIM] = w.top;
    to[DIM + 1] = w.sum;
  } else if (a.lse) {
    att_write_lse(a, row, head, w.top, w.sum, none);
  }
}

// Steps [t0, t1) of unit `unit` of run r, by one wave.  whole: that is the unit's every step and the result is written, else
// this part goes to `slot`, in LDS.  Returns whether a page was not one of the cache's.
//
// A key that one row of the run sees and another does not has a weight of 0 in the other's column, and 0 times an infinity or
// a NaN in V would reach it.  So where rows differ and a result is not finite, the part is taken again row by row, with what
// the row does not see left out of V.  And 16-bit weights have a second term that may be 0 or negative, which times an infinity in V is
// a NaN beside the first term's infinity: a row that is not finite by itself is taken once more, with two terms above 0.  (A weight
// of fp16 below 2^-34 of the largest is 0 in its first term all the same, and 0 times an infinity a NaN.)
//
// Lanes are switched off in here for the write of a result alone (which, row by row, other rows follow): what a lane must not load it
// loads from where another may, and drops.  With lanes off, the compiler (ROCm 7.2) has been seen to move whole-wave values to
// accumulator registers and back for the lanes that were on alone.  It has none to move to: builds that use them, or scratch, or
// more than 256 vector registers are refused (vits_amd/build.py).
template <typename T, int DIM>
__device__ __forceinline__ bool att_part(const PagedAttArgs& a, const AttPlan& p, const Run& r, int unit, int t0, int t1, bool whole, float* slot) {
  using Tile = AttTile<T, DIM>;
  constexpr int SUB = Tile::SUB, STEP = Tile::STEP, KL = Tile::KL, CH = Tile::CH, PASSES = Tile::PASSES;
  const int lane = threadIdx.x & (WAVE - 1);
  const int col = lane & 15, lg = lane >> 4;
  const int group = p.group, hk = p.tiles == 1 ? unit : unit / p.tiles, tile = unit - hk * p.tiles;
  Tile w;
  int my_row, my_head;
  const bool real = att_column(col, r.n, group, tile, my_row, my_head);
  my_row = real ? my_row : 0;
  my_head = real ? my_head : 0;
  int begin = r.from, end = r.end;
  if (r.n > 1) att_row_keys(a, r.row + my_row, begin, end);
  {
    const T* q = (const T*)a.q + (long long)(r.row + my_row) * a.q_row + (long long)(hk * group + my_head) * a.q_head;
#pragma unroll
    for (int i = 0; i < KL; ++i) w.q[i] = *(const u32x4*)(q + (64 * i + 16 * lg) / (int)sizeof(T));
  }
  const float scale = a.scale * 1.4426950408889634f;     // scores in powers of two

  // Where the 16-key parts of the next 64 / SUB steps lie, one part a lane: elements from the cache's beginning
  // (16 keys never straddle a page), 0 and a bit in `out` for a part that no row sees or whose page is none.
  const int* table = a.table + (long long)r.req * a.table_stride;
  const long long head_off = (long long)hk * a.page_size * DIM;
  long long at = 0;
  unsigned long long out = 0, stray = 0;
  auto locate = [&](int first) {
    const int t = first + lane / SUB;
    const int key = r.begin + t * STEP + 16 * (lane % SUB);
    const bool seen = t < t1 && key < r.end;
    const int part = (seen ? key : r.begin) / 16, page = part / p.per_page;
    const int id = table[page];
    const bool there = id >= 0 && id < a.pages;
    stray |= __ballot(seen && !there);
    out = __ballot(!seen || !there);
    at = seen && there ? (long long)id * a.page_stride + head_off + (long long)(part - page * p.per_page) * 16 * DIM : 0;
  };
  auto part_at = [&](int i) -> long long {               // the part that lane i has located, the same for the wave
    const unsigned lo = __builtin_amdgcn_readlane((unsigned)at, i), hi = __builtin_amdgcn_readlane((unsigned)(at >> 32), i);
    return (long long)((unsigned long long)hi << 32 | lo);
  };
  const T *kc = (const T*)a.k_cache, *vc = (const T*)a.v_cache;
  constexpr int ROUND = WAVE / SUB;                      // steps that one call of locate() serves

  bool lifted = false;
  for (int alone = -1;;) {                               // -1: all rows together, else the row that is taken
    // keys that any and that every column in question sees
    const bool mine = real && (alone < 0 || my_row == alone);
    int all_from = mine ? begin : 0, all_to = mine ? end : 0x7fffffff, any_from = mine ? begin : 0x7fffffff, any_to = mine ? end : 0;
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
      all_from = max(all_from, __shfl_xor(all_from, d, WAVE));
      all_to = min(all_to, __shfl_xor(all_to, d, WAVE));
      any_from = min(any_from, __shfl_xor(any_from, d, WAVE));
      any_to = max(any_to, __shfl_xor(any_to, d, WAVE));
    }
    all_from = __builtin_amdgcn_readfirstlane(all_from);
    all_to = __builtin_amdgcn_readfirstlane(all_to);
    any_from = __builtin_amdgcn_readfirstlane(any_from);
    any_to = __builtin_amdgcn_readfirstlane(any_to);
#pragma unroll
    for (int c = 0; c < CH; ++c) w.o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    w.top = -INFINITY;
    w.sum = 0.f;
    int t = t0, in = 0;
    long long here[SUB];
    locate(t);
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      here[u] = part_at(u);
      w.load_k(u, kc + here[u], lane, 0);
    }
#pragma unroll
    for (int u = 0; u < SUB; ++u) w.load_v(u, vc + here[u], lane, 0);
    while (t < t1) {
      const int key0 = r.begin + t * STEP;
      const unsigned bad = (unsigned)(out >> (in * SUB)) & ((1u << SUB) - 1);
      f32x4 s[SUB];
#pragma unroll
      for (int u = 0; u < SUB; ++u) s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int pass = 0; pass < PASSES; ++pass) {
        if (pass > 0) {
#pragma unroll
          for (int u = 0; u < SUB; ++u) w.load_k(u, kc + here[u], lane, pass);
        }
        w.scores(s, pass);
      }
      ++t;
      ++in;
      long long next[SUB];
#pragma unroll
      for (int u = 0; u < SUB; ++u) next[u] = here[u];
      if (t < t1) {
        if (in == ROUND) {
          locate(t);
          in = 0;
        }
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
          next[u] = part_at(in * SUB + u);
          w.load_k(u, kc + next[u], lane, 0);
        }
      }
#pragma unroll
      for (int u = 0; u < SUB; ++u) s[u] *= scale;
      const bool all = bad == 0 && key0 >= all_from && key0 + STEP <= all_to;
      // this lane's keys that lie in [from, to): one bit each, 4 * part + row
      auto sees = [&](int from, int to) {
        unsigned m = 0;
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + 16 * u + 4 * lg + e;
            m |= (unsigned)(key >= from && key < to && !(bad >> u & 1)) << (4 * u + e);
          }
        return m;
      };
      if (!all) {
        const unsigned m = sees(begin, end);
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[u][e] = m >> (4 * u + e) & 1 ? s[u][e] : -INFINITY;
      }
      w.soften(s);
      const typename Tile::Weights x = Tile::weights(s, lifted);
#pragma unroll
      for (int pass = 0; pass < PASSES; ++pass) {
        if (pass > 0) {
#pragma unroll
          for (int u = 0; u < SUB; ++u) w.load_v(u, vc + here[u], lane, pass);
        }
        if (!all) w.mask_v(sees(any_from, any_to));
#pragma unroll
        for (int d = 0; d < Tile::VP; ++d) w.weigh(&w.o[(pass * Tile::VP + d) * Tile::PER], d, x);
      }
#pragma unroll
      for (int u = 0; u < SUB; ++u) here[u] = next[u];
      if (t < t1) {
#pragma unroll
        for (int u = 0; u < SUB; ++u) w.load_v(u, vc + here[u], lane, 0);
      }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) ATT_SETTLE(w.o[c]);
    w.sum = col_sum(w.sum);
    w.top -= Tile::LIFT;                                  // from here on what a weight of 1 stands for
    if ((alone < 0 && r.n > 1) || (Tile::HALF && !lifted)) {
      bool wild = false;
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) wild |= !(fabsf(w.o[c][e]) < INFINITY);
      if (__ballot(wild && mine)) {
        lifted = r.n == 1 || alone >= 0;
        alone = max(alone, 0);
        continue;
      }
    }
    bool none = begin >= end;
    const bool zero = whole && mine && !none && w.sum == 0.f;
    if (__ballot(zero)) {                                 // as att_any_page does, all lanes side by side over the run's pages
      bool any = !zero;
      for (int page = r.begin / a.page_size; page * a.page_size < r.end && __ballot(!any); ++page) {
        const int id = table[page], key = page * a.page_size;
        any = any || (id >= 0 && id < a.pages && key < end && key + a.page_size > begin);
      }
      none = none || !any;
    }
    if (mine) att_leave<T, DIM>(a, p, w, col, lg, r.row + my_row, hk * group + my_head, none, whole, slot);
    if (alone < 0 || ++alone == r.n) return stray != 0;
    lifted = false;
  }
}

// requests and positions outside the table are not followed
__device__ __forceinline__ void att_flag_row(const PagedAttArgs& a, int row) {
  const int req = a.row_request[row];
  int b, e;
  if (req >= a.requests || (req >= 0 && att_row_keys(a, row, b, e))) atomicOr(a.err_flag, 1);
}

// Joins a block's parts of one unit, N of them in LDS (those that are none have a null pointer), a thread a quad of channels.
// slot: where the joined part goes; null: it is the whole unit and the result is written.
template <typename T, int DIM, int N, int THREADS>
__device__ __forceinline__ void att_join(const PagedAttArgs& a, const AttPlan& p, int row0, int n_rows, int unit, int begin, int end,
                                         const float* const (&part)[N], const float* any, float* slot) {
  constexpr int ROW = DIM + 4, QUADS = DIM / 4;
  const int hk = p.tiles == 1 ? unit : unit / p.tiles, tile = unit - hk * p.tiles;
#pragma unroll
  for (int i0 = 0; i0 < ATT_COLS * QUADS; i0 += THREADS) {
    const int i = i0 + (int)threadIdx.x, m = i / QUADS, c = i % QUADS * 4;
    int row, head;
    if (i >= ATT_COLS * QUADS || !att_column(m, n_rows, p.group, tile, row, head)) continue;
    float tops[N], sums[N];
    f32x4 xs[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {                        // all loads at once: what is no part is read from one and has no weight
      const float* from = (part[j] ? part[j] : any) + m * ROW;
      tops[j] = from[DIM];
      sums[j] = from[DIM + 1];
      xs[j] = *(const f32x4*)(from + c);
    }
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) top = part[j] ? fmaxf(top, tops[j]) : top;
    const float base = fabsf(top) == INFINITY ? 0.f : top;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (part[j]) {
        const float f = att_exp2(tops[j] - base);
        sum += f * sums[j];
        x += f * xs[j];
      }
    if (slot) {
      *(f32x4*)(slot + m * ROW + c) = x;
      if (c == 0) {
        slot[m * ROW + DIM] = top;
        slot[m * ROW + DIM + 1] = sum;
      }
      continue;
    }
    int from = begin, to = end;
    if (n_rows > 1) att_row_keys(a, row0 + row, from, to);
    const bool none = from >= to || (sum == 0.f && !att_any_page(a, a.row_request[row0], from, to));
    att_write<T>(a, p.wide_out, row0 + row, hk * p.group + head, c, x, sum, none);
    if (a.lse && c == 0) att_write_lse(a, row0 + row, hk * p.group + head, top, sum, none);
  }
}

// A wave a unit: for so many units that they fill the chip, of lengths that a wave takes in a short time.  No workspace, no
// second launch.
template <typename T, int DIM>
__global__ __launch_bounds__(ATT_THREADS, 2) void paged_attention_wave_kernel(PagedAttArgs a, AttPlan p) {
  const long long n = (long long)blockIdx.x * ATT_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int row = (int)att_div(n, p.units), unit = (int)(n - (long long)row * p.units);
  if (row >= a.rows) return;
  Run r;
  if (att_run_wave(a, p, row, r) && att_part<T, DIM>(a, p, r, unit, 0, att_run_steps<AttTile<T, DIM>::STEP>(r), true, nullptr) && a.err_flag)
    atomicOr(a.err_flag, 1);
  if (a.err_flag && unit == 0 && threadIdx.x % WAVE == 0) att_flag_row(a, row);
}

// A block a unit, its waves a stretch of the keys each, joined in LDS: for fewer units of such lengths.
template <typename T, int DIM>
__global__ __launch_bounds__(ATT_BLOCK_WAVES * WAVE, 1) void paged_attention_block_kernel(PagedAttArgs a, AttPlan p) {
  __shared__ alignas(16) float lds[ATT_BLOCK_WAVES][ATT_COLS * AttTile<T, DIM>::ROW];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int row = blockIdx.x / (unsigned)p.units, unit = blockIdx.x - row * p.units;
  if (a.err_flag && unit == 0 && threadIdx.x == 0) att_flag_row(a, row);
  Run r;
  if (!att_run_wave(a, p, row, r)) return;
  const int steps = att_run_steps<AttTile<T, DIM>::STEP>(r);
  const int each = (steps + ATT_BLOCK_WAVES - 1) / ATT_BLOCK_WAVES, t0 = wave * each, t1 = min(t0 + each, steps);
  if (t0 < t1 && att_part<T, DIM>(a, p, r, unit, t0, t1, false, lds[wave]) && a.err_flag) atomicOr(a.err_flag, 1);
  __syncthreads();
  const float* part[ATT_BLOCK_WAVES];
#pragma unroll
  for (int w = 0; w < ATT_BLOCK_WAVES; ++w) part[w] = w * each < steps ? lds[w] : nullptr;
  att_join<T, DIM, ATT_BLOCK_WAVES, ATT_BLOCK_WAVES * WAVE>(a, p, r.row, r.n, unit, r.from, r.end, part, lds[0], nullptr);
}

// The line of work cut into p.pieces equal pieces, a wave a piece, a block four that follow each other: a long row beside
// short ones, or alone, costs every wave the same.  Each block sums up the rows' steps itself to find where its waves' pieces
// begin.  What its waves hold of one unit is joined in the block, and goes to the workspace only where the unit reaches
// into another block.
template <typename T, int DIM>
__global__ __launch_bounds__(ATT_THREADS, DIM <= 128 ? 2 : 1) void paged_attention_split_kernel(PagedAttArgs a, AttPlan p, float* ws, AttJoin* joins) {
  constexpr int STEP = AttTile<T, DIM>::STEP, ROW = AttTile<T, DIM>::ROW;
  struct Part {             // what a wave leaves of a unit: [0] one that began in an earlier wave, [1] one that goes on in the next
    int live, row, n, unit, from, to;
    int more;               // [0]: it goes on in the next wave; [1]: blocks behind this one that hold some of it
  };
  __shared__ alignas(16) float lds[ATT_WAVES][2][ATT_COLS * ROW];
  __shared__ Part left[ATT_WAVES][2];
  __shared__ long long wave_sum[ATT_WAVES];
  __shared__ long long found_at[ATT_WAVES];
  __shared__ Run found[ATT_WAVES];
  const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
  const int each = (a.rows + ATT_THREADS - 1) / ATT_THREADS;
  const int row0 = min(tid * each, a.rows), row1 = min(row0 + each, a.rows);
  long long mine = 0;
  Run r;
  for (int row = row0; row < row1; ++row) {
    if (att_run(a, p, row, r)) mine += att_run_steps<STEP>(r);
    if (a.err_flag && blockIdx.x == 0) att_flag_row(a, row);
  }
  long long upto = mine;
#pragma unroll
  for (int d = 1; d < WAVE; d <<= 1) {
    const long long x = __shfl_up(upto, d, WAVE);
    if (lane >= d) upto += x;
  }
  if (lane == WAVE - 1) wave_sum[wave] = upto;
  if (tid < 2 * ATT_WAVES) left[tid >> 1][tid & 1].live = 0;
  __syncthreads();
  long long before = upto - mine, total = 0;
  for (int w = 0; w < ATT_WAVES; ++w) {
    if (w < wave) before += wave_sum[w];
    total += wave_sum[w];
  }
  total *= p.units;
  long long size = att_div(total + p.pieces - 1, p.pieces);
  if (size < ATT_MIN_STEPS) size = ATT_MIN_STEPS;
  if (tid == 0) joins[blockIdx.x].parts = 0;
  if (blockIdx.x * ATT_WAVES * size >= total) return;      // the whole block
  for (int w = 0; w < ATT_WAVES; ++w) {                  // the thread whose rows hold the beginning of wave w's piece
    const long long first = (blockIdx.x * ATT_WAVES + w) * size;
    if (first >= total || before * p.units > first || first >= (before + mine) * p.units) continue;
    long long run_at = before;
    for (int row = row0; row < row1; ++row) {
      if (each > 1 && !att_run(a, p, row, r)) continue;    // with a row a thread, r is still that row's
      const int steps = att_run_steps<STEP>(r);
      if (first < (run_at + steps) * p.units) {
        found[w] = r;
        found_at[w] = run_at;
        break;
      }
      run_at += steps;
    }
  }
  __syncthreads();
  const int piece = blockIdx.x * ATT_WAVES + wave;
  const long long first = piece * size, last = first + size < total ? first + size : total;
  if (first < last) {
    auto same = [](int x) { return __builtin_amdgcn_readfirstlane(x); };     // the same for the wave: kept in scalar registers
    const Run f = found[wave];
    r = Run{same(f.row), same(f.n), same(f.req), same(f.begin), same(f.end), same(f.from)};
    const long long at = found_at[wave];
    long long run_at = (long long)((unsigned long long)(unsigned)same((int)(at >> 32)) << 32 | (unsigned)same((int)at)) * p.units;
    long long pos = first;
    int row = r.row;
    bool stray = false;
    for (;;) {
      const int steps = att_run_steps<STEP>(r);
      for (int unit = (int)att_div(pos - run_at, steps); unit < p.units && pos < last; ++unit) {
        const long long unit_at = run_at + (long long)unit * steps;
        const int t0 = (int)(pos - unit_at), t1 = (int)(last - unit_at < steps ? last - unit_at : steps);
        const bool whole = t0 == 0 && t1 == steps;
        if (!whole && lane == 0)
          left[wave][t0 == 0] = Part{1, r.row, r.n, unit, r.from, r.end,
                                     t0 == 0 ? (int)att_div(unit_at + steps - 1, size * ATT_WAVES) - (int)blockIdx.x : t1 < steps};
        stray |= att_part<T, DIM>(a, p, r, unit, t0, t1, whole, lds[wave][t0 == 0]);
        pos = unit_at + t1;
      }
      if (pos >= last) break;
      run_at += (long long)steps * p.units;
      do ++row; while (!att_run_wave(a, p, row, r));         // pos < total: there is one
    }
    if (stray && a.err_flag) atomicOr(a.err_flag, 1);
  }
  __syncthreads();

  // A chain: what the block holds of one unit, beginning with a wave's [1], or (k == 0) with what an earlier block began,
  // and going on in the [0] of the waves behind
  bool live[ATT_WAVES][2], more[ATT_WAVES];
#pragma unroll
  for (int w = 0; w < ATT_WAVES; ++w) {
    live[w][0] = left[w][0].live;
    live[w][1] = left[w][1].live;
    more[w] = left[w][0].more;
  }
#pragma unroll
  for (int k = 0; k <= ATT_WAVES; ++k) {
    if (!(k == 0 ? live[0][0] : live[k - 1][1])) continue;
    const Part head = k == 0 ? left[0][0] : left[k - 1][1];
    const float* part[ATT_WAVES + 1];
    part[0] = k > 0 ? lds[k - 1][1] : nullptr;
    bool goes_on = true;
#pragma unroll
    for (int w = 0; w < ATT_WAVES; ++w) {
      part[w + 1] = w >= k && goes_on ? lds[w][0] : nullptr;
      if (w >= k) goes_on = goes_on && more[w];
    }
    if (k > 0 && goes_on && tid == 0) joins[blockIdx.x] = AttJoin{head.row, head.n, head.unit, head.more};
    att_join<T, DIM, ATT_WAVES + 1, ATT_THREADS>(a, p, head.row, head.n, head.unit, head.from, head.to, part, k == 0 ? lds[0][0] : lds[k - 1][1],
                     k > 0 && !goes_on ? nullptr : att_slot(ws, blockIdx.x, k > 0, DIM));
  }
}

// Joins the parts of the unit that begins in block blockIdx.x of the split and ends in a later one, `cols` columns a block: four,
// a wave each, where there are many units and so, as a rule, few parts of each (where one has many after all, the block takes
// them one after the other); one, where few units have many parts (one row over a long context).  dim / 4 threads hold a part, the
// team as many parts as that leaves threads for and eight times that in flight, each its parts in the order of the keys, so that
// the result does not depend on which block was done first.  Latency: 5.0 us for 200 units of 2 to 3 parts, 8.1 us for 8 units of 64
// parts each; as an "all parts, then the last block joins" in the kernel before, it would need a counter to be cleared by a launch
// of its own and a release of every part to the other dies' caches.
constexpr int JOIN_FEW = 16;
template <typename T>
__global__ __launch_bounds__(ATT_THREADS) void paged_join_kernel(PagedAttArgs a, AttPlan p, float* ws, const AttJoin* joins, int cols) {
  constexpr int AHEAD = 8;
  __shared__ f32x4 acc[ATT_THREADS];
  __shared__ float wave_sum[ATT_WAVES];
  const AttJoin j = joins[blockIdx.x];
  const int parts = j.parts + 1, wave = threadIdx.x / WAVE;
  if (parts == 1) return;
  const int ROW = a.dim + 4, quads = a.dim / 4, hk = p.tiles == 1 ? j.unit : j.unit / p.tiles;
  const bool few = parts <= JOIN_FEW && cols == ATT_WAVES;
  const int team = few ? WAVE : ATT_THREADS, me = few ? threadIdx.x % WAVE : threadIdx.x;
  const int at_once = team / quads, mine = me / quads, quad = me - mine * quads;
  for (int i = 0; i < (few ? 1 : cols); ++i) {
    const int m = blockIdx.y * cols + (few ? wave : i);
    int row, head;
    const bool real = att_column(m, j.n, p.group, j.unit - hk * p.tiles, row, head);
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    float top = -INFINITY, base = 0.f, sum = 0.f;
    int from = 0, to = 0;
    if (real) {
      att_row_keys(a, j.row + row, from, to);
      auto part = [&](int k) { return att_slot(ws, blockIdx.x + k, k == 0, a.dim) + m * ROW; };
      f32x4 v[AHEAD];
      float v_top[AHEAD], v_sum[AHEAD];
      auto load = [&](int k0) {                            // what there is not is read from the last part, and has no weight
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          const float* from = part(min(k0 + u * at_once + mine, parts - 1));
          v[u] = *(const f32x4*)(from + 4 * quad);
          v_top[u] = from[a.dim];
          v_sum[u] = from[a.dim + 1];
        }
      };
      load(0);
      for (int k = me % WAVE; k < parts; k += WAVE) top = fmaxf(top, part(k)[a.dim]);
#pragma unroll
      for (int d = 1; d < WAVE; d <<= 1) top = fmaxf(top, __shfl_xor(top, d, WAVE));
      base = fabsf(top) == INFINITY ? 0.f : top;
      for (int k0 = 0; k0 < parts; k0 += AHEAD * at_once) {
        if (k0 > 0) load(k0);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          const int k = k0 + u * at_once + mine;
          const bool there = mine < at_once && k < parts;
          const float g = att_exp2(v_top[u] - base);
          sum += there && quad == 0 ? g * v_sum[u] : 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] += there ? g * v[u][e] : 0.f;
        }
      }
#pragma unroll
      for (int d = 1; d < WAVE; d <<= 1) sum += __shfl_xor(sum, d, WAVE);
    }
    if (threadIdx.x % WAVE == 0) wave_sum[wave] = sum;
    acc[threadIdx.x] = x;
    __syncthreads();
    if (real && mine == 0) {
      const f32x4* other = acc + (few ? wave * WAVE : 0) + quad;
      for (int k = 1; k < at_once; ++k) x += other[k * quads];
      if (!few) {
        sum = 0.f;
        for (int w = 0; w < ATT_WAVES; ++w) sum += wave_sum[w];
      }
      const bool none = from >= to || (sum == 0.f && !att_any_page(a, a.row_request[j.row], from, to));
      att_write<T>(a, p.wide_out, j.row + row, hk * p.group + head, 4 * quad, x, sum, none);
      if (a.lse && quad == 0) att_write_lse(a, j.row + row, hk * p.group + head, top, sum, none);
    }
    if (!few) __syncthreads();                             // before the LDS is written again
  }
}

// How a call's work is shared out: a wave a unit, a block a unit, or equal pieces of the line.  By the number of units and
// the steps of the longest one as far as the host knows; microseconds of the three on requests of 1/16 to all of that length
// (8 key-value heads of 128 in bf16: 8 units a row, 32 keys a step):
//   rows x steps     1 x 32         4 x 63         16 x 63        16 x 125         64 x 2          64 x 125        256 x 16       256 x 32
//   wave/block/split 44 / 14 / 16   86 / 24 / 21   87 / 25 / 31   178 / 51 / 40    8.7 / 11 / 18   192 / 125 / 126  71 / 79 / 83   125 / 117 / 128
// A block's waves take the longest unit's steps by eights at 0.14 us a KiB of a step (fp32: 0.19), whatever else there is to do; the
// pieces even that out for about 9 us more (their sums at the start, the join, its launch), and for more the more units there are.
// So the border lies at so many KiB of the longest unit as those are worth.  Block / split beside it, at KiB:
//   units             2 - 8                12 - 24           40 - 80           120 - 240
//   bf16 of 128       608: 17/16           608: 16/19        1000: 25/21       1000: 25/31
//   bf16 / fp16 of 64 500: 16/15           500: 16/17        750: 22/22        750: 24/30
//   fp16 of 256       500: 15/16           800: 21/20        1200: 29/34       3000: 91/92
//   fp32 of 96, 128   384: 15/15           384: 15/17        600: 21/17        1200: 43/42
//   fp32 of 32, 64    400: 15/14           600: 19/16        600: 21/20        750: 28/24 (32), 34/38 (64)
// Beyond 128 steps the pieces even out more than their start costs, but for steps of 4 KiB; block / split at units x steps:
//   bf16 of 128   240 x 128 50/54   240 x 200 102/95   512 x 128 115/115   512 x 160 137/130   512 x 250 229/195   1024 x 128 216/217   1024 x 250 393/389
//   fp16 of 64    256 x 128 30/37   256 x 200 46/53    256 x 300 81/78     512 x 128 57/56     512 x 200 102/94    1024 x 128 117/118   1024 x 200 173/163
//   bf16 of 32    56 x 128 16/18    56 x 160 19/20     128 x 160 21/24     128 x 200 25/26     512 x 160 32/42     512 x 200 41/48
// 512 units of one or two steps take a wave each, more steps a block: wave / block at 1, 2, 3, 4 steps
//   bf16 of 128, 512 units   9.8/11.4 10.6/11.2 12.2/12.2 13.3/12.0      1024 units   9.4/20 11.6/21 12.0/23 15/26
//   fp16 of 64, 512 units    7.3/6.3 8.0/7.1 8.3/6.8 9.5/7.3             1024 units   6.7/11 7.9/12 8.7/12 9.8/12
// (from 1024 units on a wave would be the faster one for up to 8 steps: 21 / 30 and 14 / 17 us there.)
// More units than the chip has SIMDs need no splitting while they are short (fp16, 8 heads of 64, rows x steps, wave / block / split):
//   256 x 19 37/38/48   512 x 19 77/79/95   512 x 47 177/149/170   2048 x 8 116/210/176   2048 x 19 257/293/295
// Rows of prompts (16 and more a request: more cannot be told here) stand in runs, and a block or wave for every row of a run but
// the first has nothing to do, which costs a block of eight waves its start all the same.  One prompt, bf16, 32 / 8 heads of 128:
//   256 rows 26/55/30   512 rows 63/119/52   2048 rows 647/909/412   4096 rows 2340/2940/1220
// `requests` is the table's size, the only number of requests that the host has: a prompt of 2048 rows with a table of 129 requests and
// more is not told from single rows, and takes 901 us for 409.
enum AttForm { ATT_WAVE, ATT_BLOCK, ATT_SPLIT };

AttPlan att_plan(int requests, int rows, int heads, int kv_heads, int dim, int dtype, long long max_keys, AttForm& form) {
  AttPlan p{};
  p.group = heads / kv_heads;
  p.run_shift = p.group <= 1 ? 4 : p.group <= 2 ? 3 : p.group <= 4 ? 2 : p.group <= 8 ? 1 : 0;
  p.tiles = (p.group + ATT_COLS - 1) / ATT_COLS;
  p.units = kv_heads * p.tiles;
  p.pieces = ATT_PIECES;
  if (max_keys <= 0 || max_keys > (1 << 30)) max_keys = 1 << 30;
  const int size = dtype == VITS_TYPE_F32 ? 4 : 2, step = att_step(size, dim);
  const long long units = (long long)rows * p.units, steps = (max_keys + step - 1) / step;
  const bool prompts = rows >= 16ll * requests;
  if (prompts ? steps <= 8 : steps <= (units >= 8192 ? 32 : units >= 2048 ? 20 : units >= 512 ? 2 : 0)) form = ATT_WAVE;
  else if (!prompts && steps <= 128 && steps * (step * dim * size / 512) <= (size == 4 ? 380 + 4 * units : 450 + 7 * units)) form = ATT_BLOCK;
  else form = ATT_SPLIT;
  if (units > 1 << 21) form = ATT_SPLIT;                   // more blocks than a grid of the other forms should have
  if (steps < (1 << 20)) {                                 // no more pieces than their least size fills
    const long long most = units * (steps + 1) / ATT_MIN_STEPS + 1;
    if (most < p.pieces) p.pieces = (int)(most + ATT_WAVES - 1) / ATT_WAVES * ATT_WAVES;
  }
  return p;
}

template <typename T, int DIM>
hipError_t start_attention(const PagedAttArgs& a, const AttPlan& p, AttForm form, void* ws, hipStream_t s) {
  const long long units = (long long)a.rows * p.units;      // below 2^22 where a grid is made of it
  if (form == ATT_WAVE) {
    hipLaunchKernelGGL((paged_attention_wave_kernel<T, DIM>), dim3((unsigned)((units + ATT_WAVES - 1) / ATT_WAVES)), dim3(ATT_THREADS), 0, s, a, p);
  } else if (form == ATT_BLOCK) {
    hipLaunchKernelGGL((paged_attention_block_kernel<T, DIM>), dim3((unsigned)units), dim3(ATT_BLOCK_WAVES * WAVE), 0, s, a, p);
  } else {
    const int blocks = p.pieces / ATT_WAVES;
    AttJoin* joins = (AttJoin*)att_slot((float*)ws, blocks, 0, DIM);
    hipLaunchKernelGGL((paged_attention_split_kernel<T, DIM>), dim3(blocks), dim3(ATT_THREADS), 0, s, a, p, (float*)ws, joins);
    const int cols = min(ATT_COLS, p.group * min(1 << p.run_shift, a.rows)), each = units > ATT_FEW ? ATT_WAVES : 1;
    hipLaunchKernelGGL((paged_join_kernel<T>), dim3(blocks, (cols + each - 1) / each), dim3(ATT_THREADS), 0, s, a, p, (float*)ws, joins, each);
  }
  return hipGetLastError();
}

template <typename T>
hipError_t start_attention_t(const PagedAttArgs& a, const AttPlan& p, AttForm form, void* ws, hipStream_t s) {
  switch (a.dim) {
    case 32: return start_attention<T, 32>(a, p, form, ws, s);
    case 64: return start_attention<T, 64>(a, p, form, ws, s);
    case 96: return start_attention<T, 96>(a, p, form, ws, s);
    case 128: return start_attention<T, 128>(a, p, form, ws, s);
    case 160: return start_attention<T, 160>(a, p, form, ws, s);
    case 192: return start_attention<T, 192>(a, p, form, ws, s);
    case 224: return start_attention<T, 224>(a, p, form, ws, s);
    case 256: return start_attention<T, 256>(a, p, form, ws, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_page_plan(const PagePlanArgs& a, hipStream_t s) {
  const int tiles = (a.rows + PLAN_ROWS - 1) / PLAN_ROWS, shares = (a.requests + PLAN_SHARE - 1) / PLAN_SHARE;
  hipLaunchKernelGGL(page_plan_kernel, dim3(tiles > shares ? tiles : shares), dim3(PLAN_THREADS), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_rotary_store(const RotaryArgs& a, hipStream_t s) {
  if (a.dtype == VITS_TYPE_F32) return start_rotary_t<float>(a, s);
  return a.dtype == VITS_TYPE_F16 ? start_rotary_t<_Float16>(a, s) : start_rotary_t<__bf16>(a, s);
}

int64_t paged_attention_workspace(int requests, int rows, int heads, int kv_heads, int dim, int dtype, long long max_keys) {
  AttForm form;
  const AttPlan p = att_plan(requests, rows, heads, kv_heads, dim, dtype, max_keys, form);
  return form == ATT_SPLIT ? (int64_t)(p.pieces / ATT_WAVES) * (2 * ATT_COLS * (dim + 4) * sizeof(float) + sizeof(AttJoin)) : 0;
}

hipError_t launch_paged_attention(const PagedAttArgs& a, long long max_keys, void* ws, hipStream_t s) {
  AttForm form;
  AttPlan p = att_plan(a.requests, a.rows, a.heads, a.kv_heads, a.dim, a.dtype, max_keys, form);
  const int size = a.dtype == VITS_TYPE_F32 ? 4 : 2;
  p.per_page = a.page_size / 16;
  p.wide_out = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.out_row * size % 16 == 0 && a.out_head * size % 16 == 0;
  if (a.dtype == VITS_TYPE_F32) return start_attention_t<float>(a, p, form, ws, s);
  return a.dtype == VITS_TYPE_F16 ? start_attention_t<_Float16>(a, p, form, ws, s) : start_attention_t<__bf16>(a, p, form, ws, s);
}

}  // namespace vits
