// Operators around a paged key-value cache (gfx950 / CDNA4 only): the step's plan, rotary rows stored to the cache, and
// attention of single rows over it.  The cache holds pages of page_size tokens, [pages][kv_heads][page_size][dim], so a
// head's tokens of one page are one contiguous run.
#include "paged.h"
#include "../../include/vits_amd.h"

namespace vits {
namespace {

constexpr int WAVE = 64;

// ---------------------------------------------------------------------------------------------------------
// page plan.  With a = max(grow, 0), held = ceil(length / page), fresh = ceil((length + a) / page) - held and back =
// held of a request that ends, three prefix sums over the requests say which rows, which free pages and which ring
// places are whose.  Every block takes those sums over all requests itself (two passes over 8 bytes a request, from
// L2) and then serves its own tile of rows and its own share of the requests: one launch, no second pass over memory,
// and every block comes to the same verdict on whether the step fits before anything is written.
// A fresh page p of a request begins at position p * page >= length, so the row at that position is the one that
// writes the table entry.  Pages are taken at the ring's head and returned at its tail; head .. tail never holds more
// pages than the ring, so no place is read by one block and written by another.
// ---------------------------------------------------------------------------------------------------------
constexpr int PLAN_THREADS = 256;
constexpr int PLAN_ROWS = 1024;              // rows of a block: four consecutive ones a thread, 16-byte stores

struct PlanSums {
  long long rows, fresh, back;
};

__device__ __forceinline__ long long shfl_up64(long long v, int d) { return __shfl_up(v, d, WAVE); }

__device__ __forceinline__ PlanSums plan_of(int len, int grow, unsigned page) {
  PlanSums p;
  const unsigned l = len < 0 ? 0u : (unsigned)len, a = grow < 0 ? 0u : (unsigned)grow;
  const long long held = l / page + (l % page != 0);
  const unsigned after = l + a;              // below 2^32
  p.rows = a;
  p.fresh = (long long)(after / page + (after % page != 0)) - held;
  p.back = grow < 0 ? held : 0;
  return p;
}

__global__ __launch_bounds__(PLAN_THREADS) void page_plan_kernel(PagePlanArgs a) {
  __shared__ PlanSums wave_sum[PLAN_THREADS / WAVE];
  __shared__ int wave_bad[PLAN_THREADS / WAVE], wave_mark[PLAN_THREADS / WAVE];
  __shared__ int mark[PLAN_ROWS], m_base[PLAN_ROWS], m_held[PLAN_ROWS], m_fresh[PLAN_ROWS];
  __shared__ int gone[PLAN_THREADS], gone_held[PLAN_THREADS], gone_at[PLAN_THREADS], n_gone;
  const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
  const unsigned page = (unsigned)a.page_size;
  const int each = (a.requests + PLAN_THREADS - 1) / PLAN_THREADS;
  const int s0 = min(tid * each, a.requests), s1 = min(s0 + each, a.requests);

  // pass 1: this thread's requests
  PlanSums mine = {0, 0, 0};
  int bad = 0;
  for (int s = s0; s < s1; ++s) {
    const int len = a.lengths[s], g = a.grow[s];
    if (len < 0 || g < -1 || (g > 0 && len > 0x7fffffff - g)) { bad |= VITS_PLAN_BAD_LENGTH; continue; }
    const PlanSums p = plan_of(len, g, page);
    if (((long long)len + (g > 0 ? g : 0) + page - 1) / page > a.width) bad |= VITS_PLAN_TABLE_FULL;
    mine.rows += p.rows; mine.fresh += p.fresh; mine.back += p.back;
  }
  PlanSums upto = mine;                      // inclusive over the wave
#pragma unroll
  for (int d = 1; d < WAVE; d <<= 1) {
    const long long r = shfl_up64(upto.rows, d), f = shfl_up64(upto.fresh, d), b = shfl_up64(upto.back, d);
    if (lane >= d) { upto.rows += r; upto.fresh += f; upto.back += b; }
    bad |= __shfl_xor(bad, d, WAVE);
  }
  if (lane == WAVE - 1) { wave_sum[wave] = upto; wave_bad[wave] = bad; }
  for (int i = tid; i < PLAN_ROWS; i += PLAN_THREADS) mark[i] = -1;
  if (tid == 0) n_gone = 0;
  __syncthreads();
  PlanSums total = {0, 0, 0}, before = {upto.rows - mine.rows, upto.fresh - mine.fresh, upto.back - mine.back};
  bad = 0;
#pragma unroll
  for (int w = 0; w < PLAN_THREADS / WAVE; ++w) {
    if (w < wave) { before.rows += wave_sum[w].rows; before.fresh += wave_sum[w].fresh; before.back += wave_sum[w].back; }
    total.rows += wave_sum[w].rows; total.fresh += wave_sum[w].fresh; total.back += wave_sum[w].back;
    bad |= wave_bad[w];
  }
  const long long head = a.cursor[0], tail = a.cursor[1], free_pages = tail - head;
  if (head < 0 || free_pages < 0 || free_pages > a.pages || free_pages + total.back > a.pages) bad |= VITS_PLAN_BAD_RING;
  if (total.rows > a.rows) bad |= VITS_PLAN_ROWS_FULL;
  if (total.fresh > free_pages) bad |= VITS_PLAN_NO_PAGES;
  const int ring0 = bad ? 0 : (int)(head % a.pages), ring1 = bad ? 0 : (int)(tail % a.pages);

  // pass 2: mark where requests begin in this block's rows; write what belongs to this block's share of the requests
  const int row0 = blockIdx.x * PLAN_ROWS;
  const int own0 = blockIdx.x * PLAN_THREADS, own1 = own0 + PLAN_THREADS;
  for (int s = s0; s < s1; ++s) {
    const int len = a.lengths[s], g = a.grow[s];
    const bool own = s >= own0 && s < own1;
    if (bad) {
      if (own) { a.lengths_out[s] = len; a.row_start[s] = 0; }
      continue;
    }
    const PlanSums p = plan_of(len, g, page);
    if (own) {
      a.lengths_out[s] = g < 0 ? 0 : len + g;
      a.row_start[s] = (int)before.rows;
      if (p.back > 0) {
        const int n = atomicAdd(&n_gone, 1);           // the order in this list does not reach the results
        gone[n] = s; gone_held[n] = (int)p.back; gone_at[n] = (int)before.back;
      }
    }
    if (p.rows > 0 && before.rows < (long long)row0 + PLAN_ROWS && before.rows + p.rows > row0) {
      const int at = before.rows > row0 ? (int)(before.rows - row0) : 0;
      mark[at] = s;
      m_base[at] = len - (int)before.rows;
      m_held[at] = (int)(len / page + (len % page != 0));
      m_fresh[at] = (int)before.fresh;
    }
    before.rows += p.rows; before.fresh += p.fresh; before.back += p.back;
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
// rotary rows, stored to the cache
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
__device__ __forceinline__ void rotary_angle(int position, double freq, float scale, float& c, float& s) {
  const double turns = (double)position * freq * 0.15915494309189533577;      // 1 / (2 pi)
  const double whole = rint(turns);
  const double part = turns - whole;                     // -1/2 .. 1/2
  const double quarter = rint(part * 4.0);
  float s0, c0;
  sincospif((float)((part - quarter * 0.25) * 2.0), &s0, &c0);
  const int k = (int)quarter & 3;
  c = scale * (k == 0 ? c0 : k == 1 ? -s0 : k == 2 ? -c0 : s0);
  s = scale * (k == 0 ? s0 : k == 1 ? c0 : k == 2 ? -s0 : -c0);
}

// written as products and sums of its own choice, so that every variant below gives the same bits
__device__ __forceinline__ void rotary_turn(float& u, float& w, float c, float s) {
  const float x = fmaf(u, c, -(w * s)), y = fmaf(w, c, u * s);
  u = x;
  w = y;
}

constexpr int ROT_THREADS = 256;

// N channels an item: 16 bytes where sizes and addresses allow, else one.  An item that turns holds N channels of either
// half in the half layout, N channels = N / 2 pairs in the interleaved one (and one pair where N is 1).
template <typename T, int N, bool INTER>
__global__ __launch_bounds__(ROT_THREADS) void rotary_store_kernel(RotaryArgs a, int rows_per_block) {
  extern __shared__ float cs[];                          // [rows_per_block][pairs][2]
  const int tid = threadIdx.x;
  const int row0 = blockIdx.x * rows_per_block, rows = min(rows_per_block, a.rows - row0);
  for (int i = tid; i < rows * a.pairs; i += ROT_THREADS) {
    const int r = i / a.pairs, p = i % a.pairs;
    rotary_angle(a.position[row0 + r], a.freq[p], a.scale, cs[2 * i], cs[2 * i + 1]);
  }
  __syncthreads();
  const int turn = INTER && N > 1 ? 2 * a.pairs / N : a.pairs / N;   // items of a head that turn
  const int pass = (a.dim - 2 * a.pairs) / N, whole = a.dim / N;     // ... that pass through; of a value head
  const int per_head = turn + pass;
  const int n_q = a.heads * per_head, n_k = a.kv_heads * per_head, n_v = a.kv_heads * whole;
  const int per_row = n_q + n_k + n_v;
  const int64_t slots = (int64_t)a.pages * a.page_size;
  using P = Pack<T, N>;
  for (int i = tid; i < rows * per_row; i += ROT_THREADS) {
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
    if (j >= n_q + n_k) {
      j -= n_q + n_k;
      const int h = j / whole, c = (j - h * whole) * N;
      const T* src = (const T*)a.v + row * a.v_row + h * a.v_head + c;
      *(P*)((T*)a.v_cache + cell + (int64_t)h * a.page_size * a.dim + c) = *(const P*)src;
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
    if (j >= turn) {
      const int c = 2 * a.pairs + (j - turn) * N;
      *(P*)(dst + c) = *(const P*)(src + c);
      continue;
    }
    const float* ang = cs + (size_t)r * a.pairs * 2;
    if constexpr (INTER && N == 1) {
      float u = Conv<T>::to(src[2 * j]), w = Conv<T>::to(src[2 * j + 1]);
      rotary_turn(u, w, ang[2 * j], ang[2 * j + 1]);
      dst[2 * j] = Conv<T>::from(u);
      dst[2 * j + 1] = Conv<T>::from(w);
    } else if constexpr (INTER) {
      P x = *(const P*)(src + j * N);
#pragma unroll
      for (int e = 0; e < N / 2; ++e) {
        float u = Conv<T>::to(x.v[2 * e]), w = Conv<T>::to(x.v[2 * e + 1]);
        rotary_turn(u, w, ang[j * N + 2 * e], ang[j * N + 2 * e + 1]);
        x.v[2 * e] = Conv<T>::from(u);
        x.v[2 * e + 1] = Conv<T>::from(w);
      }
      *(P*)(dst + j * N) = x;
    } else {
      P x = *(const P*)(src + j * N), y = *(const P*)(src + a.pairs + j * N);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        float u = Conv<T>::to(x.v[e]), w = Conv<T>::to(y.v[e]);
        rotary_turn(u, w, ang[2 * (j * N + e)], ang[2 * (j * N + e) + 1]);
        x.v[e] = Conv<T>::from(u);
        y.v[e] = Conv<T>::from(w);
      }
      *(P*)(dst + j * N) = x;
      *(P*)(dst + a.pairs + j * N) = y;
    }
  }
}

template <typename T, int N, bool INTER>
hipError_t start_rotary(const RotaryArgs& a, hipStream_t s) {
  const int per_row = (a.heads + (a.k ? 2 * a.kv_heads : 0)) * (a.dim / N);
  int rpb = per_row >= 1024 ? 1 : (1024 + per_row - 1) / per_row;    // about four items a thread
  rpb = min(rpb, min(16, a.rows));
  while (rpb > 1 && (a.rows + rpb - 1) / rpb < 256) rpb = (rpb + 1) / 2;   // few rows: spread them over the CUs
  const size_t lds = (size_t)rpb * a.pairs * 2 * sizeof(float);      // at most 16 KiB
  hipLaunchKernelGGL((rotary_store_kernel<T, N, INTER>), dim3((a.rows + rpb - 1) / rpb), dim3(ROT_THREADS), lds, s, a, rpb);
  return hipGetLastError();
}

template <typename T>
hipError_t start_rotary_t(RotaryArgs a, hipStream_t s) {
  constexpr int N = 16 / sizeof(T);
  if (!a.k) a.kv_heads = 0;
  if (!a.q) a.heads = 0;
  // sixteen-byte items need halves (or pairs) and rests in whole items, and every row and head on a 16-byte address
  bool wide = a.dim % N == 0 && (a.interleaved ? 2 * a.pairs : a.pairs) % N == 0;
  auto on16 = [&](const void* p, long long row, long long head) {
    wide = wide && reinterpret_cast<uintptr_t>(p) % 16 == 0 && row % N == 0 && head % N == 0;
  };
  if (a.q) { on16(a.q, a.q_row, a.q_head); on16(a.out, a.out_row, a.out_head); }
  if (a.k) {
    on16(a.k, a.k_row, a.k_head); on16(a.v, a.v_row, a.v_head);
    on16(a.k_cache, a.page_stride, 0); on16(a.v_cache, a.page_stride, 0);
  }
  if (a.interleaved) return wide ? start_rotary<T, N, true>(a, s) : start_rotary<T, 1, true>(a, s);
  return wide ? start_rotary<T, N, false>(a, s) : start_rotary<T, 1, false>(a, s);
}

// ---------------------------------------------------------------------------------------------------------
// attention of single rows over the cache
// ---------------------------------------------------------------------------------------------------------
constexpr int ATT_WAVES = 4;

// One block per row and query head; the waves take keys in turn, lanes hold channels lane, lane + 64, ...
template <typename T>
__global__ __launch_bounds__(ATT_WAVES * WAVE) void paged_attention_kernel(PagedAttArgs a) {
  __shared__ float part[ATT_WAVES][PAGED_MAX_DIM + 2];
  const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int req = a.row_request[row];
  if (req < 0) return;
  if (req >= a.requests) {
    if (a.err_flag && threadIdx.x == 0) atomicOr(a.err_flag, 1);
    return;
  }
  long long end = (long long)a.row_position[row] + 1;
  const long long cap = (long long)a.width * a.page_size;
  if (end > cap) {
    end = cap;
    if (a.err_flag && threadIdx.x == 0) atomicOr(a.err_flag, 1);
  }
  const long long begin = a.window > 0 && end > a.window ? end - a.window : 0;
  const int hk = h / (a.heads / a.kv_heads);
  const T* q = (const T*)a.q + row * a.q_row + h * a.q_head;
  float qv[4], o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) qv[i] = lane + 64 * i < a.dim ? Conv<T>::to(q[lane + 64 * i]) * a.scale : 0.f;
  for (long long t = begin + wave; t < end; t += ATT_WAVES) {
    const int id = a.table[req * a.table_stride + t / a.page_size];
    if (id < 0 || id >= a.pages) {
      if (a.err_flag && lane == 0) atomicOr(a.err_flag, 1);
      continue;
    }
    const long long cell = id * a.page_stride + ((long long)hk * a.page_size + t % a.page_size) * a.dim;
    float d = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 64 * i < a.dim) d += qv[i] * Conv<T>::to(((const T*)a.k_cache)[cell + lane + 64 * i]);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) d += __shfl_xor(d, x, 64);
    const float top = fmaxf(m, d), base = top == -INFINITY ? 0.f : top;
    const float keep = __expf(m - base), p = __expf(d - base);
    l = l * keep + p;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 64 * i < a.dim) o[i] = o[i] * keep + p * Conv<T>::to(((const T*)a.v_cache)[cell + lane + 64 * i]);
    m = top;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) part[wave][lane + 64 * i] = o[i];
  if (lane == 0) { part[wave][PAGED_MAX_DIM] = m; part[wave][PAGED_MAX_DIM + 1] = l; }
  __syncthreads();
  float top = -INFINITY, sum = 0, w[ATT_WAVES];
  for (int i = 0; i < ATT_WAVES; ++i) top = fmaxf(top, part[i][PAGED_MAX_DIM]);
  const float base = top == -INFINITY ? 0.f : top;
  for (int i = 0; i < ATT_WAVES; ++i) {
    w[i] = __expf(part[i][PAGED_MAX_DIM] - base);
    sum += w[i] * part[i][PAGED_MAX_DIM + 1];
  }
  const bool none = end <= 0;
  for (int c = threadIdx.x; c < a.dim; c += ATT_WAVES * WAVE) {
    float v = 0;
    for (int i = 0; i < ATT_WAVES; ++i) v += w[i] * part[i][c];
    ((T*)a.out)[row * a.out_row + h * a.out_head + c] = Conv<T>::from(none ? 0.f : v / sum);
  }
  if (a.lse && threadIdx.x == 0) a.lse[(long long)row * a.heads + h] = none ? -INFINITY : base + logf(sum);
}

}  // namespace

hipError_t launch_page_plan(const PagePlanArgs& a, hipStream_t s) {
  const int tiles = (a.rows + PLAN_ROWS - 1) / PLAN_ROWS, shares = (a.requests + PLAN_THREADS - 1) / PLAN_THREADS;
  hipLaunchKernelGGL(page_plan_kernel, dim3(tiles > shares ? tiles : shares), dim3(PLAN_THREADS), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_rotary_store(const RotaryArgs& a, hipStream_t s) {
  if (a.dtype == VITS_TYPE_F32) return start_rotary_t<float>(a, s);
  return a.dtype == VITS_TYPE_F16 ? start_rotary_t<_Float16>(a, s) : start_rotary_t<__bf16>(a, s);
}

int64_t paged_attention_workspace(int, int, int, int, long long) { return 0; }

hipError_t launch_paged_attention(const PagedAttArgs& a, long long, void*, hipStream_t s) {
  const dim3 grid(a.rows, a.heads), block(ATT_WAVES * WAVE);
  if (a.dtype == VITS_TYPE_F32) hipLaunchKernelGGL(paged_attention_kernel<float>, grid, block, 0, s, a);
  else if (a.dtype == VITS_TYPE_F16) hipLaunchKernelGGL(paged_attention_kernel<_Float16>, grid, block, 0, s, a);
  else hipLaunchKernelGGL(paged_attention_kernel<__bf16>, grid, block, 0, s, a);
  return hipGetLastError();
}

}  // namespace vits
