// Pages of a cache handed to requests and taken back, from the lengths that the requests want (dlt_page_assign), for gfx950.
//
// With P(x) = ceil(x / page) request b needs max(P(want) - P(held), 0) pages or gives back max(P(held) - P(want), 0).  Exclusive sums of both over the requests, in
// order, say everything else: page k of all that are needed is entry F + R - 1 - k of the stack "F free pages, then the R that come back, last request's last
// page first", and request b is served iff its sum of needs, itself included, is at most F + R.  So every page and every slot is found by itself, from two sums, and
// nothing is added atomically: equal calls give equal pages.
//
// Every workgroup forms the two sums of all requests (8 B of lengths each, from the L2) and keeps them in LDS with what every request holds and gains, then takes a share of
// the new columns, of the pages that come back and of the slots.  A table's row is read (a request that gives back) or written (one that gains), never both; the pool is read
// below F and written from F on.  Lengths and the pool's count, which all workgroups read before all else, are written by the last one to have read them: a count in the
// pool's second word tells which that is; nobody waits.
//
// Bound by latency: 64 requests, a token more and back, 4.9 + 4.4 us on the GPU (lengths, sums, pages, rows); 1000 requests, 4000 slots each,
// 16 MB of slots written, and back, 13.6 + 7.9: about 3.4 for the slots, 2.6 for counts that meet in one word (10 ns each), the rest a chain in every workgroup that more of them do
// not shorten: launch, sums of 1000 requests, then columns, pages that come back and slots one after the other.
#include <algorithm>
#include "dlt_internal.hpp"
#include "kernargs.h"

namespace {

struct AssignArgs {
  int32_t *table, *seq, *pool, *n_new, *slots;
  const int32_t* want;
  int64_t ts;
  int32_t B, cols, page, n_pages, T;
  uint32_t mp, sp, mt, st;   // divisions by page and T
};

struct Wish { int held, want, need, back; };
// what a request of `seq` tokens that wants `want` holds and needs or gives back, in pages
__device__ inline Wish wish_of(const AssignArgs& a, int seq, int want) {
  Wish w;
  const int room = a.cols * a.page;   // < 2^31
  w.held = dlt_imax(0, dlt_imin(seq, room));
  w.want = want;
  w.need = w.back = 0;
  if (w.want < 0) w.want = w.held;
  if (w.want > room || (a.T >= 0 && w.want - w.held > a.T)) w.want = w.held;
  const int p0 = (int)dlt_fastdiv((uint32_t)(w.held + a.page - 1), a.mp, a.sp), p1 = (int)dlt_fastdiv((uint32_t)(w.want + a.page - 1), a.mp, a.sp);
  w.need = dlt_imax(p1 - p0, 0);
  w.back = dlt_imax(p0 - p1, 0);
  return w;
}
__device__ inline int pages_of(const AssignArgs& a, int tokens) { return (int)dlt_fastdiv((uint32_t)(tokens + a.page - 1), a.mp, a.sp); }

// the last b with start[b] <= x; start[0] = 0, start[B] > x
__device__ inline int owner_of(const int32_t* start, int B, int x) {
  int lo = 0, hi = B;   // start[lo] <= x < start[hi]
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (start[m] <= x) lo = m;
    else hi = m;
  }
  return lo;
}

struct Stack {
  const AssignArgs& a;
  const int32_t *back, *held, *gain;   // exclusive sums of what comes back, [B + 1]; of every request
  int F, R;
  // r-th of the pages that come back: the last request's last page first
  __device__ int returned(int r) const {
    const int x = R - 1 - r, b = owner_of(back, a.B, x);
    return a.table[b * a.ts + (pages_of(a, held[b] + gain[b]) + x - back[b])];
  }
  // k-th page that is taken
  __device__ int taken(int k) const {
    const int at = F + R - 1 - k;
    return at < F ? a.pool[2 + at] : returned(at - F);
  }
};

// inclusive sums of two numbers over the workgroup's threads, and their totals
template <int NT>
__device__ inline void scan2(int& x, int& y, int& sum_x, int& sum_y, int (*wave)[2]) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int ux = __shfl_up(x, d), uy = __shfl_up(y, d);
    if (lane >= d) { x += ux; y += uy; }
  }
  if (lane == 63) { wave[w][0] = x; wave[w][1] = y; }
  __syncthreads();
  sum_x = sum_y = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; i++) {
    if (i == w) { x += sum_x; y += sum_y; }
    sum_x += wave[i][0];
    sum_y += wave[i][1];
  }
}

template <int NT>
__global__ __launch_bounds__(NT) void page_assign_kernel(AssignArgs a) {
  dlt_kernargs_in<sizeof(AssignArgs)>();
  extern __shared__ int32_t sums[];   // needs [B + 1], back [B + 1], held [B], gains [B]: tokens gained, or given back where negative
  __shared__ int wave[NT / 64][2], most[NT / 64], last;
  int32_t *need = sums, *back = need + a.B + 1, *held = back + a.B + 1, *gain = held + a.B;
  const int tid = threadIdx.x;

  // sums of needs and of what comes back: a run of requests to a thread
  const int per = (a.B + NT - 1) / NT, b0 = dlt_imin(tid * per, a.B), b1 = dlt_imin(b0 + per, a.B);
  int n = 0, r = 0, sum_n, sum_r;
  constexpr int PER = DLT_ASSIGN_MAX / NT;
  int seq[PER], want[PER];
  Wish w{};
  if (per == 1) {
    if (b0 < b1) w = wish_of(a, a.seq[b0], a.want[b0]);
    n = w.need;
    r = w.back;
  } else {   // their lengths together, not one after the other (8000 requests, a token more and back: 46 -> 38 us)
#pragma unroll
    for (int k = 0; k < PER; k++) {
      seq[k] = want[k] = 0;
      if (k < per) {
        const int b = dlt_imin(b0 + k, a.B - 1);
        seq[k] = a.seq[b];
        want[k] = a.want[b];
      }
    }
#pragma unroll
    for (int k = 0; k < PER; k++)
      if (b0 + k < b1) {
        w = wish_of(a, seq[k], want[k]);
        n += w.need;
        r += w.back;
      }
  }
  const int own_n = n, own_r = r;
  const int F = dlt_imax(0, dlt_imin(a.pool[0], a.n_pages));
  scan2<NT>(n, r, sum_n, sum_r, wave);
  n -= own_n;
  r -= own_r;
  const int64_t room = (int64_t)F + sum_r;
  int served = 0;   // pages taken
  auto keep = [&](int b) __attribute__((always_inline)) {
    need[b] = n;
    back[b] = r;
    n += w.need;
    r += w.back;
    held[b] = w.held;
    gain[b] = w.need > 0 && n > room ? 0 : w.want - w.held;
    if (w.need > 0 && n <= room) served = n;
  };
  if (per == 1) {
    if (b0 < b1) keep(b0);
  } else {
#pragma unroll
    for (int k = 0; k < PER; k++)
      if (b0 + k < b1) {
        w = wish_of(a, seq[k], want[k]);
        keep(b0 + k);
      }
  }
  if (tid == 0) {
    need[a.B] = sum_n;
    back[a.B] = sum_r;
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) served = dlt_imax(served, __shfl_xor(served, d));
  if ((tid & 63) == 0) most[tid >> 6] = served;
  asm volatile("" ::"v"(F));   // waves without a request need it only behind the count: a barrier waits for no load from memory
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NT / 64; i++) served = dlt_imax(served, most[i]);
  // Every load of lengths and of the pool's count by this workgroup has returned: as far as it is concerned they may be written.  Counted here, beside the work, and looked at behind
  // it (4000 requests, a token more and back, 22.4 -> 21.2 us); by many workgroups, which would queue up here (10 ns each), behind it too (1000 requests, 4000 slots 21.9 -> 21.0).
  // Nothing that one workgroup writes is read by another, so the addition needs no release and acquire, which would write caches back and empty them (1000 requests, 4000 slots and back
  // 20.0 -> 27.1; 4000 requests, a token more and back, 21.7 -> 22.6): what has to come before it are loads, and those are waited for.
  const bool early = gridDim.x <= 64;
  int before = 0;
  auto count = [&]() __attribute__((always_inline)) {
    if (tid == 0) before = __hip_atomic_fetch_add(&a.pool[1], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  if (gridDim.x > 1 && early) count();
  const int left = (int)(room - served < a.n_pages ? room - served : a.n_pages);
  const Stack stack{a, back, held, gain, F, sum_r};
  // Every kind of work begins with waves of its own: on a small call, one workgroup, none waits for another kind's memory (64 requests, a token more: 6.0 us by eight
  // workgroups, 5.2 by this one)
  const int64_t wg0 = (int64_t)blockIdx.x * NT, step = (int64_t)gridDim.x * NT;

  for (int64_t k = wg0 + tid; k < served; k += step) {
    const int b = owner_of(need, a.B, (int)k);
    a.table[b * a.ts + (pages_of(a, held[b]) + (int)k - need[b])] = stack.taken((int)k);
  }
  for (int64_t i = wg0 + (tid ^ NT / 4); F + i < left; i += step) a.pool[2 + F + i] = stack.returned((int)i);
  for (int64_t b = wg0 + (tid ^ NT / 8); b < a.B; b += step) a.n_new[b] = dlt_imax(gain[b], 0);
  // slots, four in a row of all to a thread: they share their request and mostly their page
  const int64_t slots = a.T > 0 ? (int64_t)a.B * a.T : 0;
  // (from the last workgroup on: on a small call others have the columns)
  for (int64_t i = 4 * ((int64_t)(gridDim.x - 1 - blockIdx.x) * NT + (tid ^ NT / 2)); i < slots; i += 4 * step) {
    int b = (int)dlt_fastdiv((uint32_t)i, a.mt, a.st), t = (int)i - b * a.T, page = -1, until = 0;   // `page` holds tokens below `until` of request b
    int has = held[b], more = gain[b], out[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      if (t == a.T) {
        t = until = 0;
        if (++b == a.B) break;
        has = held[b];
        more = gain[b];
      }
      const int p = has + t;
      out[k] = -1;
      if (t < more) {
        if (p >= until) {
          const int col = (int)dlt_fastdiv((uint32_t)p, a.mp, a.sp), p0 = pages_of(a, has);
          page = col < p0 ? a.table[b * a.ts + col] : stack.taken(need[b] + col - p0);
          until = (col + 1) * a.page;
        }
        out[k] = (page + 1) * a.page - (until - p);
      }
      t++;
    }
    if (i + 4 <= slots) *reinterpret_cast<int4*>(a.slots + i) = int4{out[0], out[1], out[2], out[3]};
    else
      for (int k = 0; i + k < slots; k++) a.slots[i + k] = out[k];
  }

  // the last workgroup to be counted writes them.  (Nothing else that a workgroup writes is read by another.)
  if (gridDim.x > 1) {
    if (!early) count();
    if (tid == 0) last = before == (int)gridDim.x - 1;
    __syncthreads();
    if (!last) return;
  }
  for (int b = tid; b < a.B; b += NT)
    if (gain[b] != 0) a.seq[b] = held[b] + gain[b];
  if (tid == 0) {
    a.pool[0] = left;
    if (gridDim.x > 1) a.pool[1] = 0;
  }
}

}  // namespace

extern "C" int dlt_page_assign(int32_t* table, int64_t table_stride, int32_t* seq_len, const int32_t* want, int32_t* pool, int32_t B, int32_t cols, int32_t page,
                               int32_t n_pages, int32_t T, int32_t* n_new, int32_t* slots, void* stream_) {
  const char* who = "page_assign";
  hipStream_t stream = (hipStream_t)stream_;
  DLT_REQUIRE(B >= 0 && cols > 0 && page > 0 && n_pages > 0 && T >= -1, "%s: B=%d cols=%d page=%d n_pages=%d T=%d", who, B, cols, page, n_pages, T);
  if (B > DLT_ASSIGN_MAX) return dlt_set_error(DLT_ERR_UNSUPPORTED, "%s: %d requests, at most %d are supported", who, B, DLT_ASSIGN_MAX);
  if ((int64_t)B * cols > 0x3fffffff || (int64_t)cols * page > 0x3fffffff || n_pages > 0x3fffffff || (int64_t)n_pages * page > 0x7fffffff || (int64_t)B * T > 0x7fffffff)
    return dlt_set_error(DLT_ERR_UNSUPPORTED, "%s: too many pages or tokens", who);
  if (B == 0) return DLT_OK;
  DLT_REQUIRE(table != nullptr && seq_len != nullptr && want != nullptr && pool != nullptr && n_new != nullptr && (slots != nullptr || T <= 0), "%s: a tensor is NULL", who);
  DLT_REQUIRE((uintptr_t)slots % 16 == 0, "%s: slots must start at a multiple of 16 bytes", who);
  DLT_REQUIRE(B == 1 || table_stride >= cols, "%s: rows of the table overlap (stride %lld, %d columns)", who, (long long)table_stride, cols);
  AssignArgs a{};
  a.table = table; a.seq = seq_len; a.pool = pool; a.n_new = n_new; a.slots = slots; a.want = want; a.ts = table_stride;
  a.B = B; a.cols = cols; a.page = page; a.n_pages = n_pages; a.T = T;
  dlt_fastdiv_make((uint32_t)page, a.mp, a.sp);
  dlt_fastdiv_make((uint32_t)dlt_imax(T, 1), a.mt, a.st);
  constexpr int NT = 1024;
  // 256 requests, as many threads of slots by fours, or 4096 columns that requests can gain (give back, without a limit to the slots) to a workgroup, up to a workgroup a CU.  Each is
  // another addition to the pool's word, so they are large.  us, 1000 requests, 4000 slots each, by 32 / 64 / 128 / 256 workgroups 37.3 / 23.6 / 16.9 / 14.0, and back, a million
  // columns that may be given, 7.9 / 7.7 / 8.1 / 9.7.
  const int64_t slots4 = (int64_t)B * dlt_imax(T, 0) / 4, columns = (int64_t)B * (T >= 0 ? dlt_imin(T / page + 2, cols) : cols), cus = dlt_device_cus();
  const int64_t grid = std::max<int64_t>(1, std::min<int64_t>((B + slots4) / 256 + columns / 4096, cus));
  const int lds = 4 * (B + 1) * 4;
  const int rc = dlt_ensure_lds(reinterpret_cast<const void*>(page_assign_kernel<NT>), lds);
  if (rc != DLT_OK) return rc;
  dlt_timing_before(DLT_K_PAGES, stream);
  hipLaunchKernelGGL(page_assign_kernel<NT>, dim3((unsigned)grid), dim3(NT), lds, stream, a);
  dlt_timing_after(stream);
  DLT_CHECK_LAUNCH("page_assign launch");
  return DLT_OK;
}
