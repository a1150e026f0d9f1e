// Tables, positions and slots of the tokens that rows get next, made on the device.
//
// Row r has n tokens and gets c more.  With  need = ceil((n + c) / ps) - ceil(n / ps)  and exclusive sums over the rows
//   page j of its new ones is  free[taken + sum need + j],  and token i of them stands at position n + i, in place (n + i) % ps of
//   page (n + i) / ps of its table, and at  sum c + i  of the call's tokens (or, a place a row, at r).
// Every workgroup sums up all rows by itself, four a thread at a time, and so knows alike whether all of the call fits, and none reads
// what another writes.  Lengths and the pages taken may be written over the inputs: that is left to a second launch where there is more
// than one workgroup.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/dz_amd.h"
#include "dz_attend.h"

namespace {

constexpr int ROWS = 4;                // rows, and tokens, that a thread takes side by side
constexpr int MOST = 1 << 24;          // tokens of a call: of 64 rows no more than 2^30

struct ExtendParams {
  int* tables;
  const int *lengths, *counts, *free, *taken;
  int *lengths_out, *taken_out, *starts;
  long long *positions, *slots;
  unsigned* status;
  long long table_row;
  int rows, width, shift, free_n, tokens, packed;
  int tokens_too, rows_too;            // what this launch writes
  int each;                            // tokens of a workgroup
};

struct Sums {
  long long tokens, pages;
};

// A row's tokens and the pages that it needs; false where a length or a count is below 0 or more than its table, or the call, holds.
__device__ __forceinline__ bool row_fits(const ExtendParams& P, int r, int& n, int& c, int& need) {
  n = P.lengths[r], c = P.counts[r];
  const long long room = (long long)P.width << P.shift;
  const bool fits = n >= 0 && c >= 0 && n + (long long)c <= room && c <= (P.packed ? P.tokens : 1);
  if (!fits) n = c = 0;
  const long long up = (1ll << P.shift) - 1;
  need = (int)((n + c + up) >> P.shift) - (int)((n + up) >> P.shift);
  return fits;
}

// Sums over the rows in front of each thread's, and of all.  A thread's, at most MOST + 1 tokens, stay within 32 bits over a wavefront, where they
// cost half the steps; wavefronts' are added in 64.  (With the numbers stored in pairs, 1777 rows 7.35 us in 64 bits, 6.7 so, 800000 tokens of 400 rows 11.0, 9.9.)
template <int THREADS>
__device__ __forceinline__ Sums sums_before(int c, int need, Sums& all, int (*shared)[2]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tokens = scan_add(c), pages = scan_add(need);
  if (lane == 63) shared[wave][0] = tokens, shared[wave][1] = pages;
  __syncthreads();
  Sums before = {tokens - c, pages - need};
  all = Sums{0, 0};
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    const int x = shared[w][0], y = shared[w][1];
    if (w < wave) before.tokens += x, before.pages += y;
    all.tokens += x, all.pages += y;
  }
  __syncthreads();
  return before;
}

// Four numbers of 64 bits side by side.
typedef long long l2_t __attribute__((ext_vector_type(2), aligned(8)));
__device__ __forceinline__ void put4(long long* to, const long long* x) {
  *(l2_t*)to = l2_t{x[0], x[1]};
  *(l2_t*)(to + 2) = l2_t{x[2], x[3]};
}

template <int THREADS>
__global__ __launch_bounds__(THREADS) void dz_extend_kernel(const ExtendParams P) {
  constexpr int ROUND = THREADS * ROWS;
  __shared__ int shared[THREADS / 64][2];
  __shared__ int upto[ROUND], had[ROUND], page_at[ROUND];            // of a round's rows: tokens up to its end, length, its first page in the list
  const int tid = threadIdx.x, ps = 1 << P.shift;
  const long long taken = P.taken[0];
  int n[ROWS], c[ROWS], need[ROWS], bad = 0;
  auto load = [&](int r0) __attribute__((always_inline)) {
    bool fits = true;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      n[i] = c[i] = need[i] = 0;
      if (r0 + i < P.rows) fits &= row_fits(P, r0 + i, n[i], c[i], need[i]);
    }
    return fits;
  };
  auto sums = [&](Sums& all) __attribute__((always_inline)) {
    int tokens = 0, pages = 0;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) tokens += c[i], pages += need[i];
    tokens = min(tokens, MOST + 1);    // (which is more than there is room for)
    return sums_before<THREADS>(tokens, pages, all, shared);
  };
  Sums total = {0, 0}, all = {0, 0}, before = {0, 0};
  for (int r0 = 0; r0 < P.rows; r0 += ROUND) {
    bad |= !load(r0 + tid * ROWS);
    before = sums(all);
    total.tokens += all.tokens, total.pages += all.pages;
  }
  bad |= taken < 0 || taken + total.pages > P.free_n || (P.packed && total.tokens > P.tokens);
  bad = __syncthreads_or(bad);
  const bool first = blockIdx.x == 0;
  if (bad && first && tid == 0 && P.tokens_too) atomicOr(P.status, 4u);
  const int lo = blockIdx.x * P.each, hi = min(P.tokens, lo + P.each);
  if (P.tokens_too) {                  // places of no token (all of them, where the call does not fit)
    const int end = bad ? 0 : P.packed ? (int)total.tokens : P.tokens;
    for (int t = max(lo, end) + tid; t < hi; t += THREADS) P.positions[t] = 0, P.slots[t] = -1;
  }
  Sums front = {0, 0};                 // of the rounds before
  for (int r0 = 0; r0 < P.rows; r0 += ROUND) {
    const int mine = r0 + tid * ROWS;
    if (P.rows > ROUND) {              // (one round: they are still there)
      load(mine);
      before = sums(all);
    }
    int start = (int)(front.tokens + before.tokens);
    long long page = taken + front.pages + before.pages;
    int* entry[ROWS];
    int id[ROWS];
    if (P.tokens_too && !bad && !P.packed) {
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int r = mine + i;
        entry[i] = nullptr, id[i] = 0;
        if (r < P.rows && r >= lo && r < hi && c[i]) {
          entry[i] = P.tables + r * P.table_row + (n[i] >> P.shift);
          id[i] = need[i] ? P.free[page + (i > 0 ? need[0] : 0) + (i > 1 ? need[1] : 0) + (i > 2 ? need[2] : 0)] : *entry[i];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int r = mine + i;
      if (P.tokens_too) {
        if (first && r < P.rows) P.starts[r] = bad ? 0 : P.packed ? start : r;
        if (!bad && !P.packed && r < P.rows && r >= lo && r < hi) {
          if (need[i]) *entry[i] = id[i];
          if (c[i] && id[i] < 0) atomicOr(P.status, 4u);
          P.positions[r] = c[i] ? n[i] : 0;
          P.slots[r] = c[i] && id[i] >= 0 ? (long long)id[i] * ps + (n[i] & (ps - 1)) : -1;
        }
        if (!bad && P.packed) upto[tid * ROWS + i] = start + c[i], had[tid * ROWS + i] = n[i], page_at[tid * ROWS + i] = (int)page;
      }
      if (P.rows_too && first && r < P.rows) P.lengths_out[r] = bad ? P.lengths[r] : n[i] + c[i];
      start += c[i], page += need[i];
    }
    if (P.tokens_too && !bad && P.packed) {
      __syncthreads();
      // four tokens a thread of those that are this workgroup's, of the rows at hand
      const int from = max(lo, (int)front.tokens), to = min(hi, (int)(front.tokens + all.tokens)), t0 = lo + tid * ROWS;
      int a = 0;
      if (t0 + ROWS > from && t0 < to) {
        int b = ROUND - 1;             // the first row that ends behind the first of them
        while (a < b) {
          const int mid = (a + b) >> 1;
          if (upto[mid] > max(t0, from))
            b = mid;
          else
            a = mid + 1;
        }
      }
      long long at[ROWS], slot[ROWS];
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int t = t0 + i;
        at[i] = 0, slot[i] = -1;
        if (t < from || t >= to) continue;
        while (upto[a] <= t) ++a;      // (some row ends behind t)
        const int pos = had[a] + t - (a ? upto[a - 1] : (int)front.tokens);
        const int used = (had[a] + ps - 1) >> P.shift, place = pos >> P.shift;
        int* to_entry = P.tables + (r0 + a) * P.table_row + place;
        const int page_id = place < used ? *to_entry : P.free[page_at[a] + place - used];
        if (place >= used && (pos & (ps - 1)) == 0) *to_entry = page_id;   // (a new page begins with a new token)
        if (page_id < 0) atomicOr(P.status, 4u);
        at[i] = pos;
        slot[i] = page_id < 0 ? -1 : (long long)page_id * ps + (pos & (ps - 1));
      }
      if (t0 >= from && t0 + ROWS <= to) {
        put4(P.positions + t0, at);
        put4(P.slots + t0, slot);
      } else {
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
          if (t0 + i >= from && t0 + i < to) P.positions[t0 + i] = at[i], P.slots[t0 + i] = slot[i];
      }
      __syncthreads();
    }
    front.tokens += all.tokens, front.pages += all.pages;
  }
  if (first && tid == 0) {
    if (P.tokens_too) P.starts[P.rows] = bad ? 0 : P.packed ? (int)total.tokens : P.rows;
    if (P.rows_too) P.taken_out[0] = bad ? (int)taken : (int)(taken + total.pages);
  }
}

}  // namespace

extern "C" {

int dz_extend_tables(const dz_extend_args* a, void* stream) {
  if (!a || a->bytes != (int64_t)sizeof(*a)) return DZ_EINVAL;
  if (a->rows < 0 || a->rows > (1 << 20) || a->pages_per_row < 0 || a->page_size < 8 || a->page_size > 1024 || (a->page_size & (a->page_size - 1)) ||
      (long long)a->pages_per_row * a->page_size > (1ll << 30) || a->free_n < 0 || a->tokens < 0 || a->tokens > MOST || (!a->packed && a->tokens != a->rows) ||
      a->table_row < 0)
    return DZ_EPAGES;
  if ((a->rows && (!a->lengths || !a->counts || !a->lengths_out || (!a->tables && a->pages_per_row))) || (!a->free_pages && a->free_n) || !a->taken ||
      !a->taken_out || !a->starts || (a->tokens && (!a->positions || !a->slots)) || !a->status)
    return DZ_EINVAL;
  if ((((uintptr_t)a->tables | (uintptr_t)a->lengths | (uintptr_t)a->counts | (uintptr_t)a->free_pages | (uintptr_t)a->taken | (uintptr_t)a->lengths_out |
        (uintptr_t)a->taken_out | (uintptr_t)a->starts | (uintptr_t)a->status) & 3) || (((uintptr_t)a->positions | (uintptr_t)a->slots) & 7))
    return DZ_EALIGN;
  ExtendParams P;
  P.tables = a->tables, P.lengths = a->lengths, P.counts = a->counts, P.free = a->free_pages, P.taken = a->taken;
  P.lengths_out = a->lengths_out, P.taken_out = a->taken_out, P.starts = a->starts;
  P.positions = (long long*)a->positions, P.slots = (long long*)a->slots, P.status = a->status;
  P.table_row = a->table_row;
  P.rows = a->rows, P.width = a->pages_per_row, P.shift = __builtin_ctz(a->page_size), P.free_n = a->free_n, P.tokens = a->tokens, P.packed = a->packed != 0;
  // threads for all rows in one round, where these are enough (16 rows 6.3 us with 1024, 5.0 with 64, sums in 64 bits); of a token a row each few a workgroup, as
  // their pages lie apart (1777 rows 8.1 -> 7.4 us, likewise), of others four a thread
  const int threads = a->rows <= 64 * ROWS && a->tokens <= 64 * ROWS ? 64 : a->rows <= 256 * ROWS ? 256 : 1024;
  P.each = a->packed ? threads * ROWS : 256;
  const int grid = a->tokens > P.each ? (a->tokens + P.each - 1) / P.each : 1;
  const bool over = a->lengths_out == a->lengths || a->taken_out == a->taken;
  P.tokens_too = 1, P.rows_too = grid == 1 || !over;
  const hipStream_t st = (hipStream_t)stream;
  auto launch = [&](int workgroups) {
    if (threads == 64)
      hipLaunchKernelGGL(dz_extend_kernel<64>, dim3(workgroups), dim3(64), 0, st, P);
    else if (threads == 256)
      hipLaunchKernelGGL(dz_extend_kernel<256>, dim3(workgroups), dim3(256), 0, st, P);
    else
      hipLaunchKernelGGL(dz_extend_kernel<1024>, dim3(workgroups), dim3(1024), 0, st, P);
  };
  launch(grid);
  if (!P.rows_too) {
    P.tokens_too = 0, P.rows_too = 1;
    launch(1);
  }
  return hipGetLastError() == hipSuccess ? DZ_OK : DZ_ELAUNCH;
}

}  // extern "C"
