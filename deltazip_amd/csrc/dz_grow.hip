// Tables, positions and slots of the tokens that rows get next, made on the device.
//
// Row r has n tokens and gets c more.  With  need = ceil((n + c) / ps) - ceil(n / ps)  and exclusive sums over the rows
//   page j of its new ones is  free[taken + sum need + j],  and token i of them stands at position n + i, in place (n + i) % ps of
//   page (n + i) / ps of its table, and at  sum c + i  of the call's tokens (or, a place a row, at r).
// Every workgroup sums up all rows by itself, 1024 at a time, and so knows alike whether all of the call fits, and none reads
// what another writes.  Lengths and the pages taken may be written over the inputs: that is left to a second launch where there is more
// than one workgroup.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/dz_amd.h"
#include "dz_attend.h"

namespace {

constexpr int THREADS = 1024;
constexpr int EACH = 4096;             // tokens of a workgroup
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

// Sums over the rows in front of each thread's, and of all.
__device__ __forceinline__ Sums sums_before(int c, int need, Sums& all, int (*shared)[2]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tokens = scan_add(c), pages = scan_add(need);
  if (lane == 63) shared[wave][0] = tokens, shared[wave][1] = pages;
  __syncthreads();
  Sums before = {tokens - c, pages - need};
  all = Sums{0, 0};
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    const int a = shared[w][0], b = shared[w][1];
    if (w < wave) before.tokens += a, before.pages += b;
    all.tokens += a, all.pages += b;
  }
  __syncthreads();
  return before;
}

__global__ __launch_bounds__(THREADS) void dz_extend_kernel(const ExtendParams P) {
  __shared__ int shared[THREADS / 64][2];
  __shared__ int upto[THREADS], had[THREADS], page_at[THREADS];      // of a round's rows: tokens up to its end, length, its first page in the list
  const int tid = threadIdx.x, ps = 1 << P.shift;
  const long long taken = P.taken[0];
  int n = 0, c = 0, need = 0, bad = 0;
  Sums total = {0, 0}, all = {0, 0}, before = {0, 0};
  for (int r0 = 0; r0 < P.rows; r0 += THREADS) {
    n = c = need = 0;
    if (r0 + tid < P.rows) bad |= !row_fits(P, r0 + tid, n, c, need);
    before = sums_before(c, need, all, shared);
    total.tokens += all.tokens, total.pages += all.pages;
  }
  bad |= taken < 0 || taken + total.pages > P.free_n || (P.packed && total.tokens > P.tokens);
  bad = __syncthreads_or(bad);
  if (bad && blockIdx.x == 0 && tid == 0 && P.tokens_too) atomicOr(P.status, 4u);
  const bool first = blockIdx.x == 0;
  const int lo = blockIdx.x * EACH, hi = min(P.tokens, lo + EACH);
  if (P.tokens_too) {                  // places of no token (all of them, where the call does not fit)
    const int end = bad ? 0 : P.packed ? (int)total.tokens : P.tokens;
    for (int t = max(lo, end) + tid; t < hi; t += THREADS) P.positions[t] = 0, P.slots[t] = -1;
  }
  Sums front = {0, 0};                 // of the rounds before
  for (int r0 = 0; r0 < P.rows; r0 += THREADS) {
    const int r = r0 + tid;
    if (P.rows > THREADS) {            // (one round: they are still there)
      n = c = need = 0;
      if (r < P.rows) row_fits(P, r, n, c, need);
      before = sums_before(c, need, all, shared);
    }
    const int start = (int)(front.tokens + before.tokens);
    const long long page = taken + front.pages + before.pages;
    if (P.tokens_too) {
      if (first && r < P.rows) P.starts[r] = bad ? 0 : P.packed ? start : r;
      if (!bad && !P.packed) {
        if (r < P.rows && r >= lo && r < hi) {
          long long slot = -1;
          if (c) {
            int* entry = P.tables + r * P.table_row + (n >> P.shift);
            const int id = need ? P.free[page] : *entry;
            if (need) *entry = id;
            if (id < 0)
              atomicOr(P.status, 4u);
            else
              slot = (long long)id * ps + (n & (ps - 1));
          }
          P.positions[r] = c ? n : 0;
          P.slots[r] = slot;
        }
      } else if (!bad) {
        upto[tid] = start + c, had[tid] = n, page_at[tid] = (int)page;
        __syncthreads();
        const int from = max(lo, (int)front.tokens), to = min(hi, (int)(front.tokens + all.tokens));
        for (int t = from + tid; t < to; t += THREADS) {
          int a = 0, b = THREADS - 1;  // the first row that ends behind t
          while (a < b) {
            const int mid = (a + b) >> 1;
            if (upto[mid] > t)
              b = mid;
            else
              a = mid + 1;
          }
          const int at = had[a] + t - (a ? upto[a - 1] : (int)front.tokens);
          const int used = (had[a] + ps - 1) >> P.shift, place = at >> P.shift;
          int* entry = P.tables + (r0 + a) * P.table_row + place;
          const int id = place < used ? *entry : P.free[page_at[a] + place - used];
          if (place >= used && (at & (ps - 1)) == 0) *entry = id;      // (a new page begins with a new token)
          if (id < 0) atomicOr(P.status, 4u);
          P.positions[t] = at;
          P.slots[t] = id < 0 ? -1 : (long long)id * ps + (at & (ps - 1));
        }
        __syncthreads();
      }
    }
    if (P.rows_too && first && r < P.rows) P.lengths_out[r] = bad ? P.lengths[r] : n + c;
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
  const int grid = a->tokens > EACH ? (a->tokens + EACH - 1) / EACH : 1;
  const bool over = a->lengths_out == a->lengths || a->taken_out == a->taken;
  P.tokens_too = 1, P.rows_too = grid == 1 || !over;
  const hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(dz_extend_kernel, dim3(grid), dim3(THREADS), 0, st, P);
  if (!P.rows_too) {
    P.tokens_too = 0, P.rows_too = 1;
    hipLaunchKernelGGL(dz_extend_kernel, dim3(1), dim3(THREADS), 0, st, P);
  }
  return hipGetLastError() == hipSuccess ? DZ_OK : DZ_ELAUNCH;
}

}  // extern "C"
