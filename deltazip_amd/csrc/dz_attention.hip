// Attention of one new token per row over a paged key/value cache.
//
//   o = sum_t 2^(s_t - m) v_t / sum_t 2^(s_t - m),   s_t = scale log2(e) q.k_t,   max(0, n - window) <= t < n
//
// for every row (a sequence with its length n and its table of pages) and head; the heads / kv_heads heads that
// share a key head are taken together, up to 16 at once, so that every key and value is read once.  What bounds it
// is the reading of keys and values: 4 flops per byte and head against the 300 that the card has.
//
// A wavefront walks 32 tokens at a time and holds all of it in registers (dz_attend.h).
//
// The work is cut on the device, which alone knows the lengths: every wavefront reads the lengths of the launch's
// rows (up to 256, up to four a lane) and cuts them into as many equal parts as make 512 or 768 workgroups together.
// Rows of much work go first: 200 rows of 1 to 4000 tokens 96 -> 78 us.  Parts are joined by the workgroup that is done last
// of up to 16 of them, and these joined ones again (counters say who is last), in the order of the tokens: results
// do not depend on timing.
//
// Measured (keys and values over the time of a call among others): 128 rows of 1025 tokens of 32 key heads of 128 325 us, 6.6 TB/s;
// 32 of 1024 84 us, 6.4; one of 131071 tokens of 8 94 us, 5.7, of which 76 at the rate of a kernel that only reads (7.1 TB/s with
// loads that keep nothing in the caches, 6.2 with others; a copy moves 4.9 to 5.4); one of 17 tokens 5 us, of which an empty
// launch takes 2.5.  32 rows of 1024 tokens of 16 key heads of 256 89 us, 6.0 TB/s; of 200 185 us, 2.3: the form of heads of 200 to 248 takes
// more than half of the registers, so one wavefront a SIMD asks for keys no step ahead.  A compute unit has some 64 KB on their way at most, which at 2 us is 30 GB/s: what long
// rows lose is the uneven ends of their parts (63 to 86 us) and the two joins (9 us).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/dz_amd.h"
#include "dz_attend.h"

pthread_mutex_t dz_attention_launches = PTHREAD_MUTEX_INITIALIZER;

namespace {

constexpr int WAVES = 4;               // wavefronts of a workgroup
constexpr int HEADS = 16;              // heads taken together: columns of a matrix instruction
constexpr int GROUP_ROWS = 256;        // rows of a launch: four lengths a lane
constexpr int TARGET = 768;            // workgroups that the work of a launch is cut into at most, rows' last parts apart
constexpr int FEW_ROWS = 16;           // below: two workgroups for each of 256 compute units
constexpr int COUNTERS = DZ_ATTENTION_COUNTERS / 2;   // workgroups of a launch with parts, at most
constexpr size_t LDS_MOST = 96 << 10;
constexpr float CACHED = 64 << 20;     // bytes of keys and values up to which they may be in the last cache, of 256 MB (24 rows of 1000
                                       // tokens, 40 MB, in turn with two others': 20 us, past the caches 25)
constexpr int GROUP = 16;              // parts joined at once
constexpr int WHOLE = 12;              // tiles up to which a row has one part: a join takes as long as three steps (300 tokens 9.7 -> 8.7 us)
constexpr int LONG = 32;               // tiles of a part up to which no row has more than GROUP: joins in two takes cost 3 us more (8000 tokens 18.5 -> 16)

struct AttnParams {
  const char *q, *k, *v;
  const int *tables, *lengths;
  uint16_t* out;
  float* parts;
  unsigned* counters;
  unsigned* status;
  long long q_row, q_head, k_page, k_head, k_token, v_page, v_head, v_token, out_row, out_head, table_row;   // bytes; out, table: elements
  unsigned num_pages;
  int rows, heads, kv_heads, share, head_tiles, dim, shift, pages_per_row, window, part_floats, stat_at, single, once, shared;
  float scale, cut;
};

// Tokens [first, end) of a row, end <= the table's room.
__device__ __forceinline__ void span(const AttnParams& P, int length, int& first, int& end) {
  const int room = P.pages_per_row << P.shift;
  end = length < 0 ? 0 : length > room ? room : length;
  first = P.window > 0 && end > P.window ? end - P.window : 0;
}

__device__ __forceinline__ int tiles_of(const AttnParams& P, int length) {
  int first, end;
  span(P, length, first, end);
  return end > first ? (end + TILE - 1) / TILE - first / TILE : 0;
}

// The part of the launch that a workgroup is, as each of its wavefronts works it out: part `nth` of `nparts` of `row`.
struct Part {
  int row, length, nth, nparts;
  bool once;                           // whether the launch's keys and values are more than the caches keep
};

__device__ __forceinline__ Part find_part(const AttnParams& P, int part, int items, int lane) {
  Part found = {-1, 0, 0, 1, false};
  if (P.single) {                      // (no row can have a second part)
    found.row = part;
    found.length = P.lengths[part];
    found.once = P.once;
    return found;
  }
  // lane l has rows l * each_lane .. ; their tiles, and the parts in front of them
  const int each_lane = (P.rows + 63) / 64, row0 = lane * each_lane;
  int length[4], tiles[4], before[4];
  float mine = 0.0f;
#pragma unroll
  for (int r = 0; r < 4; ++r) length[r] = r < each_lane && row0 + r < P.rows ? P.lengths[row0 + r] : 0;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    tiles[r] = tiles_of(P, length[r]);
    mine += (float)tiles[r];
  }
  const float total = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, scan_add(mine)), 63)) * (float)items;
  found.once = !P.shared && total * (TILE * 4.0f) * (float)P.dim > CACHED;
  // tiles of a part, in whole steps of the workgroup (sums above 2^24 are rounded, which may come to one part more)
  const float most = ceilf(total * P.cut);
  const unsigned each = WAVES * (unsigned)fminf(fmaxf(most, 1.0f), (float)(1 << 24));
  int parts[4], heavy = 0, light = 0;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    parts[r] = 0;
    if (r < each_lane) {
      parts[r] = tiles[r] <= WHOLE ? 1 : (int)((tiles[r] + each - 1) / each);      // (an empty row has its zeros written)
      if (parts[r] > GROUP && tiles[r] <= GROUP * LONG) parts[r] = GROUP;
      if (row0 + r >= P.rows) parts[r] = 0;
    }
    const bool is = 2 * tiles[r] > (int)each;
    before[r] = is ? heavy : light;
    if (is)
      heavy += parts[r];
    else
      light += parts[r];
  }
  // rows of much work first: they are dealt to the compute units evenly, and the others fill up
  const int upto = scan_add(heavy), front_heavy = upto - heavy;
  const int front_light = scan_add(light) - light + __builtin_amdgcn_readlane(upto, 63);
#pragma unroll
  for (int r = 0; r < 4; ++r) before[r] += 2 * tiles[r] > (int)each ? front_heavy : front_light;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (r >= each_lane) break;
    const int at = part - before[r];
    const unsigned long long hit = __ballot(at >= 0 && at < parts[r]);
    if (hit) {
      const int src = __builtin_ctzll(hit);
      found.row = src * each_lane + r;
      found.length = __builtin_amdgcn_readlane(length[r], src);
      found.nth = __builtin_amdgcn_readlane(at, src);
      found.nparts = __builtin_amdgcn_readlane(parts[r], src);
    }
  }
  return found;
}

// Sums of parts go from one workgroup to another past the caches of the eight dies (sc1: agent scope): a fence there writes
// back and empties a whole cache, which took six times as long as the attention itself.
struct Shared {
  __amdgpu_buffer_rsrc_t at;
  __device__ __forceinline__ explicit Shared(float* base) : at(__builtin_amdgcn_make_buffer_rsrc(base, 0, 0xffffffff, 0x00027000)) {}
  __device__ __forceinline__ void put(unsigned offset, f4_t x) const {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4_t, x), at, offset, 0, 16);
  }
  __device__ __forceinline__ void put(unsigned offset, f2_t x) const {
    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u2_t, x), at, offset, 0, 16);
  }
  __device__ __forceinline__ f4_t get4(unsigned offset) const {
    return __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(at, offset, 0, 16));
  }
  __device__ __forceinline__ f2_t get2(unsigned offset) const {
    return __builtin_bit_cast(f2_t, __builtin_amdgcn_raw_buffer_load_b64(at, offset, 0, 16));
  }
};

// (heads of 64 fit four wavefronts a SIMD: with three, 64 rows of 1024 tokens of 8 key heads 28 -> 33 us)
template <int KC, bool FULL, bool BF>
__global__ __launch_bounds__(64 * WAVES, KC == 8 && !FULL ? 1 : KC == 2 && FULL ? 4 : 2) void dz_attention_kernel(const AttnParams P) {
  typedef Type<BF> Ty;
  typedef typename Ty::v8 v8;
  constexpr int NB = (KC + 3) / 4;     // blocks of 128 dims
  extern __shared__ float lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const int items = P.kv_heads * P.head_tiles;
  const int part = blockIdx.x / items, item = blockIdx.x % items;
  const int kvh = item / P.head_tiles, head0 = kvh * P.share + item % P.head_tiles * HEADS;
  const int nheads = min(HEADS, (kvh + 1) * P.share - head0);

  const Part mine = find_part(P, part, items, lane);
  const int row = mine.row, length = mine.length, nth = mine.nth, nparts = mine.nparts;
  if (row < 0) return;
  int first, end;
  span(P, length, first, end);
  if (length > end && nth == 0 && item == 0 && threadIdx.x == 0) atomicOr(P.status, 4u);
  const int tiles = end > first ? (end + TILE - 1) / TILE - first / TILE : 0, tile0 = first / TILE;
  // this part's tiles, and this wavefront's of them
  const int lo = (int)((long long)tiles * nth / nparts), hi = (int)((long long)tiles * (nth + 1) / nparts);
  int t0 = tile0 + lo + (hi - lo) * wave / WAVES;
  const int t1 = tile0 + lo + (hi - lo) * (wave + 1) / WAVES;

  // queries: lane holds dims 32 c + 8 g .. + 7 of head `col`
  Walk<KC, FULL, BF, false> walk;
#pragma unroll
  for (int c = 0; c < KC; ++c) {
    u4_t w = {0, 0, 0, 0};
    if (col < nheads && 32 * c + 8 * g < P.dim)
      w = *(const u4_t*)(P.q + row * P.q_row + (head0 + col) * P.q_head + (32 * c + 8 * g) * 2);
    walk.q[c] = __builtin_bit_cast(v8, w);
  }
  const int* table = P.tables + row * P.table_row;
  if (mine.once)
    walk.template run<true, false>(P, table, kvh, first, end, t0, t1, end, end);
  else
    walk.template run<false, false>(P, table, kvh, first, end, t0, t1, end, end);
  const auto& acc = walk.acc;
  const float top = walk.top;
  float sum = walk.sum;
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);

  // the four wavefronts' sums joined: [wave][head][dim], then maxima and sums
  const int ld = P.dim + 4;
  float* sums = lds + wave * nheads * ld;
  float* stat = lds + P.stat_at;
  if (col < nheads) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 128 * b + 8 * (4 * g + i);
        if (d < P.dim) {
          *(f4_t*)(sums + col * ld + d) = f4_t{acc[8 * b][i], acc[8 * b + 1][i], acc[8 * b + 2][i], acc[8 * b + 3][i]};
          *(f4_t*)(sums + col * ld + d + 4) = f4_t{acc[8 * b + 4][i], acc[8 * b + 5][i], acc[8 * b + 6][i], acc[8 * b + 7][i]};
        }
      }
    if (g == 0) {
      stat[(wave * HEADS + col) * 2] = top;
      stat[(wave * HEADS + col) * 2 + 1] = sum;
    }
  }
  __syncthreads();
  const int quads = P.dim / 4, spots = nheads * quads;
  const Shared parts(P.parts);
  const unsigned record = P.part_floats * 4u, stats = nheads * P.dim * 4u;      // bytes of a part, of its values
  auto store = [&](int h, int d, f4_t o, float l) {
    const f4_t y = tiles ? o / l : f4_t{0, 0, 0, 0};
    uint16_t* at = P.out + row * P.out_row + (head0 + h) * P.out_head + d;
    const u2_t w = {(unsigned)Ty::round(y[0]) | (unsigned)Ty::round(y[1]) << 16,
                    (unsigned)Ty::round(y[2]) | (unsigned)Ty::round(y[3]) << 16};
    *(u2_t*)at = w;
  };
  auto leave = [&](unsigned slot, int h, int d, f4_t o, float m, float l) {
    parts.put(slot * record + (h * P.dim + d) * 4, o);
    if (d == 0) parts.put(slot * record + stats + 8 * h, f2_t{m, l});
  };
  for (int x = threadIdx.x; x < spots; x += 64 * WAVES) {
    const int h = x / quads, d = x % quads * 4;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) m = fmaxf(m, stat[(w * HEADS + h) * 2]);
    float l = 0.0f;
    f4_t o = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float lw = stat[(w * HEADS + h) * 2 + 1], mw = stat[(w * HEADS + h) * 2];
      const float f = weight_of(mw, m);
      l += lw * f;
      o += *(const f4_t*)(lds + (w * nheads + h) * ld + d) * f;
    }
    if (nparts > 1)
      leave(blockIdx.x, h, d, o, m, l);
    else
      store(h, d, o, l);
  }
  if (nparts <= 1) return;

  // The last to be done of up to GROUP parts joins them; in a row of more it leaves the result behind the parts, and the last to
  // be done of these joins those.
  int* flag = (int*)(stat + 2 * WAVES * HEADS);
  auto last_of = [&](unsigned* counter, int n) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this wavefront's sums have arrived
    __syncthreads();
    if (threadIdx.x == 0) {
      const bool last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)n - 1;
      if (last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // as the next call wants it
      *flag = last;
    }
    __syncthreads();
    return *flag != 0;
  };
  // a thread takes four values of a head over every `slices`-th part; threads that have none of their own share the
  // parts of others'
  int slices = 1;
  while (2 * slices * spots <= 64 * WAVES) slices *= 2;
  auto join = [&](unsigned slot, unsigned step, int n, auto emit) {
    auto gather = [&](auto at_once) {
      constexpr int N = decltype(at_once)::value;      // parts that a thread asks for at a time
      for (int x = threadIdx.x; x < spots * slices; x += 64 * WAVES) {
        const int spot = x % spots, h = spot / quads, d = spot % quads * 4;
        float m = -INFINITY, l = 0.0f;
        f4_t o = {0, 0, 0, 0};
        for (int s = x / spots; s < n; s += N * slices) {
          f4_t w[N];
          f2_t ml[N];
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const unsigned at = (slot + min(s + i * slices, n - 1) * step) * record;
            ml[i] = parts.get2(at + stats + 8 * h);
            w[i] = parts.get4(at + (h * P.dim + d) * 4);
          }
          float up = m;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            if (s + i * slices >= n) ml[i][0] = -INFINITY;
            up = fmaxf(up, ml[i][0]);
          }
          const float f = weight_of(m, up);
          l *= f, o *= f, m = up;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const bool none = s + i * slices >= n;       // (the last part a second time)
            const float fs = weight_of(ml[i][0], up);
            l += none ? 0.0f : ml[i][1] * fs;
            o += none ? f4_t{0, 0, 0, 0} : w[i] * fs;
          }
        }
        if (slices == 1) {
          emit(h, d, o, m, l);
        } else {
          *(f4_t*)(lds + 8 * x) = o;                   // [slice][spot]: values, maximum and sum
          *(f2_t*)(lds + 8 * x + 4) = f2_t{m, l};
        }
      }
    };
    if (slices >= 4)
      gather(std::integral_constant<int, GROUP / 4>());
    else
      gather(std::integral_constant<int, GROUP>());
    if (slices == 1) return;
    __syncthreads();
    for (int spot = threadIdx.x; spot < spots; spot += 64 * WAVES) {
      float m = -INFINITY, l = 0.0f;
      f4_t o = {0, 0, 0, 0};
      for (int c = 0; c < slices; ++c) m = fmaxf(m, lds[8 * (c * spots + spot) + 4]);
      for (int c = 0; c < slices; ++c) {
        const float* at = lds + 8 * (c * spots + spot);
        const float f = weight_of(at[4], m);
        l += at[5] * f;
        o += *(const f4_t*)at * f;
      }
      emit(spot / quads, spot % quads * 4, o, m, l);
    }
  };
  const auto finish = [&](int h, int d, f4_t o, float m, float l) { store(h, d, o, l); };
  const unsigned slot0 = blockIdx.x - nth * items, mine0 = slot0 + nth / GROUP * GROUP * items;      // of the row's, the group's first part
  const int members = min(GROUP, nparts - nth / GROUP * GROUP), groups = (nparts + GROUP - 1) / GROUP;
  if (!last_of(P.counters + mine0, members)) return;
  if (groups == 1) {
    join(slot0, items, members, finish);
    return;
  }
  join(mine0, items, members, [&](int h, int d, f4_t o, float m, float l) { leave(gridDim.x + mine0, h, d, o, m, l); });
  if (!last_of(P.counters + COUNTERS + slot0, groups)) return;
  join(gridDim.x + slot0, GROUP * items, groups, finish);
}

// Rows that go in one launch.
inline int group_rows(int items) { return min(GROUP_ROWS, (COUNTERS - TARGET) / items - 1); }

inline long long most_groups(int rows, int items, long long room) {
  const long long whole = (room + TILE - 1) / TILE;              // tiles of the longest row
  const long long parts = whole <= WHOLE ? 1 : (whole + WAVES - 1) / WAVES;
  const long long all = parts * rows * items, cut = TARGET + (rows + 1ll) * items;
  return all < cut ? all : cut;
}

typedef void (*kernel_t)(const AttnParams);
template <int KC, bool BF>
kernel_t kernel_of(int dim) {
  return dim == 32 * KC ? dz_attention_kernel<KC, true, BF> : dz_attention_kernel<KC, false, BF>;
}
inline int chunks_of(int dim) { return dim <= 64 ? 2 : dim <= 96 ? 3 : dim <= 128 ? 4 : dim <= 192 ? 6 : 8; }
template <bool BF>
kernel_t kernel_for(int dim) {
  const int kc = chunks_of(dim);
  return kc == 2 ? kernel_of<2, BF>(dim) : kc == 3 ? kernel_of<3, BF>(dim) : kc == 4 ? kernel_of<4, BF>(dim)
         : kc == 6 ? kernel_of<6, BF>(dim) : kernel_of<8, BF>(dim);
}

inline bool shapes_fit(int rows, int heads, int kv_heads, int dim, int page_size, int pages_per_row) {
  return rows >= 0 && heads >= 1 && kv_heads >= 1 && heads <= 4096 && heads % kv_heads == 0 && dim >= 8 && dim <= 256 && dim % 8 == 0 &&
         page_size >= 8 && page_size <= 1024 && (page_size & (page_size - 1)) == 0 && pages_per_row >= 0 &&
         (long long)pages_per_row * page_size <= (1ll << 30);
}

}  // namespace

extern "C" {

size_t dz_paged_attention_bytes(int rows, int heads, int kv_heads, int dim, int page_size, int pages_per_row) {
  if (!shapes_fit(rows, heads, kv_heads, dim, page_size, pages_per_row)) return 0;
  const int share = heads / kv_heads, items = kv_heads * ((share + HEADS - 1) / HEADS);
  const int most = share < HEADS ? share : HEADS;
  const int together = group_rows(items) < rows ? group_rows(items) : rows;
  const long long groups = most_groups(together, items, (long long)pages_per_row * page_size);
  return groups > (long long)together * items ? 2 * (size_t)groups * most * (dim + 4) * 4 : 0;   // (no row has parts)
}

unsigned long long dz_capture_id(void* stream) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (hipStreamGetCaptureInfo((hipStream_t)stream, &status, &id) != hipSuccess) {
    (void)hipGetLastError();
    return 0;
  }
  return status == hipStreamCaptureStatusActive ? id : 0;
}

int dz_paged_attention(const dz_attention_args* a, void* stream) {
  if (!a || a->bytes != (int64_t)sizeof(*a)) return DZ_EINVAL;
  if (!shapes_fit(a->rows, a->heads, a->kv_heads, a->dim, a->page_size, a->pages_per_row)) return DZ_EPAGES;
  if (a->dtype != DZ_F16 && a->dtype != DZ_BF16) return DZ_EINVAL;
  if (a->rows == 0) return DZ_OK;
  if (!a->q || !a->k_pages || !a->v_pages || (!a->tables && a->pages_per_row) || !a->lengths || !a->out || !a->status || a->window < 0)
    return DZ_EINVAL;
  if (a->num_pages < 1 || a->num_pages > 0x7fffffffll) return DZ_EPAGES;
  const int64_t strides[] = {a->q_row, a->q_head, a->k_page, a->k_head, a->k_token, a->v_page, a->v_head, a->v_token, a->out_row, a->out_head};
  for (int64_t s : strides)
    if (s < 0 || s % 8) return DZ_EALIGN;
  if (((uintptr_t)a->q | (uintptr_t)a->k_pages | (uintptr_t)a->v_pages | (uintptr_t)a->out) & 15) return DZ_EALIGN;
  if (((uintptr_t)a->tables | (uintptr_t)a->lengths | (uintptr_t)a->status) & 3) return DZ_EALIGN;
  if (a->table_row < 0) return DZ_EPAGES;
  const size_t need = dz_paged_attention_bytes(a->rows, a->heads, a->kv_heads, a->dim, a->page_size, a->pages_per_row);
  if (need && (!a->work || (size_t)a->work_bytes < need || ((uintptr_t)a->work & 15) || !a->counters || ((uintptr_t)a->counters & 3)))
    return DZ_EWORKSPACE;

  AttnParams P;
  P.k = (const char*)a->k_pages;
  P.v = (const char*)a->v_pages;
  P.parts = (float*)a->work;
  P.counters = a->counters;
  P.status = a->status;
  P.q_row = 2 * a->q_row, P.q_head = 2 * a->q_head;
  P.k_page = 2 * a->k_page, P.k_head = 2 * a->k_head, P.k_token = 2 * a->k_token;
  P.v_page = 2 * a->v_page, P.v_head = 2 * a->v_head, P.v_token = 2 * a->v_token;
  P.out_row = a->out_row, P.out_head = a->out_head, P.table_row = a->table_row;
  P.num_pages = (unsigned)a->num_pages;
  P.heads = a->heads, P.kv_heads = a->kv_heads, P.share = a->heads / a->kv_heads;
  P.head_tiles = (P.share + HEADS - 1) / HEADS;
  P.dim = a->dim, P.shift = __builtin_ctz(a->page_size), P.pages_per_row = a->pages_per_row, P.window = a->window;
  P.shared = a->shared && a->rows > 1;                             // (one row reads its pages once)
  const int most = P.share < HEADS ? P.share : HEADS, items = P.kv_heads * P.head_tiles;
  P.part_floats = most * (a->dim + 4);
  P.scale = a->scale * 1.44269504088896340736f;
  // the wavefronts' sums; or what threads add up for others
  const size_t sums = (size_t)WAVES * most * (a->dim + 4), joins = 8 * 64 * WAVES;
  const size_t lds = ((sums > joins ? sums : joins) + 2 * WAVES * HEADS + 4) * 4;
  P.stat_at = (int)(lds / 4) - (2 * WAVES * HEADS + 4);
  const kernel_t kern = a->dtype == DZ_BF16 ? kernel_for<true>(a->dim) : kernel_for<false>(a->dim);
  const int kc = chunks_of(a->dim), which = kc * 4 + (a->dim == 32 * kc) * 2 + a->dtype;
  static std::atomic<unsigned long long> attr_done[36];        // one per kernel
  if (lds > 65536 && !dz_lds_limit_once(attr_done[which], (const void*)kern, (int)LDS_MOST)) return DZ_ELAUNCH;
  const hipStream_t st = (hipStream_t)stream;
  const int together = group_rows(items);
  const Launches held;
  for (long long row = 0; row < a->rows; row += together) {
    P.rows = a->rows - row < together ? (int)(a->rows - row) : together;
    P.q = (const char*)a->q + row * P.q_row;
    P.out = (uint16_t*)a->out + row * P.out_row;
    P.tables = a->tables + row * P.table_row;
    P.lengths = a->lengths + row;
    long long seen = (long long)a->pages_per_row * a->page_size;
    if (a->window && a->window + 2ll * TILE < seen) seen = a->window + 2ll * TILE;             // (it may begin and end inside a tile)
    const long long groups = most_groups(P.rows, items, seen);
    P.once = !P.shared && (float)P.rows * items * seen * 4.0f * a->dim > CACHED;
    P.cut = 1.0f / (WAVES * (P.rows < FEW_ROWS ? 512 : TARGET));
    P.single = groups == (long long)P.rows * items;
    hipLaunchKernelGGL(kern, dim3((unsigned)groups), dim3(64 * WAVES), lds, st, P);
  }
  return hipGetLastError() == hipSuccess ? DZ_OK : DZ_ELAUNCH;
}

}  // extern "C"
