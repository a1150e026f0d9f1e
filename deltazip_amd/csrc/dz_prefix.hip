// Attention of the new tokens of a batch over a paged key/value cache, where groups of rows share their first tokens.
//
//   o_i = sum_t 2^(s_t - m) v_t / sum_t 2^(s_t - m),   s_t = scale log2(e) q_i.k_t,   t < n - (c - 1 - i)
//
// for token i of the c new ones of a row with n tokens, and every head.  A group's rows see the same first tokens: the sums over
// these are taken for all of the group's tokens and heads at once, so that its keys and values are read once (per 128 queries)
// and not once per row, and joined with the sums over what is each row's own:
//   m = max m_p,  l = sum l_p 2^(m_p - m),  o = sum o_p 2^(m_p - m) / l
//
// The work is units (a group's prefix; a row's own tokens) of tiles of 128 queries (a token and one of the heads that share a key)
// times pieces of the tokens that these see.  dz_prefix_plan_kernel, one workgroup, makes the list of them from the lengths, which only
// the device knows; a workgroup of dz_prefix_kernel takes one of them for one key head; dz_prefix_join_kernel joins.
//
// A tile's workgroup brings 64 tokens' keys and values into LDS (two steps' room, loads that pass the registers by) and has 32 queries a
// wavefront.  As in dz_attend.h scores are C[token, query] = K Q^T, so that a lane's weights are just what the second product's
// operand wants of it; the values' operand is read from LDS by the transposing read.  A query tile's operand from LDS serves two
// matrix instructions; with more queries a wavefront their sums fill the registers that a second workgroup on the compute unit needs.
// A weight is held in two values of the type in tiles of up to 64 queries, as for few queries: half as many matrix instructions again, which cost nothing there (32
// rows 31.2 and 30.8 us, 128 rows in 4 groups 230 and 230, 48 rows of drafted tokens 32.0 and 32.6), and outputs are off by their own rounding.  In larger ones they
// would cost (two values: 80 queries behind 131072 tokens 120 -> 130 us, 203 rows of 8 heads a key 361 -> 390, nine prompts 32.5 -> 36.8, 8192 tokens 567 -> 742): there it is one
// value, times 2^14 in fp16.  Outputs are then 2.0e-3 to 2.1e-3 (bf16) off in the root mean square where their own rounding is 1.65e-3, 2.2e-4 and 2.0e-4 in fp16.
//
// What bounds it: reading keys and values once up to some 180 queries a key, the matrix cores above.  Measured, a pass among others:
//   a prompt of 8192 tokens of 32 heads of 128, 8 key heads     573 to 591 us from one card to another, 930 to 960 TFLOP/s (a library product of 8192^3
//                                                               1171 to 1220)
//   16 rows behind 131072 tokens of 8 key heads                 119 us, 4.7 TB/s; 5.8 while all workgroups read
//   128 rows in 4 groups behind 4096 tokens of 32 key heads     230 us, 5.9 TB/s
//   203 rows of 64 heads in 3 groups behind 20000 of 8          365 us, 3.9 TB/s and 376 TFLOP/s: neither one's bound; a compute unit's two workgroups are
//                                                               too few to wait for memory and to multiply at the same time
//   32 rows behind 2048 of 32                                   31 us: plan 5, pieces 22 (a piece takes 14: memory is waited for in turn), join 5
// What did not pay: the exponentials of 32 tokens beside the products of the next 32 (more instructions, 560 -> 621 us for 8192 tokens) or of one
// query tile beside the other's (680: operands read twice); priorities of wavefronts (the same); a queue of items that workgroups which stay take from (203 rows 360 -> 588:
// registers to keep the plan, and no two tiles of a key head at once); 768 to 1536 pieces (16 rows 122 -> 133 to 147, 128 rows 238 -> 245).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/dz_amd.h"
#include "dz_attend.h"

namespace {

typedef short s4_t __attribute__((ext_vector_type(4)));
typedef short s8_t __attribute__((ext_vector_type(8)));

constexpr int ROWS = 128;              // queries of a workgroup
// Queries of a unit up to which wavefronts share out its tokens and not its queries: they wait for memory by themselves and hold weights in two
// values (128 rows behind 4096 tokens, one query a row's own, 256 -> 239 us).
constexpr int FEW = 16;
constexpr int SHORT = 256;             // tokens of such a unit up to which a wavefront may take it alone
constexpr float CACHED = 64 << 20;     // bytes of keys and values up to which they may be in the last cache
constexpr int STEP = 64;               // tokens of a step
constexpr int TARGET = 512;            // pieces that the work is cut into at most, units' last ones apart
constexpr int TARGET_FEW = 2048;       // and those of units of few queries, whose sums take little room
constexpr int LEAST = 256, ENOUGH = 1024;   // tokens of a piece; where there are enough tiles without them
constexpr int GROUPS = DZ_PREFIX_GROUPS;

struct Unit {
  int tok0, ntok;                      // its queries' tokens
  int k0, n;                           // tokens seen: k0 .. n - 1 (by the last of its queries)
  int np, tiles;                       // pieces, tiles
  int row, pref;                       // whose table; of a row: its group's unit, or -1
  long long part;                      // records of its sums, or -1: it has one piece, and nothing else to join
  int causal, pad;
};
// What the join needs of a row, its group's part of it among that.
struct Row {
  int tok0, ntok, n, np;
  long long part, pre_part;
  int pre_tok0, pre_ntok, pre_np, pad;
};
struct Item {
  Unit unit;
  int tile, piece, pad[2];
};

struct PrefixParams {
  const char *q, *k, *v;
  const int *tables, *lengths, *starts, *groups, *prefixes;
  uint16_t* out;
  unsigned* status;
  int* head;                           // [0]: how many items there are, [1]: whether keys and values are more than
                                       // the caches keep; [3]: whether no row has any tokens, as what says so does not fit; [4]: items of short
                                       // units, in a list from the end, and [5] how many of them a workgroup takes; [6]: whether outputs are
                                       // left to the join
  Unit* units;                         // the groups'
  Row* row;                            // the rows'
  Item* items;
  float* parts;                        // records of dim + 4 floats: values, maximum, sum
  long long q_row, q_head, k_page, k_head, k_token, v_page, v_head, v_token, out_row, out_head, table_row;   // bytes; out, table: elements
  long long room_parts;
  unsigned num_pages;
  int tokens, rows, ngroups, heads, kv_heads, share, dim, shift, pages_per_row, room_items, near;
  unsigned line;                       // workgroups of a line of the grid
  float scale;
};

__device__ __forceinline__ int tiles_for(const PrefixParams& P, int tokens) { return (int)(((long long)tokens * P.share + ROWS - 1) / ROWS); }

// The last i in [0, n) with at[i] <= x, or -1.
template <typename T>
__device__ __forceinline__ int last_upto(const T* at, int n, T x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= x)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo - 1;
}

// The plan, as N threads of a workgroup make it together.  KEPT: rows and groups together are no more than these, and what is known of them stays in
// LDS.  The code runs once and from memory: what it need not do is left out of it.
template <int N, bool KEPT>
struct PlanRoom {
  static constexpr int G = KEPT ? N : GROUPS;
  int first[G + 1], cut[G], leader[G], alone[G];       // of groups: rows, prefix, row whose table, tiles apart
  int length[KEPT ? N : 1], start[KEPT ? N + 1 : 1];
  long long wave_parts[N / 64];
  int wave_items[N / 64], wave_shorts[N / 64];
  float wave_work[N / 64], wave_few[N / 64], wave_tiles[N / 64];
};

template <int N, bool KEPT>
struct Planner {
  const PrefixParams& P;
  PlanRoom<N, KEPT>& S;
  const int tid, lane, wave, room;
  int rows, groups;                    // that count
  int each, each_few;                  // tokens of a piece
  bool once;                           // keys and values are more than the caches keep
  int items, shorts;                   // in front of the round of units that `place` is at
  long long parts;

  __device__ __forceinline__ Planner(const PrefixParams& p, PlanRoom<N, KEPT>& s)
      : P(p), S(s), tid(threadIdx.x), lane(tid & 63), wave(tid >> 6), room(p.pages_per_row << p.shift), items(0), shorts(0), parts(0) {}

  __device__ __forceinline__ int length_of(int r) const { return KEPT ? S.length[r] : max(0, min(P.lengths[r], room)); }
  __device__ __forceinline__ int start_of(int r) const { return KEPT ? (P.rows ? S.start[r] : 0) : P.starts ? P.starts[r] : r; }
  __device__ __forceinline__ int count_of(int r) const { return start_of(r + 1) - start_of(r); }
  __device__ __forceinline__ int group_of(int r) const {
    const int g = groups ? last_upto(S.first, groups, r) : -1;
    return g >= 0 && r < S.first[g + 1] ? g : -1;
  }

  // Checks what the device alone knows and finds the prefixes that are taken apart from their rows.
  __device__ __forceinline__ void begin() {
    int bad = 0, bad_groups = 0, beyond = 0;
    int group[3] = {0, 0, 0};          // (asked for together with the rows')
    if (tid < P.ngroups) group[0] = P.groups[tid], group[1] = P.groups[tid + 1], group[2] = P.prefixes[tid];
    for (int r = tid; r < P.rows; r += N) {
      const int n = P.lengths[r], a = P.starts ? P.starts[r] : r, b = P.starts ? P.starts[r + 1] : r + 1;
      bad |= a < 0 || b < a || b > P.tokens;
      beyond |= n > room;
      if (KEPT) S.length[r] = max(0, min(n, room)), S.start[r] = a, S.start[r + 1] = b;      // (neighbours write the same)
    }
    for (int g = tid; g < P.ngroups; g += N) {
      if (g >= N) group[0] = P.groups[g], group[1] = P.groups[g + 1], group[2] = P.prefixes[g];
      const int a = group[0], b = group[1];
      bad_groups |= a < 0 || b < a || b > P.rows;
      S.first[g] = a, S.first[g + 1] = b;
      S.cut[g] = min(group[2], room);
      S.leader[g] = P.rows;
      S.alone[g] = 0;
    }
    if (beyond) atomicOr(P.status, 4u);
    bad = __syncthreads_or(bad);
    if (P.ngroups) bad_groups = __syncthreads_or(bad_groups);
    if ((bad || bad_groups) && tid == 0) atomicOr(P.status, 4u);
    rows = bad ? 0 : P.rows, groups = bad || bad_groups ? 0 : P.ngroups;
    if (!groups) return;
    // a prefix ends where the first of its rows' new tokens sees no more of it
    for (int r = tid; r < rows; r += N) {
      const int g = group_of(r), n = length_of(r), c = count_of(r);
      if (g >= 0 && n > 0 && c > 0) {
        atomicMin(&S.cut[g], max(0, n - c + 1));
        atomicMin(&S.leader[g], r);
        atomicAdd(&S.alone[g], tiles_for(P, c));
      }
    }
    __syncthreads();
    // and is taken apart from the rows only where that spares tiles
    for (int g = tid; g < groups; g += N) {
      const int tokens = start_of(S.first[g + 1]) - start_of(S.first[g]);
      if (S.cut[g] <= 0 || S.leader[g] >= rows || tiles_for(P, tokens) >= S.alone[g]) S.cut[g] = 0;
    }
    __syncthreads();
  }

  __device__ __forceinline__ int units() const { return groups + rows; }

  __device__ __forceinline__ Unit unit_of(int u) const {
    Unit x = {0, 0, 0, 0, 0, 0, 0, -1, -1, 0, 0};
    if (u < groups) {
      if (S.cut[u]) {
        x.tok0 = start_of(S.first[u]);
        x.ntok = start_of(S.first[u + 1]) - x.tok0;
        x.n = S.cut[u];
        x.row = S.leader[u];
      }
    } else if (u < units()) {
      const int r = u - groups, g = group_of(r);
      x.tok0 = start_of(r);
      x.ntok = count_of(r);
      x.n = length_of(r);
      x.row = r;
      x.causal = 1;
      if (g >= 0 && S.cut[g] && x.n > 0 && x.ntok > 0) {
        x.k0 = S.cut[g];
        x.pref = g;
      }
    }
    x.tiles = tiles_for(P, x.ntok);
    return x;
  }

  __device__ __forceinline__ bool few(const Unit& x) const { return (long long)x.ntok * P.share <= FEW; }

  // How long pieces are: tokens times tiles, over the pieces aimed at.  x: this thread's unit, of the last N of them.
  __device__ __forceinline__ void lengths_of_pieces(Unit& x) {
    float all = 0.0f, of_few = 0.0f, tiles = 0.0f;
#pragma unroll 1
    for (int u0 = 0; u0 < units(); u0 += N) {
      x = unit_of(u0 + tid);
      const float w = (float)x.tiles * (float)(x.n - x.k0);
      all += w;
      if (few(x))
        of_few += w;
      else if (x.n > x.k0)
        tiles += (float)x.tiles;
    }
    all = scan_add(all), of_few = scan_add(of_few), tiles = scan_add(tiles);
    if (lane == 63) S.wave_work[wave] = all, S.wave_few[wave] = of_few, S.wave_tiles[wave] = tiles;
    __syncthreads();
    all = of_few = tiles = 0.0f;
#pragma unroll 2
    for (int w = 0; w < N / 64; ++w) all += S.wave_work[w], of_few += S.wave_few[w], tiles += S.wave_tiles[w];
    // in whole steps (sums above 2^24 are rounded: a piece is a little longer)
    auto each_of = [&](float work, int target, int least) {
      const float want = ceilf(work * 1.0001f * (float)P.kv_heads * (1.0f / (float)target) * (1.0f / STEP));
      return STEP * (int)fminf(fmaxf(want, (float)(least / STEP)), (float)(1 << 24));
    };
    // (whole tiles that are enough by themselves are spared the join)
    each = each_of(all, TARGET, tiles * (float)P.kv_heads >= TARGET / 2 ? ENOUGH : LEAST);
    each_few = min(each, each_of(of_few, TARGET_FEW, LEAST));
    once = all * (float)P.kv_heads * (4.0f * (float)P.dim) > CACHED;
  }

  __device__ __forceinline__ int pieces_of(const Unit& x) const {
    const int most = few(x) ? each_few : each;
    return x.tiles ? (x.n - x.k0 + most - 1) / most : 0;
  }

  // (queries that see as much as each other: 32 rows of up to 200 tokens of their own 34 -> 32 us.  Of several new tokens it goes by how unlike the rows are: 48 of up
  // to 333 tokens of their own 34 -> 42, 64 of 3 behind their 200 each 55 -> 58, 32 of 128 31 -> 31, but 64 of 2 of 64 37 -> 33, 128 of 32 57 -> 38)
  __device__ __forceinline__ bool is_short(const Unit& x) const { return few(x) && x.np == 1 && x.n - x.k0 <= SHORT && (x.ntok == 1 || !x.causal); }

  // The pieces of this thread's unit, of the next N of them: its items (those of short units in a list of their own) end at what is returned, its
  // records begin at x.part.
  __device__ __forceinline__ int place(Unit& x) {
    x.np = pieces_of(x);
    const bool apart = is_short(x);
    const int mine = apart ? 0 : x.tiles * x.np, mine_short = apart;
    const long long records = x.np > 1 || x.k0 > 0 || !x.causal ? (long long)x.np * x.ntok * P.heads : 0;
    const int upto = scan_add(mine), shorts_upto = scan_add(mine_short);
    long long records_upto = records;
    if (KEPT) {                        // (fewer than 2^31)
      records_upto = scan_add((int)records);
    } else {
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const long long y = __shfl_up(records_upto, d);
        if (lane >= d) records_upto += y;
      }
    }
    if (lane == 63) S.wave_items[wave] = upto, S.wave_shorts[wave] = shorts_upto, S.wave_parts[wave] = records_upto;
    __syncthreads();
    int before = items, shorts_before = shorts;
    long long parts_before = parts;
#pragma unroll 2
    for (int w = 0; w < N / 64; ++w) {
      if (w < wave) before += S.wave_items[w], shorts_before += S.wave_shorts[w], parts_before += S.wave_parts[w];
      items += S.wave_items[w], shorts += S.wave_shorts[w], parts += S.wave_parts[w];
    }
    if (records) x.part = parts_before + records_upto - records;
    const int at = P.room_items - shorts_before - shorts_upto;
    if (apart && at >= 0) P.items[at] = Item{x, 0, 0, {0, 0}};             // (from the list's end)
    return before + upto;
  }

  __device__ __forceinline__ bool fits() const { return items + shorts <= P.room_items && parts <= P.room_parts; }

  // What others need to know of all of it.
  __device__ __forceinline__ void tell() const {
    if (!fits()) atomicOr(P.status, 4u);
    P.head[0] = fits() ? items : 0;
    P.head[1] = once;
    P.head[3] = rows < P.rows || !fits();
    P.head[4] = fits() ? shorts : 0;
    P.head[5] = (long long)shorts * P.kv_heads > TARGET ? 4 : 1;
  }
};

// One workgroup.
template <int N, bool KEPT>
__global__ __launch_bounds__(N) void dz_prefix_plan_kernel(const PrefixParams P) {
  __shared__ PlanRoom<N, KEPT> room;
  __shared__ int upto[N], of_groups;
  __shared__ __attribute__((aligned(16))) Unit made[N];        // a round's units
  Planner<N, KEPT> plan(P, room);
  const int tid = threadIdx.x;
  int unfinished = 0;                    // whether anything is left to the join
  plan.begin();
  Unit x = {0, 0, 0, 0, 0, 0, 0, -1, -1, 0, 0};
  plan.lengths_of_pieces(x);
  for (int u0 = 0; u0 < plan.units(); u0 += N) {
    const int u = u0 + tid, begin = plan.items;
    if (!KEPT) x = plan.unit_of(u);
    upto[tid] = plan.place(x);
    made[tid] = x;
    if (!KEPT && u < plan.groups) P.units[u] = x;
    // Items in the order in which they are taken: prefixes' pieces, which keep the matrix cores busy, and rows' own, which wait for memory, a compute
    // unit each of both, then the others (where rows and groups are few).
    if (u == plan.groups - 1) of_groups = upto[tid];
    __syncthreads();
    if (u >= plan.groups && u < plan.units()) {
      unfinished |= x.ntok > 0 && (x.np != 1 || x.part >= 0);
      Row row = {x.tok0, x.ntok, x.n, x.np, x.part, -1, 0, 0, 0, 0};
      if (x.pref >= 0) {
        const Unit pre = KEPT ? made[x.pref] : P.units[x.pref];
        row.pre_part = pre.part, row.pre_tok0 = pre.tok0, row.pre_ntok = pre.ntok, row.pre_np = pre.np;
      }
      P.row[u - plan.groups] = row;
    }
    const int shared = KEPT && plan.groups ? of_groups : 0, round = max(1, 256 / P.kv_heads), pairs = min(shared, plan.items - shared) / round;
    auto place_of = [&](int i) {
      if (!pairs) return i;
      const int k = i < shared ? i : i - shared;
      return k < pairs * round ? k / round * 2 * round + (i < shared ? 0 : round) + k % round : i < shared ? i + pairs * round : i;
    };
    for (int i = begin + tid; i < plan.items; i += N) {
      const int at = last_upto(upto, N, i) + 1;                // the first unit that ends behind i
      const Unit& y = made[at];
      const int tiles = y.tiles, rest = i - (upto[at] - tiles * y.np);
      // tiles that share keys and values next to each other; of a row's, those that see most first
      const int to = place_of(i);
      if (to < P.room_items) P.items[to] = Item{y, tiles - 1 - rest % tiles, rest / tiles, {0, 0}};
    }
    if (KEPT) break;
    __syncthreads();
  }
  unfinished = __syncthreads_or(unfinished);
  if (tid == 0) {
    plan.tell();
    P.head[6] = unfinished || !plan.fits() || plan.rows < P.rows || !P.rows || plan.start_of(0) > 0 || plan.start_of(P.rows) < P.tokens;
  }
}

// Requests of 16 bytes of a token's row lie in LDS in the order c ^ swizzled(token): 8 tokens' one request, which a key's operand reads at
// a time, and 4 tokens' two, which a transposing read of values does, are then in banks of their own.
template <int KC>
__device__ __forceinline__ int swizzled(int token) {
  return KC % 4 == 0 ? 2 * (token & 7) : KC % 2 == 0 ? 2 * (token >> 1 & 3) : 2 * (token >> 2 & 1);
}

// A piece of a unit of up to FEW queries, with keys and values in registers: a wavefront walks it alone, or four a quarter of its tokens each, and
// join their sums.
template <int KC, bool FULL, bool BF>
__device__ __forceinline__ void few_queries(const PrefixParams& P, const Unit& U, int piece, int kvh, int lo, int hi, bool once, bool alone, float* lds) {
  typedef Type<BF> Ty;
  typedef typename Ty::v8 v8;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const int queries = U.ntok * P.share;
  auto limit_of = [&](int x) { return U.causal ? max(U.n - (U.ntok - 1 - x / P.share), 0) : U.n; };
  Walk<KC, FULL, BF, true> walk;
  const int mine = min(col, queries - 1);
  const char* from = P.q + (U.tok0 + mine / P.share) * P.q_row + (kvh * P.share + mine % P.share) * P.q_head;
#pragma unroll
  for (int c = 0; c < KC; ++c) {
    u4_t w = {0, 0, 0, 0};
    if (col < queries && 32 * c + 8 * g < P.dim) w = *(const u4_t*)(from + (32 * c + 8 * g) * 2);
    walk.q[c] = __builtin_bit_cast(v8, w);
  }
  const int* table = P.tables + U.row * P.table_row;
  const int tile0 = lo / TILE, tiles = lo < hi ? (hi + TILE - 1) / TILE - tile0 : 0;
  const int t0 = alone ? tile0 : tile0 + tiles * wave / 4, t1 = alone ? tile0 + tiles : tile0 + tiles * (wave + 1) / 4, limit = min(limit_of(mine), hi), seen_by_all = min(limit_of(0), hi);
  if (seen_by_all < hi)
    walk.template run<false, true>(P, table, kvh, lo, hi, t0, t1, limit, seen_by_all);
  else if (once)
    walk.template run<true, false>(P, table, kvh, lo, hi, t0, t1, hi, hi);
  else
    walk.template run<false, false>(P, table, kvh, lo, hi, t0, t1, hi, hi);
  float sum = walk.sum;
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  const int ld = P.dim + 4;
  if (alone) {
    if (col >= queries) return;
    float* record = P.parts + (U.part + ((long long)piece * P.kv_heads + kvh) * queries + col) * ld;
    uint16_t* out = P.out + (U.tok0 + mine / P.share) * P.out_row + (kvh * P.share + mine % P.share) * P.out_head;
    const float part = limit_of(mine) > 0 ? 1.0f / sum : 0.0f;
#pragma unroll
    for (int b = 0; b < walk.NB; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 128 * b + 8 * (4 * g + i);
        if (d >= P.dim) continue;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = walk.acc[8 * b + j][i];
        if (U.part >= 0) {
          *(f4_t*)(record + d) = f4_t{x[0], x[1], x[2], x[3]};
          *(f4_t*)(record + d + 4) = f4_t{x[4], x[5], x[6], x[7]};
        } else {
          u4_t w;
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = (unsigned)Ty::round(x[2 * j] * part) | (unsigned)Ty::round(x[2 * j + 1] * part) << 16;
          *(u4_t*)(out + d) = w;
        }
      }
    if (U.part >= 0 && g == 0) *(f2_t*)(record + P.dim) = f2_t{walk.top, sum};
    return;
  }
  float *sums = lds + wave * queries * ld, *stat = lds + 4 * FEW * ld;       // [wave][query][dim], then maxima and sums
  if (col < queries) {
#pragma unroll
    for (int b = 0; b < walk.NB; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 128 * b + 8 * (4 * g + i);
        if (d < P.dim) {
          *(f4_t*)(sums + col * ld + d) = f4_t{walk.acc[8 * b][i], walk.acc[8 * b + 1][i], walk.acc[8 * b + 2][i], walk.acc[8 * b + 3][i]};
          *(f4_t*)(sums + col * ld + d + 4) = f4_t{walk.acc[8 * b + 4][i], walk.acc[8 * b + 5][i], walk.acc[8 * b + 6][i], walk.acc[8 * b + 7][i]};
        }
      }
    if (g == 0) *(f2_t*)(stat + (wave * FEW + col) * 2) = f2_t{walk.top, sum};
  }
  __syncthreads();
  const int quads = P.dim / 4;
  for (int x = threadIdx.x; x < queries * quads; x += 256) {
    const int y = x / quads, d = x % quads * 4;
    float m = -INFINITY, l = 0.0f;
    f4_t o = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < 4; ++w) m = fmaxf(m, stat[(w * FEW + y) * 2]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = weight_of(stat[(w * FEW + y) * 2], m);
      l += stat[(w * FEW + y) * 2 + 1] * f;
      o += *(const f4_t*)(lds + (w * queries + y) * ld + d) * f;
    }
    if (U.part >= 0) {
      float* record = P.parts + (U.part + ((long long)piece * P.kv_heads + kvh) * queries + y) * ld;
      *(f4_t*)(record + d) = o;
      if (d == 0) *(f2_t*)(record + P.dim) = f2_t{m, l};
    } else {
      o = limit_of(y) > 0 ? o * (1.0f / l) : f4_t{0, 0, 0, 0};
      const u2_t w = {(unsigned)Ty::round(o[0]) | (unsigned)Ty::round(o[1]) << 16, (unsigned)Ty::round(o[2]) | (unsigned)Ty::round(o[3]) << 16};
      *(u2_t*)(P.out + (U.tok0 + y / P.share) * P.out_row + (kvh * P.share + y % P.share) * P.out_head + d) = w;
    }
  }
}

template <int KC, bool FULL, bool BF>
__global__ __launch_bounds__(256, KC <= 4 ? 2 : 1) void dz_prefix_kernel(const PrefixParams P) {
  typedef Type<BF> Ty;
  typedef typename Ty::v8 v8;
  constexpr int ROW = KC * 64;                         // bytes of a token in LDS
  constexpr int HALF = STEP * ROW, STAGE = 2 * HALF;   // keys, values
  constexpr unsigned BAD = BF ? 0x7f80u : 0x7c00u;     // exponent of what is not finite
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const unsigned id = blockIdx.y * P.line + blockIdx.x;
  const int turn = id / P.kv_heads, kvh = id % P.kv_heads;
  if (turn >= P.room_items) return;    // (behind a grid's last line)
  Item item = P.items[turn];           // (asked for together with what says whether it is one; there are as many places as turns)
  const int all = P.head[0], shorts = P.head[4], together = P.head[5];
  const bool once = P.head[1] != 0, is_short = turn >= all;
  if (is_short) {
    // four at once, where there are many of them: each waits by itself for what it asks for
    const int at = (turn - all) * together + (together > 1 ? wave : 0);
    if (at >= shorts) return;
    item = P.items[P.room_items - 1 - at];
  }
  const Unit U = item.unit;
  const int tile = item.tile, piece = item.piece;
  const int queries = U.ntok * P.share, x0 = tile * ROWS, in_tile = min(ROWS, queries - x0);
  auto limit_of = [&](int x) { return U.causal ? max(U.n - (U.ntok - 1 - x / P.share), 0) : U.n; };      // tokens that query x sees
  const int end = max(limit_of(x0 + in_tile - 1), U.k0);
  const long long len = end - U.k0;
  // pieces meet between steps, and steps lie in whole pages or hold whole pages
  auto bound = [&](int p) { return p == U.np ? end : p == 0 ? U.k0 : max(U.k0, (U.k0 + (int)(len * p / U.np)) & ~(STEP - 1)); };
  const int lo = bound(piece), hi = bound(piece + 1), begin = lo < hi ? lo & ~(STEP - 1) : hi;

  if (queries <= FEW) {
    few_queries<KC, FULL, BF>(P, U, piece, kvh, lo, hi, once, is_short && together > 1, (float*)lds);
    return;
  }
  const int last_page = (hi - 1) >> P.shift, in_page = (1 << P.shift) - 1;
  const int* table = P.tables + U.row * P.table_row;
  int page0 = begin >> P.shift;        // of the 64 page numbers that the lanes hold
  auto fetch = [&](int base) {
    const int at = base + lane;
    unsigned id = at <= last_page && begin < hi ? (unsigned)table[at] : 0u;
    if (id >= P.num_pages) {
      atomicOr(P.status, 4u);
      id = 0;
    }
    return id;
  };
  unsigned ids = fetch(page0), next_ids = fetch(page0 + 64);

  const int per_row = P.dim / 8;       // requests of a token's row
  if (!FULL) {                         // behind the head's end: zeros, which meet the queries' zeros
    for (int i = threadIdx.x; i < 2 * STAGE / 16; i += 256) *(u4_t*)(lds + 16 * i) = u4_t{0, 0, 0, 0};
    __syncthreads();
  }
  // A wavefront brings in 16 tokens of each step; request i of a lane is for token (64 i + lane) / (4 KC) of them.
  struct Request {
    int token, at;                     // bytes into the token's row, -1: behind the head's end
  };
  auto request = [&](int i, int of_lane) __attribute__((always_inline)) {
    const int token = (64 * i + of_lane) / (4 * KC), c = (64 * i + of_lane) % (4 * KC) ^ swizzled<KC>(token);
    return Request{token, FULL || c < per_row ? 16 * c : -1};
  };
  auto bring = [&](const char* from, char* to) __attribute__((always_inline)) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
  };
  auto issue = [&](int s, int buf) __attribute__((always_inline)) {
    if (((min(s + STEP, hi) - 1) >> P.shift) >= page0 + 64) {
      ids = next_ids;
      page0 += 64;
      next_ids = fetch(page0 + 64);
    }
    char* to = lds + buf * STAGE + wave * 16 * ROW;
    const int t0 = s + 16 * wave;
    int of_lane = lane;
    if (KC == 8) asm volatile("" : "+v"(of_lane));         // (worked out anew for each step: no registers to keep it)
    if (P.near && t0 + 16 <= hi) {     // all of one page: its place is the wavefront's
      const long long id = __builtin_amdgcn_readlane(ids, (t0 >> P.shift) - page0);
      const char* k = P.k + id * P.k_page + kvh * P.k_head + (t0 & in_page) * P.k_token;
      const char* v = P.v + id * P.v_page + kvh * P.v_head + (t0 & in_page) * P.v_token;
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        const Request r = request(i, of_lane);
        if (FULL || r.at >= 0) {
          bring(k + (unsigned)(r.token * (unsigned)P.k_token + r.at), to + i * 1024);
          bring(v + (unsigned)(r.token * (unsigned)P.v_token + r.at), to + HALF + i * 1024);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        const Request r = request(i, of_lane);
        const int t = min(t0 + r.token, hi - 1);           // (behind the end: the last one again)
        const unsigned id = __shfl(ids, (t >> P.shift) - page0);
        if (FULL || r.at >= 0) {
          bring(P.k + id * P.k_page + kvh * P.k_head + (t & in_page) * P.k_token + r.at, to + i * 1024);
          bring(P.v + id * P.v_page + kvh * P.v_head + (t & in_page) * P.v_token + r.at, to + HALF + i * 1024);
        }
      }
    }
  };
  if (begin < hi) issue(begin, 0);

  auto work = [&](auto cols) __attribute__((always_inline)) {
    constexpr int NC = decltype(cols)::value;          // tiles of 16 queries of a wavefront
    constexpr bool TWO = NC == 1;                      // weights held in two values
    const int mine = wave * 16 * NC;                   // its first query in the tile
    const bool active = mine < in_tile;
    v8 q[NC][KC];
    int lim[NC];
    f4_t acc[NC][2 * KC];
    float top[NC], ref[NC], by[NC];    // maximum; a weight is 2^(score by + ref)
    f4_t sum[NC];                      // of the weights as they are rounded (a product with ones: what rounding does to a large weight is gone when it is divided by)
    v8 ones;
#pragma unroll
    for (int e = 0; e < 8; ++e) ones[e] = Ty::one(1.0f);
    const float scale = fabsf(P.scale);
    bool far = false;                  // of any query's maximum
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int x = mine + 16 * n + col, xx = x0 + min(x, in_tile - 1);
      const int token = U.tok0 + xx / P.share, head = kvh * P.share + xx % P.share;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        u4_t w = {0, 0, 0, 0};
        if (x < in_tile && (FULL || 32 * c + 8 * g < P.dim)) w = *(const u4_t*)(P.q + token * P.q_row + head * P.q_head + (32 * c + 8 * g) * 2);
        q[n][c] = __builtin_bit_cast(v8, w);
      }
      if (P.scale < 0.0f) {            // (the largest score is that of the largest product)
#pragma unroll
        for (int c = 0; c < KC; ++c) q[n][c] = -q[n][c];
      }
      lim[n] = min(limit_of(xx), hi);
      top[n] = -INFINITY, ref[n] = 0.0f, by[n] = scale, sum[n] = f4_t{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 2 * KC; ++j) acc[n][j] = f4_t{0, 0, 0, 0};
    }
    const int seen_by_all = min(limit_of(x0 + min(mine, in_tile - 1)), hi), seen_by_last = min(limit_of(x0 + min(mine + 16 * NC, in_tile) - 1), hi);

    auto step = [&](int s, const char* at) __attribute__((always_inline)) {
      const bool edge = s + STEP > seen_by_all || s < lo;
      const char* keys = at + col * ROW;
      const int turn_k = swizzled<KC>(col);
      f4_t sc[NC][4];
      constexpr bool AHEAD = KC <= 6;  // (heads of 256: no registers for it)
      v8 kw[2][KC];
      auto load_keys = [&](int a) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < KC; ++c) kw[a & 1][c] = *(const v8*)(keys + a * 16 * ROW + ((4 * c + g) ^ turn_k) * 16);
      };
      load_keys(0);
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        if (!AHEAD && a) load_keys(a);
        if (AHEAD && a < 3) load_keys(a + 1);
#pragma unroll
        for (int n = 0; n < NC; ++n) sc[n][a] = f4_t{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
          for (int n = 0; n < NC; ++n) sc[n][a] = Ty::mma(kw[a & 1][c], q[n][c], sc[n][a]);
        __builtin_amdgcn_sched_barrier(0);
      }
      // a transposing read: lanes of a row of 16 name 4 tokens' 16 dims, and each gets one dim of the four
      const char* values = at + HALF + (4 * g + (col >> 2)) * ROW + (col & 1) * 8;
      const int turn_v = swizzled<KC>(4 * g + (col >> 2));
      s8_t vw[2][4];                   // of two groups of 32 dims, for 2 x 32 tokens each
      auto load_values = [&](int jj) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int j = 2 * jj + (x >> 1), h = x & 1;
          const char* from = values + 2 * h * 16 * ROW + ((2 * j + (col >> 1 & 1)) ^ turn_v) * 16;
          const s4_t a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4_t*)from);
          const s4_t a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4_t*)(from + 16 * ROW));
          vw[jj & 1][x] = s8_t{a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]};
        }
      };
      bool spoilt = false;             // values that are not finite, where some queries do not see all tokens
      auto hidden = [&](int n, int e) { return s + 16 * (e >> 2) + 4 * g + (e & 3) >= lim[n] || s + 16 * (e >> 2) + 4 * g + (e & 3) < lo; };
      if (edge) {
        unsigned found = 0;
#pragma unroll 4
        for (int i = lane; i < HALF / 16; i += 64) {
          const u4_t w = *(const u4_t*)(at + HALF + 16 * i);
#pragma unroll
          for (int e = 0; e < 4; ++e) found |= (w[e] & (BAD | BAD << 16)) + ((0x8000u - BAD) | (0x8000u - BAD) << 16);
        }
        spoilt = __any(found & 0x80008000u);
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (hidden(n, e)) sc[n][e >> 2][e & 3] = -INFINITY;
      }
      load_values(0);
      v8 p[NC][2], low[TWO ? NC : 1][2];
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        float most = sc[n][0][0];
#pragma unroll
        for (int e = 1; e < 16; ++e) most = fmaxf(most, sc[n][e >> 2][e & 3]);
        most *= scale;
        // the reference moves only where a score is more than twice above it
        if (__any(most > top[n] + 1.0f) || far) {
          most = fmaxf(most, __shfl_xor(most, 16));
          most = fmaxf(most, __shfl_xor(most, 32));
          // (each query's by its own scores: another's change nothing of it)
          const float up = most > top[n] + 1.0f ? most : top[n];
          const float f = top[n] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top[n] - up);
          top[n] = up;
          sum[n] *= f;
#pragma unroll
          for (int j = 0; j < 2 * KC; ++j) acc[n][j] *= f;
          ref[n] = up == -INFINITY ? 0.0f : Ty::BIAS - up, by[n] = scale;
          far |= __any(is_far(up));
          if (__builtin_expect(far, 0) && is_far(up)) {
            // (the maximum is a rounded product: the scores, too, before it is taken from them)
#pragma clang fp contract(off)
            by[n] = 1.0f, ref[n] = Ty::BIAS;
#pragma unroll
            for (int e = 0; e < 16; ++e) sc[n][e >> 2][e & 3] = sc[n][e >> 2][e & 3] * scale - up;
          }
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[n][e >> 2][e & 3], by[n], ref[n]));
          if (TWO) {
            // the second is above zero where the weight is, so that infinity times it is no NaN: all weights are 1 + MORE times what they are
            const auto high = Ty::cut(w);
            p[n][e >> 3][e & 7] = high;
            low[n][e >> 3][e & 7] = Ty::one(__builtin_fmaf(w, 1.0f + Ty::MORE, -(float)high));
          } else {
            p[n][e >> 3][e & 7] = Ty::one(w);
          }
        }
        sum[n] = Ty::mma(ones, p[n][1], Ty::mma(ones, p[n][0], sum[n]));
        if (TWO) sum[n] = Ty::mma(ones, low[n][1], Ty::mma(ones, low[n][0], sum[n]));
      }
      if (__builtin_expect(spoilt, 0)) {
        // a weight of 0 would take what is not finite to queries that do not see it: left out of the products, and added where it is seen
        int quad = 4 * g;
        asm volatile("" : "+v"(quad));                     // (addresses of this rare path are not worth registers all along)
#pragma unroll 1
        for (int t = 0; t < STEP; ++t)
#pragma unroll
          for (int j = 0; j < 2 * KC; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint16_t w = *(const uint16_t*)(at + HALF + t * ROW + ((2 * j + (quad >> 3)) ^ swizzled<KC>(t)) * 16 + ((quad & 7) + i) * 2);
              const float y = BF ? __builtin_bit_cast(float, (unsigned)w << 16) : (float)__builtin_bit_cast(_Float16, w);
#pragma unroll
              for (int n = 0; n < NC; ++n) acc[n][j][i] += (w & BAD) == BAD && s + t < lim[n] && s + t >= lo ? y : 0.0f;
            }
      }
#pragma unroll
      for (int jj = 0; jj < KC; ++jj) {
        if (jj + 1 < KC) load_values(jj + 1);
        if (__builtin_expect(spoilt, 0)) {
#pragma unroll
          for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (((unsigned)vw[jj & 1][x][e] & BAD) == BAD) vw[jj & 1][x][e] = 0;
        }
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int n = 0; n < NC; ++n)
            acc[n][2 * jj + (x >> 1)] = Ty::mma(__builtin_bit_cast(v8, vw[jj & 1][x]), p[n][x & 1], acc[n][2 * jj + (x >> 1)]);
        if (TWO) {
#pragma unroll
          for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int n = 0; n < NC; ++n)
              acc[n][2 * jj + (x >> 1)] = Ty::mma(__builtin_bit_cast(v8, vw[jj & 1][x]), low[n][x & 1], acc[n][2 * jj + (x >> 1)]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };

    int buf = 0;
    for (int s = begin; s < hi; s += STEP, buf ^= 1) {
      __builtin_amdgcn_s_waitcnt(0x0070);              // vmcnt(0) lgkmcnt(0): this wavefront's share of the step is in,
      __syncthreads();                                 // and the others'; no one reads the other buffer any more
      if (s + STEP < hi) issue(s + STEP, buf ^ 1);
      if (!active || s >= seen_by_last) continue;
      step(s, lds + buf * STAGE);
    }
    if (!active) return;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int x = mine + 16 * n + col;
      if (x >= in_tile) continue;
      const int xx = x0 + x;
      if (U.part >= 0) {
        // (other units' weights, which these are joined with, are what they are)
        constexpr float less = TWO ? 1.0f / (1.0f + Ty::MORE) : 1.0f;
        float* record = P.parts + (U.part + ((long long)piece * P.kv_heads + kvh) * queries + xx) * (P.dim + 4);
#pragma unroll
        for (int j = 0; j < 2 * KC; ++j)
          if (FULL || 16 * j + 4 * g < P.dim) *(f4_t*)(record + 16 * j + 4 * g) = acc[n][j] * less;
        if (g == 0) *(f2_t*)(record + P.dim) = f2_t{top[n], sum[n][0] * less};
      } else {
        uint16_t* to = P.out + (U.tok0 + xx / P.share) * P.out_row + (kvh * P.share + xx % P.share) * P.out_head;
        const bool sees = limit_of(xx) > 0;
        const float part = 1.0f / sum[n][0];
#pragma unroll
        for (int j = 0; j < 2 * KC; ++j) {
          const f4_t y = sees ? acc[n][j] * part : f4_t{0, 0, 0, 0};
          const u2_t w = {(unsigned)Ty::round(y[0]) | (unsigned)Ty::round(y[1]) << 16, (unsigned)Ty::round(y[2]) | (unsigned)Ty::round(y[3]) << 16};
          if (FULL || 16 * j + 4 * g < P.dim) *(u2_t*)(to + 16 * j + 4 * g) = w;
        }
      }
    }
  };
  if (in_tile > 64)
    work(std::integral_constant<int, 2>());
  else
    work(std::integral_constant<int, 1>());
}

// The pieces of a token's row's sums and of its group's joined, or zeros.  A thread takes four values of a head over every SLICES-th
// piece, four at once on their way; a workgroup takes 256 / SLICES such places, and every gridDim.y-th set of them.
template <int SLICES, bool BF>
__global__ __launch_bounds__(256) void dz_prefix_join_kernel(const PrefixParams P) {
  typedef Type<BF> Ty;
  constexpr int SPOTS = 256 / SLICES, AT_ONCE = 4;
  __shared__ float shared[SLICES > 1 ? 256 * 8 : 1];
  if (!P.head[6]) return;
  const bool none = P.head[3] != 0;
  for (int t = blockIdx.x; t < P.tokens; t += gridDim.x) {
    int row = t;
    if (P.starts) {
      __shared__ int found;
      if (P.rows <= 1024) {
        __syncthreads();
        if (threadIdx.x == 0) found = -1;
        __syncthreads();
        for (int r = threadIdx.x; r < P.rows; r += 256)
          if (P.starts[r] <= t && t < P.starts[r + 1]) found = r;
        __syncthreads();
        row = found;
      } else {
        row = last_upto(P.starts, P.rows, t);
        if (row >= 0 && t >= P.starts[row + 1]) row = -1;
      }
    }
    if (none) row = -1;
    Row own = {0, 0, 0, 0, -1, -1, 0, 0, 0, 0};
    bool sees = false;
    if (row >= 0) {
      own = P.row[row];
      sees = own.n - (own.ntok - 1 - (t - own.tok0)) > 0;
    }
    if (sees && own.np == 1 && own.part < 0) continue;    // (stored already)
    const int quads = P.dim / 4, places = P.heads * quads;
    const long long stride = P.dim + 4, pre_queries = (long long)own.pre_ntok * P.share, own_queries = (long long)own.ntok * P.share;
    const int pieces = sees ? own.pre_np + own.np : 0;
    const int slice = threadIdx.x / SPOTS;
    for (int x0 = blockIdx.y * SPOTS; x0 < places; x0 += gridDim.y * SPOTS) {
      const int x = x0 + threadIdx.x % SPOTS, h = min(x, places - 1) / quads, d = x % quads * 4, kvh = h / P.share, hs = h % P.share;
      const float* from_pre = P.parts + (own.pre_part + kvh * pre_queries + (long long)(t - own.pre_tok0) * P.share + hs) * stride;
      const float* from_own = P.parts + (own.part + kvh * own_queries + (long long)(t - own.tok0) * P.share + hs) * stride;
      float m = -INFINITY, l = 0.0f;
      f4_t o = {0, 0, 0, 0};
      for (int p0 = slice; p0 < pieces; p0 += SLICES * AT_ONCE) {
        f4_t w[AT_ONCE];
        f2_t ml[AT_ONCE];
        float up = m;
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
          const int p = min(p0 + i * SLICES, pieces - 1);
          const float* record = p < own.pre_np ? from_pre + p * (P.kv_heads * pre_queries * stride) : from_own + (p - own.pre_np) * (P.kv_heads * own_queries * stride);
          w[i] = *(const f4_t*)(record + d);
          ml[i] = *(const f2_t*)(record + P.dim);
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
          if (p0 + i * SLICES >= pieces) ml[i] = f2_t{-INFINITY, 0.0f}, w[i] = f4_t{0, 0, 0, 0};       // (the last one a second time)
          up = fmaxf(up, ml[i][0]);
        }
        const float f = weight_of(m, up);
        l *= f, o *= f, m = up;
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
          const float fs = weight_of(ml[i][0], up);
          l += ml[i][1] * fs;
          o += w[i] * fs;
        }
      }
      if constexpr (SLICES > 1) {
        float* mine = shared + threadIdx.x * 8;
        *(f4_t*)mine = o;
        *(f2_t*)(mine + 4) = f2_t{m, l};
        __syncthreads();
        if (slice == 0) {
          const float* all = shared + threadIdx.x * 8;
          for (int c = 1; c < SLICES; ++c) m = fmaxf(m, all[c * SPOTS * 8 + 4]);
          l = 0.0f, o = f4_t{0, 0, 0, 0};
          for (int c = 0; c < SLICES; ++c) {
            const float f = weight_of(all[c * SPOTS * 8 + 4], m);
            l += all[c * SPOTS * 8 + 5] * f;
            o += *(const f4_t*)(all + c * SPOTS * 8) * f;
          }
        }
        __syncthreads();
      }
      if (slice == 0 && x < places) {
        const f4_t y = sees ? o * (1.0f / l) : f4_t{0, 0, 0, 0};
        const u2_t w = {(unsigned)Ty::round(y[0]) | (unsigned)Ty::round(y[1]) << 16, (unsigned)Ty::round(y[2]) | (unsigned)Ty::round(y[3]) << 16};
        *(u2_t*)(P.out + t * P.out_row + h * P.out_head + d) = w;
      }
    }
  }
}

typedef void (*kernel_t)(const PrefixParams);
inline int chunks_of(int dim) { return dim <= 64 ? 2 : dim <= 96 ? 3 : dim <= 128 ? 4 : dim <= 192 ? 6 : 8; }
template <int KC, bool BF>
kernel_t kernel_of(int dim) {
  return dim == 32 * KC ? dz_prefix_kernel<KC, true, BF> : dz_prefix_kernel<KC, false, BF>;
}
template <bool BF>
kernel_t kernel_for(int dim) {
  const int kc = chunks_of(dim);
  return kc == 2 ? kernel_of<2, BF>(dim) : kc == 3 ? kernel_of<3, BF>(dim) : kc == 4 ? kernel_of<4, BF>(dim)
         : kc == 6 ? kernel_of<6, BF>(dim) : kernel_of<8, BF>(dim);
}

inline bool shapes_fit(int tokens, int rows, int groups, int heads, int kv_heads, int dim, int page_size, int pages_per_row) {
  return tokens >= 0 && rows >= 0 && rows <= (1 << 20) && groups >= 0 && groups <= GROUPS && heads >= 1 && kv_heads >= 1 && heads <= 4096 &&
         heads % kv_heads == 0 && (long long)tokens * heads < (1ll << 31) && dim >= 8 && dim <= 256 && dim % 8 == 0 && page_size >= 8 &&
         page_size <= 1024 && (page_size & (page_size - 1)) == 0 && pages_per_row >= 0 && (long long)pages_per_row * page_size <= (1ll << 30);
}

// What a call's plan comes to at most.
struct Room {
  long long items, tiles, parts;       // items of one key head, in so many tiles; records
  size_t units_at, rows_at, items_at, parts_at, bytes;
};
inline Room room_of(int tokens, int rows, int groups, int heads, int kv_heads, int dim) {
  Room m;
  const long long queries = (long long)tokens * (heads / kv_heads), whole = (queries + ROWS - 1) / ROWS;
  const long long some = rows < tokens ? rows : tokens, both = groups ? 2 : 1;
  // a unit's tiles: the last one is not full; pieces: of those aimed at one more of each tile
  m.tiles = both * whole + some + (groups < tokens ? groups : tokens);
  m.items = m.tiles + (TARGET + TARGET_FEW) / kv_heads + 2;
  // Records: a unit in several pieces has one more than aimed at for each of its queries; in groups every query has one for its row and one for its group.
  // Units that are longer than a piece have fewer tiles together than there are pieces (a piece is as long as all tiles' tokens over the pieces
  // aimed at): of them no more than two times as many queries.
  const long long cut = 2 * ((long long)ROWS * (TARGET + kv_heads) + (long long)FEW * (TARGET_FEW + kv_heads));
  m.parts = (groups ? 2ll * tokens * heads : (long long)tokens * heads < cut ? (long long)tokens * heads : cut) + cut / 2;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  m.units_at = 256;
  m.rows_at = up(m.units_at + sizeof(Unit) * (size_t)groups);
  m.items_at = up(m.rows_at + sizeof(Row) * (size_t)rows);
  m.parts_at = up(m.items_at + sizeof(Item) * (size_t)m.items);
  m.bytes = m.parts_at + (size_t)m.parts * (dim + 4) * 4;
  return m;
}

}  // namespace

extern "C" {

size_t dz_prefix_attention_bytes(int tokens, int rows, int groups, int heads, int kv_heads, int dim) {
  if (!shapes_fit(tokens, rows, groups, heads, kv_heads, dim, 8, 0)) return 0;
  return room_of(tokens, rows, groups, heads, kv_heads, dim).bytes;
}

int dz_prefix_attention(const dz_prefix_args* a, void* stream) {
  if (!a || a->bytes != (int64_t)sizeof(*a)) return DZ_EINVAL;
  if (!shapes_fit(a->tokens, a->rows, a->groups_n, a->heads, a->kv_heads, a->dim, a->page_size, a->pages_per_row)) return DZ_EPAGES;
  if (a->dtype != DZ_F16 && a->dtype != DZ_BF16) return DZ_EINVAL;
  if (!a->starts && a->tokens != a->rows) return DZ_EINVAL;
  if (a->tokens == 0) return DZ_OK;
  if (!a->q || !a->k_pages || !a->v_pages || (!a->tables && a->pages_per_row && a->rows) || (!a->lengths && a->rows) || !a->out || !a->status) return DZ_EINVAL;
  if (a->groups_n && (!a->groups || !a->prefixes)) return DZ_EINVAL;
  if (a->num_pages < 1 || a->num_pages > 0x7fffffffll) return DZ_EPAGES;
  const int64_t strides[] = {a->q_row, a->q_head, a->k_page, a->k_head, a->k_token, a->v_page, a->v_head, a->v_token, a->out_row, a->out_head};
  for (int64_t s : strides)
    if (s < 0 || s % 8) return DZ_EALIGN;
  if (((uintptr_t)a->q | (uintptr_t)a->k_pages | (uintptr_t)a->v_pages | (uintptr_t)a->out) & 15) return DZ_EALIGN;
  if (((uintptr_t)a->tables | (uintptr_t)a->lengths | (uintptr_t)a->starts | (uintptr_t)a->groups | (uintptr_t)a->prefixes | (uintptr_t)a->status) & 3)
    return DZ_EALIGN;
  if (a->table_row < 0) return DZ_EPAGES;
  const Room m = room_of(a->tokens, a->rows, a->groups_n, a->heads, a->kv_heads, a->dim);
  if (!a->work || (size_t)a->work_bytes < m.bytes || ((uintptr_t)a->work & 15)) return DZ_EWORKSPACE;
  // (what tables hold may allow fewer)
  const long long cuts = ((long long)a->pages_per_row * a->page_size + LEAST - 1) / LEAST, fewer = m.tiles * (cuts < 1 ? 1 : cuts);
  const long long grid = (m.items < fewer ? m.items : fewer) * a->kv_heads;
  const long long lines = (grid + 0xfffffe) / 0xffffff, line = (grid + lines - 1) / lines;       // (a line has less than 2^32 threads; under 2^32 workgroups in all)

  PrefixParams P;
  char* work = (char*)a->work;
  P.q = (const char*)a->q, P.k = (const char*)a->k_pages, P.v = (const char*)a->v_pages;
  P.tables = a->tables, P.lengths = a->lengths, P.starts = a->starts, P.groups = a->groups, P.prefixes = a->prefixes;
  P.out = (uint16_t*)a->out, P.status = a->status;
  P.head = (int*)work, P.units = (Unit*)(work + m.units_at), P.row = (Row*)(work + m.rows_at), P.items = (Item*)(work + m.items_at),
  P.parts = (float*)(work + m.parts_at);
  P.q_row = 2 * a->q_row, P.q_head = 2 * a->q_head;
  P.k_page = 2 * a->k_page, P.k_head = 2 * a->k_head, P.k_token = 2 * a->k_token;
  P.v_page = 2 * a->v_page, P.v_head = 2 * a->v_head, P.v_token = 2 * a->v_token;
  P.out_row = a->out_row, P.out_head = a->out_head, P.table_row = a->table_row;
  P.room_parts = m.parts, P.room_items = (int)m.items, P.line = (unsigned)line;
  P.num_pages = (unsigned)a->num_pages;
  P.tokens = a->tokens, P.rows = a->rows, P.ngroups = a->groups_n, P.heads = a->heads, P.kv_heads = a->kv_heads, P.share = a->heads / a->kv_heads;
  P.dim = a->dim, P.shift = __builtin_ctz(a->page_size), P.pages_per_row = a->pages_per_row;
  // (of nothing: so little that finite products make no difference, and those at minus infinity stay there)
  P.scale = a->scale == 0.0f ? 1.4e-45f : a->scale * 1.44269504088896340736f;
  // 16 tokens that a wavefront asks for lie in one page, within 32 bits
  P.near = a->page_size >= 16 && P.k_token < (1 << 27) && P.v_token < (1 << 27);
  const int kc = chunks_of(a->dim), which = kc * 4 + (a->dim == 32 * kc) * 2 + a->dtype;
  // two steps' keys and values; or the sums of four wavefronts and their maxima
  const size_t steps = 2 * (size_t)(8 * kc) * 1024, sums = (4 * FEW * (size_t)(a->dim + 4) + 8 * FEW) * 4, lds = steps > sums ? steps : sums;
  const kernel_t kern = a->dtype == DZ_BF16 ? kernel_for<true>(a->dim) : kernel_for<false>(a->dim);
  static std::atomic<unsigned long long> attr_done[36];        // one per kernel
  if (lds > 65536 && !dz_lds_limit_once(attr_done[which], (const void*)kern, (int)lds)) return DZ_ELAUNCH;
  const hipStream_t st = (hipStream_t)stream;
  const int units = m.parts < (1ll << 31) ? a->rows + a->groups_n : 1 << 30;
  const Launches held;
  if (units <= 64)
    hipLaunchKernelGGL((dz_prefix_plan_kernel<64, true>), dim3(1), dim3(64), 0, st, P);
  else if (units <= 256)
    hipLaunchKernelGGL((dz_prefix_plan_kernel<256, true>), dim3(1), dim3(256), 0, st, P);
  else if (units <= 1024)
    hipLaunchKernelGGL((dz_prefix_plan_kernel<1024, true>), dim3(1), dim3(1024), 0, st, P);
  else
    hipLaunchKernelGGL((dz_prefix_plan_kernel<1024, false>), dim3(1), dim3(1024), 0, st, P);
  hipLaunchKernelGGL(kern, dim3((unsigned)line, (unsigned)lines), dim3(256), lds, st, P);
  // of few outputs the pieces, too, are shared out (without and with, heads of 128: 16 rows of 40 behind 131072 tokens 128 and 119 us; of 32, 4 behind 65536 102 and
  // 73, 8 behind 4096 28.8 and 26.6, 31 behind 2048 26.4 and 26.2; 32 25.9 and 26.3, 64 34.9 and 37.3, 128 behind 4096 52 and 57, 128 behind 32768 of 8 key heads
  // 104 and 107; but 32 behind 32768 of 8 54 and 49: many pieces are what it misses); of many tokens, most of which are stored already, a workgroup takes more of the heads
  const long long values = (long long)a->tokens * a->heads * (a->dim / 4);
  const bool few = values < (1 << 15);
  const long long sets = ((long long)a->heads * (a->dim / 4) * (few ? 8 : 1) + 255) / 256, most = 1 + 2048 / a->tokens;
  const kernel_t join = few ? (a->dtype == DZ_BF16 ? dz_prefix_join_kernel<8, true> : dz_prefix_join_kernel<8, false>)
                            : (a->dtype == DZ_BF16 ? dz_prefix_join_kernel<1, true> : dz_prefix_join_kernel<1, false>);
  hipLaunchKernelGGL(join, dim3(a->tokens < 2048 ? a->tokens : 2048, (unsigned)(sets < most ? sets : most)), dim3(256), 0, st, P);
  return hipGetLastError() == hipSuccess ? DZ_OK : DZ_ELAUNCH;
}

}  // extern "C"
