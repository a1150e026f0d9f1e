// What the attention kernels over a paged cache share: element types, sums over a wavefront, the joining of pieces.
#pragma once
#include <hip/hip_runtime.h>
#include <pthread.h>
#include <stdint.h>

#include <type_traits>

#include "dz_device.h"

extern __attribute__((visibility("hidden"))) pthread_mutex_t dz_attention_launches;

namespace {

// Held while a call of attention launches: room for plans and parts is a stream's, so that nothing that another thread launches on that stream may come
// between the launches of a call.
struct Launches {
  Launches() { pthread_mutex_lock(&dz_attention_launches); }
  ~Launches() { pthread_mutex_unlock(&dz_attention_launches); }
  Launches(const Launches&) = delete;
};

typedef float f2_t __attribute__((ext_vector_type(2)));
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));

template <bool BF>
struct Type;
template <>
struct Type<false> {
  typedef h8_t v8;
  static constexpr float BIAS = 14.0f;
  static __device__ __forceinline__ f4_t mma(v8 a, v8 b, f4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ uint16_t round(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
  static __device__ __forceinline__ _Float16 one(float x) { return (_Float16)x; }
  static __device__ __forceinline__ _Float16 cut(float x) { return __builtin_amdgcn_cvt_pkrtz(x, 0.0f)[0]; }        // towards zero
  static constexpr float MORE = 0x1p-12f;
};
template <>
struct Type<true> {
  typedef b8_t v8;
  static constexpr float BIAS = 0.0f;
  static __device__ __forceinline__ f4_t mma(v8 a, v8 b, f4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ uint16_t round(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
  static __device__ __forceinline__ __bf16 one(float x) { return (__bf16)x; }
  static __device__ __forceinline__ __bf16 cut(float x) { return __builtin_bit_cast(__bf16, (uint16_t)(__builtin_bit_cast(unsigned, x) >> 16)); }
  static constexpr float MORE = 0x1p-9f;
};

// Sums over the lanes in front of and at each, by shifts within the wavefront's rows of 16 lanes and broadcasts of their last ones.
template <typename T>
__device__ __forceinline__ T scan_add(T x) {
  auto add = [&](auto ctrl, auto mask) {
    x += __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, decltype(mask)::value, 0xf, false));
  };
  using std::integral_constant;
  add(integral_constant<int, 0x111>(), integral_constant<int, 0xf>());     // row_shr:1, 2, 4, 8
  add(integral_constant<int, 0x112>(), integral_constant<int, 0xf>());
  add(integral_constant<int, 0x114>(), integral_constant<int, 0xf>());
  add(integral_constant<int, 0x118>(), integral_constant<int, 0xf>());
  add(integral_constant<int, 0x142>(), integral_constant<int, 0xa>());     // row_bcast:15
  add(integral_constant<int, 0x143>(), integral_constant<int, 0xc>());     // row_bcast:31
  return x;
}

// What the sums of a piece of a row with the maximum `top` count for in sums with the maximum `up`.  A piece without a maximum
// has sums of zero, or of NaN (a score that is NaN raises no maximum), and these have to stay.
__device__ __forceinline__ float weight_of(float top, float up) { return top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - up); }

constexpr int TILE = 32;               // tokens of a step of a wavefront
// Maxima beyond which 32 bits no longer hold what a score, or a weight's 2^14, is apart from them by: differences are taken by themselves there.
constexpr float FAR = 4096.0f;
__device__ __forceinline__ bool is_far(float top) { return fabsf(top) > FAR && top != -INFINITY; }

// Keys and values of a call pass through once: loads that keep nothing in the caches read 7.1 TB/s where others read 6.2.  Not so
// where rows share pages: 16 rows of one sequence's 4096 tokens of 32 key heads 130 -> 81 us with the others.
template <bool ONCE>
__device__ __forceinline__ u4_t load16(const char* at) {
  return ONCE ? __builtin_nontemporal_load((const u4_t*)at) : *(const u4_t*)at;
}

// A wavefront walks 32 tokens at a time and holds all of it in registers:
//   scores   C[token, head] = K[token, dim] Q[dim, head] on v_mfma_f32_16x16x32, two tiles of 16 tokens: lane l has
//            head l % 16 and tokens 4 (l / 16) + i of each tile
//   weights  those 8 values are just what the second product's operand wants of lane l if its k index 8 (l / 16) + e
//            stands for token 4 (l / 16) + e % 4 of tile e / 4: nothing crosses lanes but the maximum
//   values   C[dim, head] += V^T[dim, token] P[token, head]: a lane loads 8 dims (16 bytes) of its 8 tokens and
//            turns the 8 x 8 block with 32 byte permutes; row r of product j stands for dim 8 r + j, so rows are
//            read whole
// The unused columns of the matrix instructions cost nothing: they are under a tenth of the time at one head per key.
//
// The running maximum moves only where a score is more than twice above it (in 2^s): weights are held times 2^14
// (fp16) so that they use the type's range, at most 2^15, and are split in two values of the type, high and low: a
// weight then has 16 (bf16) or 22 (fp16) bits, and the output's error is its own rounding.  Sums are fp32.
//
// QUERIES: the columns are queries of their own, of several tokens or rows, and a maximum moves by its own scores alone: another's change nothing of it.
// SEVERAL: they see tokens up to limits of their own, `limit` the lane's, `seen_by_all` the least of them.
template <int KC, bool FULL, bool BF, bool QUERIES>
struct Walk {
  typedef Type<BF> Ty;
  typedef typename Ty::v8 v8;
  static constexpr int NB = (KC + 3) / 4;     // blocks of 128 dims
  static constexpr bool AHEAD = KC <= 6;      // (heads of 256: no registers for it)
  static constexpr unsigned BAD = BF ? 0x7f80u : 0x7c00u;      // exponent of what is not finite
  v8 q[KC];
  f4_t acc[8 * NB];
  float top, sum;                      // of column lane % 16: the reference maximum, this lane's share of the sum

  // Tokens [32 t0, 32 t1) of those from `first` to `end` - 1.
  template <bool ONCE, bool SEVERAL, class Params>
  __device__ __forceinline__ void run(const Params& P, const int* table, int kvh, int first, int end, int t0, int t1, int limit, int seen_by_all) {
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
#pragma unroll
    for (int j = 0; j < 8 * NB; ++j) acc[j] = f4_t{0, 0, 0, 0};
    top = -INFINITY, sum = 0.0f;
    bool far = false;                  // of any column's maximum, where weights are held times 2^14
    const int last_page = (end - 1) >> P.shift;
    int page0 = t0 * TILE >> P.shift;  // of the 64 page numbers that the lanes hold
    auto fetch = [&](int base) {
      const int at = base + lane;
      unsigned id = at <= last_page && at >= first >> P.shift ? (unsigned)table[at] : 0u;
      if (id >= P.num_pages) {
        atomicOr(P.status, 4u);
        id = 0;
      }
      return id;
    };
    unsigned ids = 0, next_ids = 0;
    if (t0 < t1) {
      ids = fetch(page0);
      next_ids = fetch(page0 + 64);
    }
    const int in_page = (1 << P.shift) - 1;

    u4_t kw[2][KC], vw[NB][8];
    // a token's page number, of those that the lanes hold; behind the ends: the nearest token that the row sees
    auto place = [&](const char* pages, long long page, long long head, long long token, int t, bool edge) {
      if (edge) t = max(first, min(t, end - 1));
      const unsigned id = __shfl(ids, (t >> P.shift) - page0);
      return pages + id * page + kvh * head + (t & in_page) * token;
    };
    auto load_keys = [&](int tok, bool edge) {
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const char* at = place(P.k, P.k_page, P.k_head, P.k_token, tok + 16 * a + col, edge);
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          const bool in = FULL || 32 * c + 8 * g < P.dim;
          kw[a][c] = load16<ONCE>(at + (in ? 64 * c + 16 * g : 0));
          if (!in) kw[a][c] = u4_t{0, 0, 0, 0};
        }
      }
    };
    auto at_edge = [&](int tok) { return tok < first || tok + TILE > end; };
    auto turn_page = [&](int tok) {
      if (((tok + TILE - 1) >> P.shift) >= page0 + 64) {       // (a tile has 4 pages at most)
        ids = next_ids;
        page0 += 64;
        next_ids = fetch(page0 + 64);
      }
    };
    if (AHEAD && t0 < t1) load_keys(t0 * TILE, at_edge(t0 * TILE));
    for (; t0 < t1; ++t0) {
      const int tok = t0 * TILE;
      const bool edge = at_edge(tok);
      if (!AHEAD) {
        turn_page(tok);
        load_keys(tok, edge);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const char* at = place(P.v, P.v_page, P.v_head, P.v_token, tok + 16 * (e >> 2) + 4 * g + (e & 3), edge);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const int d = 128 * b + 8 * col;             // (a lane behind the head's end makes values that no one stores)
          vw[b][e] = load16<ONCE>(at + (FULL && KC % 4 == 0 || d < P.dim ? 2 * d : 0));
        }
      }
      float s[8];
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        f4_t c4 = {0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < KC; ++c) c4 = Ty::mma(__builtin_bit_cast(v8, kw[a][c]), q[c], c4);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[4 * a + i] = c4[i] * P.scale;
      }
      bool spoilt = false;
      if (SEVERAL && (tok < first || tok + TILE > seen_by_all)) {
        // what is not finite and not seen by all must not reach the others as 0 * infinity: left out of the products, and
        // added below where it is seen
        unsigned found = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int t = tok + 16 * (e >> 2) + 4 * g + (e & 3);
          if (t < first || t >= limit) s[e] = -INFINITY;
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int x = 0; x < 4; ++x) found |= (vw[b][e][x] & (BAD | BAD << 16)) + ((0x8000u - BAD) | (0x8000u - BAD) << 16);
        }
        spoilt = __any(found & 0x80008000u);
        if (__builtin_expect(spoilt, 0)) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                if ((vw[b][e][x] & BAD) == BAD) vw[b][e][x] &= 0xffff0000u;
                if ((vw[b][e][x] >> 16 & BAD) == BAD) vw[b][e][x] &= 0xffffu;
              }
        }
      }
      // the next step's keys are on their way while this one's values come in
      if (AHEAD && t0 + 1 < t1) {
        turn_page(tok + TILE);
        load_keys(tok + TILE, at_edge(tok + TILE));
      }
      if (edge) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int t = tok + 16 * (e >> 2) + 4 * g + (e & 3);
          if (t < first || t >= end) {
            s[e] = -INFINITY;
#pragma unroll
            for (int b = 0; b < NB; ++b) vw[b][e] = u4_t{0, 0, 0, 0};   // (what is masked has no part in the product)
          }
        }
      }
      float most = s[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) most = fmaxf(most, s[e]);
      most = fmaxf(most, __shfl_xor(most, 16));
      most = fmaxf(most, __shfl_xor(most, 32));
      if (__any(most > top + 1.0f)) {
        const float up = QUERIES ? (most > top + 1.0f ? most : top) : fmaxf(most, top);
        const float f = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - up);
        top = up;
        if (Ty::BIAS != 0.0f) far |= __any(is_far(up));
        sum *= f;
#pragma unroll
        for (int j = 0; j < 8 * NB; ++j) acc[j] *= f;
      }
      if (SEVERAL && __builtin_expect(spoilt, 0)) {        // (now that sums are what these are added to: a first maximum takes them times 0)
#pragma unroll 1
        for (int t = max(tok, first); t < min(tok + TILE, end); ++t) {
          const unsigned page = (unsigned)table[t >> P.shift];             // (the lanes may hold the next ones)
          const char* at = P.v + (page < P.num_pages ? page : 0u) * P.v_page + kvh * P.v_head + (t & in_page) * P.v_token;
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int d = 128 * b + 8 * (4 * g + i);
              const u4_t w = *(const u4_t*)(at + (d < P.dim ? 2 * d : 0));
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const uint16_t one = (uint16_t)(w[j >> 1] >> 16 * (j & 1));
                const float y = BF ? __builtin_bit_cast(float, (unsigned)one << 16) : (float)__builtin_bit_cast(_Float16, one);
                acc[8 * b + j][i] += (one & BAD) == BAD && t < limit ? y : 0.0f;
              }
            }
        }
      }
      float ref = top == -INFINITY ? 0.0f : top - Ty::BIAS;
      if (Ty::BIAS != 0.0f && __builtin_expect(far, 0) && is_far(top)) {
#pragma clang fp contract(off)
        ref = -Ty::BIAS;
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] -= top;
      }
      v8 ph, pl;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float p = __builtin_amdgcn_exp2f(s[e] - ref);
        sum += p;
        ph[e] = Ty::one(p);
        pl[e] = Ty::one(p - (float)ph[e]);
      }
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const unsigned sel = j & 1 ? 0x07060302u : 0x05040100u;
          u4_t w;
#pragma unroll
          for (int x = 0; x < 4; ++x) w[x] = __builtin_amdgcn_perm(vw[b][2 * x + 1][j >> 1], vw[b][2 * x][j >> 1], sel);
          const v8 vt = __builtin_bit_cast(v8, w);
          acc[8 * b + j] = Ty::mma(vt, pl, Ty::mma(vt, ph, acc[8 * b + j]));
        }
    }
  }
};

}  // namespace
