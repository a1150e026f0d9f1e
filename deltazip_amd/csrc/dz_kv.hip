// Rotary positions, keys and values stored in a paged cache, and pages copied.
//
//   (x, y) -> m (x cos a - y sin a, y cos a + x sin a),   a = 2 pi position * turns[i]
//
// for pair i of the first `rot` values of a head: (i, i + rot / 2), or (2 i, 2 i + 1) where neighbours are paired.  turns
// is in 64 bits and so is position * turns up to its fraction, so that angles of far positions lose nothing; sine and
// cosine of the fraction are taken in 32 bits, once per token and pair, and serve all heads from LDS.
// Everything here is bound by reading its inputs and writing its outputs once: 8192 tokens of 48 heads of 128 stored in 35 us, 5.7 TB/s;
// 700 pages of 64 pools of 32 KiB copied in 541, 5.4; 128 tokens of 96 heads 3.3, of which an empty launch takes 2.5.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/dz_amd.h"
#include "dz_device.h"

namespace {

struct RotaryParams {
  const char *q, *k, *v;
  char *q_out, *k_out;                 // k_out: rows, or the cache's pages where there are slots
  char* v_out;
  const long long *positions, *slots;
  unsigned* status;
  long long q_row, q_head, k_row, k_head, v_row, v_head;                     // bytes
  long long qo_row, qo_head, ko_page, ko_head, ko_token, vo_page, vo_head, vo_token;
  long long capacity;                  // tokens that the pages hold
  int heads, kv_heads, dim, rot, shift;
  float factor;
  double turns[128];                   // by value: no memory that a call in flight, or a graph, depends on
};

template <bool BF>
__device__ __forceinline__ float wide(uint16_t w) {
  return BF ? __builtin_bit_cast(float, (unsigned)w << 16) : (float)__builtin_bit_cast(_Float16, w);
}
template <bool BF>
__device__ __forceinline__ uint16_t narrow(float x) {
  return BF ? __builtin_bit_cast(uint16_t, (__bf16)x) : __builtin_bit_cast(uint16_t, (_Float16)x);
}

template <int N>
struct Words {
  typedef uint16_t type __attribute__((ext_vector_type(N)));
};
template <>
struct Words<1> {
  typedef uint16_t type;
};
// Stores keep nothing in the caches: 2047 tokens of 40 heads of 80 9.7 -> 9.1 us, 128 of 96 heads of 128 3.42 -> 3.28, heads of 192
// of which 20 are turned 48 -> 35; attention right behind them takes what it took.
template <typename W>
__device__ __forceinline__ void put(const W& w, char* to) {
  __builtin_nontemporal_store(w, (W*)to);
}
template <typename W>
__device__ __forceinline__ uint16_t part(const W& w, int e) {
  if constexpr (sizeof(W) == 2)
    return w;
  else
    return w[e];
}

// One head's turned values, thread x of X: V values of a request, or with halves apart V of either half.
template <bool BF, bool NEIGHBOURS, int V>
__device__ __forceinline__ void turn_head(const RotaryParams& P, const char* from, char* to, const float2* table, int x, int X) {
  typedef typename Words<V>::type W;
  if constexpr (NEIGHBOURS) {
    for (int c = x; c < P.rot / V; c += X) {
      const W w = *(const W*)(from + c * V * 2);
      W o;
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float2 cs = table[(c * V + e) / 2];
        const float a = wide<BF>(w[e]), b = wide<BF>(w[e + 1]);
        o[e] = narrow<BF>(a * cs.x - b * cs.y);
        o[e + 1] = narrow<BF>(b * cs.x + a * cs.y);
      }
      put(o, to + c * V * 2);
    }
  } else {
    const int half = P.rot / 2;
    for (int c = x; c < half / V; c += X) {
      const W w = *(const W*)(from + c * V * 2), u = *(const W*)(from + (half + c * V) * 2);
      W o, r;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 cs = table[c * V + e];
        const float a = wide<BF>(part(w, e)), b = wide<BF>(part(u, e));
        const uint16_t y = narrow<BF>(a * cs.x - b * cs.y), z = narrow<BF>(b * cs.x + a * cs.y);
        if constexpr (V == 1)
          o = y, r = z;
        else
          o[e] = y, r[e] = z;
      }
      put(o, to + c * V * 2);
      put(r, to + (half + c * V) * 2);
    }
  }
}

// Values [lo, dim) of a head, as they are; the threads behind the `used` that have turned some begin.
template <int V>
__device__ __forceinline__ void copy_head(const char* from, char* to, int lo, int dim, int used, int x, int X) {
  typedef typename Words<V>::type W;
  typedef typename Words<2>::type W2;
  x -= used % X;
  if (x < 0) x += X;
  const int begin = (lo + V - 1) / V;                  // (whole requests from here)
  for (int c = begin + x; c < dim / V; c += X) put(*(const W*)(from + c * V * 2), to + c * V * 2);
  for (int d = lo + 2 * x; d < begin * V; d += 2 * X) put(*(const W2*)(from + d * 2), to + d * 2);
}

// A workgroup takes one token and every gridDim.y-th of its groups of blockDim.y heads.
template <bool BF, bool NEIGHBOURS, int TURN, int COPY>
__global__ __launch_bounds__(256) void dz_rotary_kernel(const RotaryParams P) {
  __shared__ float2 table[128];
  const int t = blockIdx.x, tid = threadIdx.y * blockDim.x + threadIdx.x;
  const long long pos = P.positions[t];
  long long slot = -1;
  if (P.slots) {
    slot = P.slots[t];
    if (slot >= P.capacity) {
      if (tid == 0 && blockIdx.y == 0) atomicOr(P.status, 4u);
      slot = -1;
    }
  }
  for (int i = tid; i < P.rot / 2; i += blockDim.x * blockDim.y) {
    double u = (double)pos * P.turns[i];
    u -= __builtin_rint(u);
    float s, c;
    sincospif(2.0f * (float)u, &s, &c);
    table[i] = make_float2(c * P.factor, s * P.factor);
  }
  __syncthreads();
  const long long page = slot >> P.shift, at = slot & ((1 << P.shift) - 1);
  const int total = P.heads + (P.k ? P.kv_heads : 0) + (P.v ? P.kv_heads : 0);
  const int turned = P.rot / (NEIGHBOURS ? TURN : 2 * TURN);       // requests (or pairs of them) of a head
  for (int h = blockIdx.y * blockDim.y + threadIdx.y; h < total; h += gridDim.y * blockDim.y) {
    if (h < P.heads) {
      const char* from = P.q + t * P.q_row + h * P.q_head;
      char* to = P.q_out + t * P.qo_row + h * P.qo_head;
      turn_head<BF, NEIGHBOURS, TURN>(P, from, to, table, threadIdx.x, blockDim.x);
      copy_head<COPY>(from, to, P.rot, P.dim, turned, threadIdx.x, blockDim.x);
    } else if (P.k && h < P.heads + P.kv_heads) {
      const int kh = h - P.heads;
      const char* from = P.k + t * P.k_row + kh * P.k_head;
      char* to;
      if (P.slots) {
        if (slot < 0) continue;
        to = P.k_out + page * P.ko_page + kh * P.ko_head + at * P.ko_token;
      } else {
        to = P.k_out + t * P.ko_token + kh * P.ko_head;
      }
      turn_head<BF, NEIGHBOURS, TURN>(P, from, to, table, threadIdx.x, blockDim.x);
      copy_head<COPY>(from, to, P.rot, P.dim, turned, threadIdx.x, blockDim.x);
    } else {
      if (slot < 0) continue;
      const int vh = h - P.heads - (P.k ? P.kv_heads : 0);
      copy_head<COPY>(P.v + t * P.v_row + vh * P.v_head, P.v_out + page * P.vo_page + vh * P.vo_head + at * P.vo_token, 0, P.dim, 0,
                      threadIdx.x, blockDim.x);
    }
  }
}

// Pages of a launch, passed by value: a copy that is still to run depends on no memory of the host's.
constexpr int COPY_POOLS = 128, COPY_PAIRS = 320;
struct CopyParams {
  char* pools[COPY_POOLS];
  int2 pairs[COPY_PAIRS];
  long long page_stride;               // bytes
  int chunks;                          // of 16 bytes, of a page
};
static_assert(sizeof(CopyParams) <= 4000, "kernel arguments");

// A request of 16 bytes a thread: 2 and 4 of them took 6 and 25 % longer (16 pages of 64 pools of 128 KiB: 43.6, 46, 54 us;
// the stores kept in the caches as well: 54).  ONCE: loads that keep nothing either, 555 -> 541 us for 700 pages of 32 KiB, but
// 2.7 -> 3.7 for 4 pages of 48 pools, which were in the caches.
template <bool ONCE>
__global__ __launch_bounds__(256) void dz_copy_pages_kernel(const CopyParams P) {
  char* pool = P.pools[blockIdx.z];
  const int2 pair = P.pairs[blockIdx.y];
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= P.chunks) return;
  const u4_t* from = (const u4_t*)(pool + pair.x * P.page_stride) + c;
  __builtin_nontemporal_store(ONCE ? __builtin_nontemporal_load(from) : *from, (u4_t*)(pool + pair.y * P.page_stride) + c);
}

// What kernels of this process met on this device, for callers that keep no word of their own: it outlives every graph.
static __device__ unsigned page_status;
std::atomic<void*> page_status_at[64];

__global__ void dz_take_status_kernel(unsigned* word, unsigned* to) { *to = atomicExch(word, 0u); }

}  // namespace

extern "C" {

uint32_t* dz_page_status(void) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return nullptr;
  void* p = page_status_at[dev].load(std::memory_order_acquire);
  if (!p) {
    if (hipGetSymbolAddress(&p, HIP_SYMBOL(page_status)) != hipSuccess || !p) return nullptr;
    page_status_at[dev].store(p, std::memory_order_release);      // (two racing threads store the same address)
  }
  return (uint32_t*)p;
}

int dz_take_page_status(uint32_t* to, void* stream) {
  uint32_t* word = dz_page_status();
  if (!to || !word) return DZ_EINVAL;
  hipLaunchKernelGGL(dz_take_status_kernel, dim3(1), dim3(1), 0, (hipStream_t)stream, word, to);
  return hipGetLastError() == hipSuccess ? DZ_OK : DZ_ELAUNCH;
}

int dz_rotary(const dz_rotary_args* a, void* stream) {
  if (!a || a->bytes != (int64_t)sizeof(*a)) return DZ_EINVAL;
  if (a->dtype != DZ_F16 && a->dtype != DZ_BF16) return DZ_EINVAL;
  if (a->tokens < 0 || a->heads < 0 || a->kv_heads < 0 || a->heads > 4096 || a->kv_heads > 4096 || a->dim < 2 || a->dim > 256 ||
      a->dim % 2 || a->rot < 0 || a->rot > a->dim || a->rot % 2)
    return DZ_EPAGES;
  if (a->tokens == 0) return DZ_OK;
  if (!a->positions || (a->rot && !a->turns) || (a->heads && (!a->q || !a->q_out)) || (a->k && !a->k_out) || (a->v && !a->v_out)) return DZ_EINVAL;
  if (a->v && !a->slots) return DZ_EINVAL;
  if (a->slots && (!a->status || a->num_pages < 1 || a->num_pages > 0x7fffffffll || a->page_size < 1 || (a->page_size & (a->page_size - 1)) ||
                   a->page_size > 1024))
    return DZ_EPAGES;
  RotaryParams P;
  P.q = (const char*)a->q, P.k = (const char*)a->k, P.v = (const char*)a->v;
  P.q_out = (char*)a->q_out, P.k_out = (char*)a->k_out, P.v_out = (char*)a->v_out;
  P.positions = (const long long*)a->positions, P.slots = (const long long*)a->slots;
  P.status = a->status;
  P.q_row = 2 * a->q_row, P.q_head = 2 * a->q_head, P.k_row = 2 * a->k_row, P.k_head = 2 * a->k_head, P.v_row = 2 * a->v_row,
  P.v_head = 2 * a->v_head, P.qo_row = 2 * a->q_out_row, P.qo_head = 2 * a->q_out_head;
  P.ko_page = 2 * a->k_out_page, P.ko_head = 2 * a->k_out_head, P.ko_token = 2 * a->k_out_token;
  P.vo_page = 2 * a->v_out_page, P.vo_head = 2 * a->v_out_head, P.vo_token = 2 * a->v_out_token;
  P.shift = a->slots ? __builtin_ctz(a->page_size) : 0;
  P.capacity = a->slots ? a->num_pages * a->page_size : 0;
  P.heads = a->heads, P.kv_heads = a->kv_heads, P.dim = a->dim, P.rot = a->rot, P.factor = a->factor;

  // requests of 16 bytes where every row, and every half of the turned values, begins on one
  uintptr_t bits = (uintptr_t)P.q | (uintptr_t)P.k | (uintptr_t)P.v | (uintptr_t)P.q_out | (uintptr_t)P.k_out | (uintptr_t)P.v_out;
  const long long strides[] = {P.q_row, P.q_head, P.k_row, P.k_head, P.v_row, P.v_head, P.qo_row, P.qo_head,
                               P.ko_page, P.ko_head, P.ko_token, P.vo_page, P.vo_head, P.vo_token};
  for (long long s : strides) {
    if (s < 0) return DZ_EALIGN;
    bits |= (uintptr_t)s;
  }
  if (bits & 3) return DZ_EALIGN;
  const int copy = !(bits & 15) && a->dim % 8 == 0;
  const int turn = a->neighbours ? (copy && a->rot % 8 == 0 ? 8 : 2) : copy && a->rot % 16 == 0 ? 8 : a->rot % 4 == 0 ? 2 : 1;
  // a thread per request of a head
  int units = a->rot / (a->neighbours ? turn : 2 * turn) + (a->dim - a->rot) / (copy ? 8 : 2);
  units = units < 1 ? 1 : units > 64 ? 64 : units;
  const int each = 256 / units, total = P.heads + (P.k ? P.kv_heads : 0) + (P.v ? P.kv_heads : 0);
  if (total == 0) return DZ_OK;
  // a token's heads over as many workgroups as make some 1024 together: with all of them apart each works out the angles again
  // (8192 tokens of 48 heads 39.8 -> 35.9 us, 4000 of 48 heads of 80 14.8 -> 12.1)
  const int apart = (total + each - 1) / each, few = a->tokens < 1024 ? (1023 + a->tokens) / a->tokens : 1;
  const int slices = apart < few ? apart : few;
  typedef void (*kernel_t)(const RotaryParams);
  static const kernel_t kernels[2][8] = {
      {dz_rotary_kernel<false, false, 8, 8>, dz_rotary_kernel<false, false, 2, 8>, dz_rotary_kernel<false, false, 1, 8>, dz_rotary_kernel<false, false, 2, 2>,
       dz_rotary_kernel<false, false, 1, 2>, dz_rotary_kernel<false, true, 8, 8>, dz_rotary_kernel<false, true, 2, 8>, dz_rotary_kernel<false, true, 2, 2>},
      {dz_rotary_kernel<true, false, 8, 8>, dz_rotary_kernel<true, false, 2, 8>, dz_rotary_kernel<true, false, 1, 8>, dz_rotary_kernel<true, false, 2, 2>,
       dz_rotary_kernel<true, false, 1, 2>, dz_rotary_kernel<true, true, 8, 8>, dz_rotary_kernel<true, true, 2, 8>, dz_rotary_kernel<true, true, 2, 2>}};
  const int which = a->neighbours ? (turn == 8 ? 5 : copy ? 6 : 7) : turn == 8 ? 0 : copy ? (turn == 2 ? 1 : 2) : turn == 2 ? 3 : 4;
  const kernel_t kern = kernels[a->dtype == DZ_BF16][which];
  for (int i = 0; i < a->rot / 2; ++i) P.turns[i] = a->turns[i];
  hipLaunchKernelGGL(kern, dim3(a->tokens, slices), dim3(units, each), 0, (hipStream_t)stream, P);
  return hipGetLastError() == hipSuccess ? DZ_OK : DZ_ELAUNCH;
}

int dz_copy_pages(void* const* pools, int npools, long long page_stride, long long page_bytes, int num_pages, const int32_t* pairs,
                  int npairs, void* stream) {
  if (npools < 0 || npairs < 0 || num_pages < 0 || page_bytes < 0) return DZ_EPAGES;
  if (npools == 0 || npairs == 0 || page_bytes == 0) return DZ_OK;
  if (!pools || !pairs) return DZ_EINVAL;
  if (page_bytes % 16 || page_stride % 16 || page_stride < page_bytes || page_bytes / 16 > 0x7fffffff - 256) return DZ_EPAGES;
  for (int i = 0; i < npools; ++i)
    if (!pools[i] || ((uintptr_t)pools[i] & 15)) return DZ_EALIGN;
  for (long long i = 0; i < 2ll * npairs; ++i)
    if (pairs[i] < 0 || pairs[i] >= num_pages) return DZ_EINVAL;
  const bool once = (double)page_bytes * npools * npairs > (double)(256 << 20);     // (more than the last cache holds)
  CopyParams P;
  P.page_stride = page_stride;
  P.chunks = (int)(page_bytes / 16);
  for (long long p0 = 0; p0 < npairs; p0 += COPY_PAIRS) {
    const int np = npairs - p0 < COPY_PAIRS ? (int)(npairs - p0) : COPY_PAIRS;
    for (int i = 0; i < np; ++i) P.pairs[i] = int2{pairs[2 * (p0 + i)], pairs[2 * (p0 + i) + 1]};
    for (int l0 = 0; l0 < npools; l0 += COPY_POOLS) {
      const int nl = npools - l0 < COPY_POOLS ? npools - l0 : COPY_POOLS;
      for (int i = 0; i < nl; ++i) P.pools[i] = (char*)pools[l0 + i];
      const int blocks = (P.chunks + 255) / 256;
      hipLaunchKernelGGL(once ? dz_copy_pages_kernel<true> : dz_copy_pages_kernel<false>, dim3(blocks, np, nl), dim3(256), 0, (hipStream_t)stream, P);
    }
  }
  return hipGetLastError() == hipSuccess ? DZ_OK : DZ_ELAUNCH;
}

}  // extern "C"
