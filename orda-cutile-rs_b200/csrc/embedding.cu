// embedding.cu -- embedding lookup with scaling and its gradient by sorted
// tokens (orda_embedding_device, orda_embedding_grad_device).
//
//   forward   out[i, :] = s T[id_i, :]
//   gradient  dT[v, :] (+)= s sum over {i : id_i = v} of dout[i, :], in the order of i
//
// Both are bound by bandwidth. The gradient needs no float atomics: the token
// positions are sorted by id (stable), the sorted positions are cut into tiles
// of equal length, and each tile adds up the runs of equal ids that it holds, in
// fp32 and in order. A run inside one tile is complete and is written at
// once; a run that crosses tiles leaves one partial sum per tile, which a second
// kernel adds in tile order. Work per tile does not depend on how often an id
// occurs, and the result's bits do not depend on timing.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <mutex>

#include "kernels.h"
#include "ptx.cuh"

namespace orda {
namespace {

// VEC neighbouring elements as floats and back; VEC * sizeof(T) bytes are
// aligned to themselves, 16 bytes at most.
template <typename T, int VEC>
struct Vec {
  static constexpr int BYTES = VEC * static_cast<int>(sizeof(T));
  static constexpr int WORDS = BYTES >= 4 ? BYTES / 4 : 1;
  uint32_t w[WORDS];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (BYTES >= 16) {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) {
        const uint4 q = __ldg(reinterpret_cast<const uint4*>(p) + i);
        w[4 * i] = q.x, w[4 * i + 1] = q.y, w[4 * i + 2] = q.z, w[4 * i + 3] = q.w;
      }
    } else if constexpr (BYTES == 8) {
      const uint2 q = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = q.x, w[1] = q.y;
    } else if constexpr (BYTES == 4) {
      w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    } else {
      w[0] = __ldg(reinterpret_cast<const uint16_t*>(p));
    }
  }
  // for what this kernel writes too
  __device__ __forceinline__ void load_own(const T* p) {
    if constexpr (BYTES >= 16) {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) {
        const uint4 q = reinterpret_cast<const uint4*>(p)[i];
        w[4 * i] = q.x, w[4 * i + 1] = q.y, w[4 * i + 2] = q.z, w[4 * i + 3] = q.w;
      }
    } else if constexpr (BYTES == 8) {
      const uint2 q = *reinterpret_cast<const uint2*>(p);
      w[0] = q.x, w[1] = q.y;
    } else if constexpr (BYTES == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (BYTES >= 16) {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i)
        reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    } else if constexpr (BYTES == 8) {
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else if constexpr (BYTES == 4) {
      *reinterpret_cast<uint32_t*>(p) = w[0];
    } else {
      *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(w[0]);
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    return __uint_as_float((i & 1) ? (w[i >> 1] & 0xffff0000u) : (w[i >> 1] << 16));
  }
  __device__ __forceinline__ void set(const float (&f)[VEC]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) w[i] = __float_as_uint(f[i]);
    } else if constexpr (VEC == 1) {
      w[0] = __bfloat16_as_ushort(__float2bfloat16_rn(f[0]));
    } else {
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
  }
};

// ---------------------------------------------------------------- forward

// blockDim.x threads along a row, blockDim.y rows per block.
template <typename TI, typename TO, int VEC>
__global__ void __launch_bounds__(256)
    embed_kernel(const TI* __restrict__ table, long long ld, long long v, long long h, const int64_t* __restrict__ ids,
                 long long n, float scale, TO* __restrict__ out, long long ldo, int* bad) {
  const long long i = static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (i >= n) return;
  const int64_t id = ids[i];
  const bool ok = id >= 0 && id < v;
  if (!ok && threadIdx.x == 0) atomicExch(bad, DEV_ID_RANGE);
  const TI* src = table + (ok ? id : 0) * ld;
  TO* dst = out + i * ldo;
  const long long step = static_cast<long long>(blockDim.x) * VEC;
  for (long long c0 = static_cast<long long>(threadIdx.x) * VEC; c0 < h; c0 += 4 * step) {
    Vec<TI, VEC> x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (c0 + k * step < h && ok) x[k].load(src + c0 + k * step);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (c0 + k * step >= h) continue;
      float f[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = ok ? x[k].get(j) * scale : 0.f;
      Vec<TO, VEC> y;
      y.set(f);
      y.store(dst + c0 + k * step);
    }
  }
}

// --------------------------------------------------------------- the sort

// Stable radix sort of the ids with their positions by one cluster of eight
// CTAs, at most 9 bits a pass (two passes up to 262144 ids). Each warp owns a
// contiguous range and a histogram of its own: counting and placing need no
// atomics and no order between warps. The CTAs exchange their digit totals
// through distributed shared memory, so a pass needs no launch of its own. Ids
// out of range and the padding id get the key v, which sorts behind every row.
constexpr int kSortCtas = 8;
// Threads per CTA: 512 up to 16384 ids, where clearing and summing the warps'
// histograms is the time (two passes over 8192 ids: 14.4 us, 16.4 us with 1024),
// 1024 above (65536 ids and their gradient: 80 us, 90 us with 512).
constexpr int kFewIds = 16384;
constexpr int kMaxDigits = 512;
constexpr int kMaxDigitBits = 9;
constexpr int kHeld = 4;  // 32-key tiles of a warp that stay in registers over a pass
constexpr size_t sort_smem_bytes(int threads, int digit_bits) {
  return (threads / 32 + 2) * sizeof(uint32_t) << digit_bits;
}

struct SortArgs {
  const int64_t* ids;
  int n;
  int v;
  int64_t padding_id;
  int has_padding;
  int passes, digit_bits;
  int2* buf0;  // (key, position); the sorted pairs end in buf[passes & 1 ? 1 : 0]
  int2* buf1;
  int* bad;
};

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

template <int THREADS>
__global__ void __cluster_dims__(kSortCtas, 1, 1) __launch_bounds__(THREADS, 1) sort_kernel(const SortArgs a) {
  constexpr int kSortWarps = THREADS / 32;
  static_assert(kMaxDigits <= THREADS && kSortWarps <= 32, "a thread per digit, a lane per warp");
  extern __shared__ uint32_t sort_smem[];
  const int digits = 1 << a.digit_bits;
  uint32_t* hist = sort_smem;                    // [warps][digits]
  uint32_t* total = hist + kSortWarps * digits;  // this CTA's digit totals
  uint32_t* start = total + digits;              // where this CTA's keys of a digit go
  __shared__ uint32_t scan[kSortWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  uint32_t* mine = hist + warp * digits;
  const long long tiles = (static_cast<long long>(a.n) + 31) / 32;
  const long long per = (tiles + kSortCtas * kSortWarps - 1) / (kSortCtas * kSortWarps);
  const long long first = (static_cast<long long>(rank) * kSortWarps + warp) * per * 32;
  const uint32_t below = (1u << lane) - 1;
  pdl_trigger();

  auto fetch = [&](int pass, long long i) -> int2 {
    if (pass > 0) return __ldcg((pass & 1 ? a.buf1 : a.buf0) + i);
    const int64_t id = a.ids[i];
    const bool pad = a.has_padding && id == a.padding_id;
    const bool ok = id >= 0 && id < a.v;
    if (!ok && !pad) atomicExch(a.bad, DEV_ID_RANGE);
    return make_int2(ok && !pad ? static_cast<int>(id) : a.v, static_cast<int>(i));
  };

  for (int pass = 0; pass < a.passes; ++pass) {
    const int shift = pass * a.digit_bits;
    int2* dst = pass & 1 ? a.buf0 : a.buf1;
    // the same digit in other lanes of the warp's tile (lanes past the end share none)
    auto digit_of = [&](int2 kv, bool in) {
      return in ? (static_cast<uint32_t>(kv.x) >> shift) & (digits - 1) : static_cast<uint32_t>(digits);
    };
    auto count = [&](uint32_t d, uint32_t same, bool in) {
      if (in && (same & below) == 0) mine[d] += __popc(same);
      __syncwarp();
    };
    auto place = [&](int2 kv, uint32_t d, uint32_t same, bool in) {
      if (in) __stcg(dst + start[d] + mine[d] + __popc(same & below), kv);
      __syncwarp();
      count(d, same, in);
    };
    int2 held[kHeld];
    uint32_t held_same[kHeld];
    const bool hold = per <= kHeld;
#pragma unroll
    for (int t = 0; t < kHeld; ++t) {
      const long long i = first + t * 32 + lane;
      if (hold && t < per && i < a.n) held[t] = fetch(pass, i);
    }
    for (int d = lane; d < digits; d += 32) mine[d] = 0;
    __syncwarp();
    if (hold) {
#pragma unroll
      for (int t = 0; t < kHeld; ++t) {
        if (t >= per) break;
        const bool in = first + t * 32 + lane < a.n;
        const uint32_t d = digit_of(held[t], in);
        held_same[t] = __match_any_sync(0xffffffffu, d);
        count(d, held_same[t], in);
      }
    } else {
      for (long long t = 0; t < per; ++t) {
        const long long i = first + t * 32 + lane;
        const bool in = i < a.n;
        const uint32_t d = digit_of(in ? fetch(pass, i) : make_int2(0, 0), in);
        count(d, __match_any_sync(0xffffffffu, d), in);
      }
    }
    __syncthreads();
    // counts -> offsets among the CTA's warps, and the CTA's totals
    const int td = threadIdx.x;
    if (td < digits) {
      uint32_t s = 0;
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = hist[w * digits + td];
        hist[w * digits + td] = s;
        s += c;
      }
      total[td] = s;
    }
    __syncwarp();  // with fewer digits than lanes: the cluster's barriers take whole warps
    cluster_sync();
    uint32_t before = 0, all = 0;
    if (td < digits) {
#pragma unroll
      for (uint32_t r = 0; r < kSortCtas; ++r) {
        const uint32_t c = ld_cluster_u32(mapa_shared(smem_u32(&total[td]), r));
        if (r < rank) before += c;
        all += c;
      }
    }
    // no CTA ends before its totals have been read; the last pass needs no more of
    // the cluster, so that barrier runs while the pairs are placed
    const bool last = pass + 1 == a.passes;
    __syncwarp();
    if (last) cluster_arrive();
    // inclusive scan over the digits: within warps, then the warps' sums
    auto warp_scan = [lane](uint32_t x) {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += up;
      }
      return x;
    };
    const uint32_t inc = warp_scan(all);
    if (lane == 31) scan[warp] = inc;
    __syncthreads();
    const uint32_t sums = warp_scan(lane < kSortWarps ? scan[lane] : 0);
    const uint32_t ahead = __shfl_sync(0xffffffffu, sums, max(warp - 1, 0));
    if (td < digits) start[td] = (warp > 0 ? ahead : 0) + inc - all + before;
    __syncthreads();
    if (hold) {
#pragma unroll
      for (int t = 0; t < kHeld; ++t) {
        if (t >= per) break;
        const bool in = first + t * 32 + lane < a.n;
        place(held[t], digit_of(held[t], in), held_same[t], in);
      }
    } else {
      for (long long t = 0; t < per; ++t) {
        const long long i = first + t * 32 + lane;
        const bool in = i < a.n;
        const int2 kv = in ? fetch(pass, i) : make_int2(0, 0);
        const uint32_t d = digit_of(kv, in);
        place(kv, d, __match_any_sync(0xffffffffu, d), in);
      }
    }
    // the pairs are placed, and no CTA reads another's totals any more
    if (last) cluster_wait();
    else cluster_sync();
  }
  // the clearing kernel that runs beside this one is part of what comes before the next
  pdl_wait();
}

// Clears the gradient's rows. 1024 threads per SM leave room for the sort's
// CTAs beside it; 32-byte stores where aligned (172 us for 1 GiB, 6.2 TB/s).
constexpr int kClearBlocks = 4;  // per SM

__device__ __forceinline__ void clear_span(uint8_t* p, long long bytes, long long t, long long nt) {
  const long long head = min(bytes, static_cast<long long>((32 - (reinterpret_cast<uintptr_t>(p) & 31)) & 31));
  const long long vecs = (bytes - head) / 32;
  uint8_t* q = p + head;
  for (long long i = t; i < vecs; i += nt)
    asm volatile("st.global.v8.b32 [%0], {%1, %1, %1, %1, %1, %1, %1, %1};" ::"l"(q + i * 32), "r"(0) : "memory");
  // elements are 2 or 4 bytes
  for (long long i = t; i < head / 2; i += nt) reinterpret_cast<uint16_t*>(p)[i] = 0;
  uint8_t* e = q + vecs * 32;
  for (long long i = t; i < (p + bytes - e) / 2; i += nt) reinterpret_cast<uint16_t*>(e)[i] = 0;
}

__global__ void __launch_bounds__(256) clear_kernel(uint8_t* p, long long rows, long long row_bytes, long long ld_bytes) {
  pdl_trigger();
  if (ld_bytes == row_bytes) {
    clear_span(p, rows * row_bytes, blockIdx.x * 256ll + threadIdx.x, gridDim.x * 256ll);
  } else {
    for (long long r = blockIdx.x; r < rows; r += gridDim.x) clear_span(p + r * ld_bytes, row_bytes, threadIdx.x, 256);
  }
}

// ------------------------------------------------------------ the gradient

struct GradArgs {
  const int2* sorted;  // (key, position) by key, n of them
  int n, v, len;       // len: sorted positions per tile
  int tiles;
  const void* g;
  long long ldg;
  long long h;
  float scale;
  void* out;
  long long ldo;
  int accumulate;
  float* part;  // [tiles][2][ldp]: a tile's first run when it began before, its last run when it goes on
  long long ldp;
};

template <typename TO, int VEC>
__device__ __forceinline__ void put_row(const GradArgs& a, int key, long long c, const float (&s)[VEC]) {
  TO* dst = static_cast<TO*>(a.out) + key * a.ldo + c;
  float f[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) f[j] = s[j] * a.scale;
  Vec<TO, VEC> y;
  if (a.accumulate) {
    Vec<TO, VEC> old;
    old.load_own(dst);
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] += old.get(j);
  }
  y.set(f);
  y.store(dst);
}

// One tile per threadIdx.y: its sorted positions in order, four rows of grad_out
// in flight per thread (eight leave fewer warps: 32768 x 2048 bf16 took 110 us,
// 98 us with four). On top of a gradient, the rows that will be read and added
// to are asked for with the rows of grad_out: 8192 tokens on top of 4096 fp32
// columns take 55 us, 72 us without, and 60 us with fp32 adds in L2 instead.
constexpr int kBatch = 4;

template <typename TI, typename TO, int VEC>
__global__ void __launch_bounds__(256) grad_tiles_kernel(const GradArgs a) {
  pdl_trigger();
  pdl_wait();
  const int tile = blockIdx.x * blockDim.y + threadIdx.y;
  const long long c = (static_cast<long long>(blockIdx.y) * blockDim.x + threadIdx.x) * VEC;
  if (tile >= a.tiles || c >= a.h) return;
  const int p0 = tile * a.len, p1 = min(a.n, p0 + a.len);
  const int before = p0 > 0 ? a.sorted[p0 - 1].x : -1;
  const int after = p1 < a.n ? a.sorted[p1].x : -1;
  float s[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) s[j] = 0.f;
  int key = a.sorted[p0].x;
  bool open_left = key == before;  // the current run began in an earlier tile
  float* part = a.part + static_cast<long long>(tile) * 2 * a.ldp + c;
  auto put_part = [&](int which) {
    float* d = part + which * a.ldp;
#pragma unroll
    for (int j = 0; j < VEC; ++j) d[j] = s[j];
  };
  for (int p = p0; p < p1; p += kBatch) {
    int2 kv[kBatch];
    Vec<TI, VEC> x[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) kv[k] = p + k < p1 ? a.sorted[p + k] : make_int2(a.v, 0);
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (kv[k].x < a.v) x[k].load(static_cast<const TI*>(a.g) + kv[k].y * a.ldg + c);
    if (a.accumulate) {
#pragma unroll
      for (int k = 0; k < kBatch; ++k)
        if (kv[k].x < a.v)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const TO*>(a.out) + kv[k].x * a.ldo + c));
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (p + k >= p1) break;
      if (kv[k].x != key) {
        if (open_left) put_part(0);
        else put_row<TO, VEC>(a, key, c, s);
        open_left = false;
        key = kv[k].x;
#pragma unroll
        for (int j = 0; j < VEC; ++j) s[j] = 0.f;
      }
      if (kv[k].x >= a.v) return;  // padding and bad ids end the sorted list
#pragma unroll
      for (int j = 0; j < VEC; ++j) s[j] += x[k].get(j);
    }
  }
  if (open_left) put_part(0);
  else if (key == after) put_part(1);
  else put_row<TO, VEC>(a, key, c, s);
}

// Runs that cross tiles: the tile in which a run begins adds its own partial
// sum (slot 1) and the following tiles' (slot 0), split over the block's
// threadIdx.y groups in contiguous parts that are added in order.
constexpr int kRunX = 64, kRunY = 4;

template <typename TO, int VEC>
__global__ void __launch_bounds__(kRunX* kRunY) grad_runs_kernel(const GradArgs a) {
  __shared__ float sum_s[kRunY][kRunX * VEC];
  pdl_wait();
  const int tile = blockIdx.x;
  const int p0 = tile * a.len, p1 = p0 + a.len;  // p1 < n: the last tile has no block
  const int key = a.sorted[p1 - 1].x, next = a.sorted[p1].x, head = a.sorted[p0].x;
  const int prev = p0 > 0 ? a.sorted[p0 - 1].x : -1;
  if (key >= a.v || next != key) return;     // the last run ends here
  if (head == key && prev == key) return;    // it began earlier
  // tiles [tile + 1, last] hold the rest of the run: those whose first key is this
  // one, looked up side by side
  const int tid = threadIdx.y * kRunX + threadIdx.x;
  int last = tile + 1;
  for (int t0 = tile + 2;; t0 += kRunX * kRunY) {
    const int t = t0 + tid;
    const int more = __syncthreads_count(t < a.tiles && a.sorted[static_cast<long long>(t) * a.len].x == key);
    last += more;
    if (more < kRunX * kRunY) break;
  }
  const int count = last - tile + 1;  // partial sums, this tile's included
  const int each = (count + kRunY - 1) / kRunY;
  const int k0 = threadIdx.y * each, k1 = min(count, k0 + each);
  const long long c = (static_cast<long long>(blockIdx.y) * kRunX + threadIdx.x) * VEC;
  float s[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) s[j] = 0.f;
  if (c < a.h) {
#pragma unroll 4
    for (int k = k0; k < k1; ++k) {
      const float* d = a.part + (static_cast<long long>(tile + k) * 2 + (k == 0 ? 1 : 0)) * a.ldp + c;
#pragma unroll
      for (int j = 0; j < VEC; ++j) s[j] += d[j];
    }
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) sum_s[threadIdx.y][threadIdx.x * VEC + j] = s[j];
  __syncthreads();
  if (threadIdx.y != 0 || c >= a.h) return;
#pragma unroll
  for (int y = 1; y < kRunY; ++y)
#pragma unroll
    for (int j = 0; j < VEC; ++j) s[j] += sum_s[y][threadIdx.x * VEC + j];
  put_row<TO, VEC>(a, key, c, s);
}

// ------------------------------------------------- the gradient, few tokens
// Few tokens need no sort: the block of a token looks through all ids, leaves if
// an earlier token has the same one, and otherwise adds up the rows of all that
// do, in order (split over threadIdx.y in contiguous parts that are added in
// order). One launch after the clearing one, which it overlaps until it writes,
// instead of three. 500 x 1024 on top of fp32 take 6.2 us, 14.5 us sorted; 1000 x
// 512 8.2 and 15.5 us; 2000 x 1000 16.4 and 18.3 us. But a run may be as long as
// the call in one block, so wide rows, which leave no second threadIdx.y to
// share it, stop at half as many tokens. The price is paid where one id fills the
// call: 500 x 1024 27 us, 512 x 4096 and 1024 x 1024 50 us; sorted, 1025 x 1024 of one
// id take 29 us (and 17 us of ids with the skew of text, 10 us here).
constexpr int kFewTokens = 1024;
constexpr int kFewBatch = 8;

template <typename TI, typename TO, int VEC>
__global__ void __launch_bounds__(256) grad_few_kernel(const EmbedGradArgs a) {
  __shared__ int list[kFewTokens];
  __shared__ int warp_n[8];
  __shared__ float sum_s[256 * VEC];
  const int i = blockIdx.x, n = static_cast<int>(a.n);
  const int tid = threadIdx.y * blockDim.x + threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t id = a.ids[i];
  if (a.has_padding && id == a.padding_id) return pdl_wait();  // every exit: the grid ends after the clearing
  if (id < 0 || id >= a.v) {
    if (tid == 0) atomicExch(a.bad, DEV_ID_RANGE);
    return pdl_wait();
  }
  int count = 0;
  for (int j0 = 0; j0 < n; j0 += 256) {
    const int j = j0 + tid;
    const bool same = j < n && a.ids[j] == id;
    const uint32_t votes = __ballot_sync(0xffffffffu, same);
    if (lane == 0) warp_n[warp] = __popc(votes);
    __syncthreads();
    int at = count;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      if (w < warp) at += warp_n[w];
      count += warp_n[w];
    }
    if (same) list[at + __popc(votes & ((1u << lane) - 1))] = j;
    __syncthreads();
    if (count > 0 && list[0] < i) return pdl_wait();  // an earlier token's block does it
  }
  const int each = (count + blockDim.y - 1) / blockDim.y;
  const int k0 = threadIdx.y * each, k1 = min(count, k0 + each);
  const long long c = (static_cast<long long>(blockIdx.y) * blockDim.x + threadIdx.x) * VEC;
  float s[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) s[j] = 0.f;
  if (c < a.h) {
    for (int k = k0; k < k1; k += kFewBatch) {
      Vec<TI, VEC> x[kFewBatch];
#pragma unroll
      for (int b = 0; b < kFewBatch; ++b)
        if (k + b < k1) x[b].load(static_cast<const TI*>(a.g) + list[k + b] * a.ldg + c);
#pragma unroll
      for (int b = 0; b < kFewBatch; ++b)
        if (k + b < k1)
#pragma unroll
          for (int j = 0; j < VEC; ++j) s[j] += x[b].get(j);
    }
  }
  if (blockDim.y > 1) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum_s[tid * VEC + j] = s[j];
    __syncthreads();
    if (threadIdx.y != 0) return pdl_wait();
    for (int y = 1; y < static_cast<int>(blockDim.y); ++y)
#pragma unroll
      for (int j = 0; j < VEC; ++j) s[j] += sum_s[(y * blockDim.x + threadIdx.x) * VEC + j];
  }
  pdl_wait();  // the rows are cleared
  if (c >= a.h) return;
  GradArgs o{};
  o.scale = a.scale;
  o.out = a.out;
  o.ldo = a.ldo;
  o.accumulate = a.accumulate;
  put_row<TO, VEC>(o, static_cast<int>(id), c, s);
}

// Largest VEC (8, 4, 2, 1 elements, 16 bytes of the first matrix) such that
// rows and their pieces are aligned for both matrices: VEC divides h, and VEC
// elements (at most 16 bytes of them at a time) divide the address and the
// leading dimension.
int pick_vec(long long h, const void* a, long long lda, int esa, const void* b, long long ldb, int esb) {
  for (int vec = 16 / esa; vec > 1; vec /= 2) {
    auto ok = [vec](const void* p, long long ld, int es) {
      const long long bytes = std::min(16, vec * es);
      return reinterpret_cast<uintptr_t>(p) % bytes == 0 && ld * es % bytes == 0;
    };
    if (h % vec == 0 && ok(a, lda, esa) && ok(b, ldb, esb)) return vec;
  }
  return 1;
}

// Threads along a row: a power of two, at least a warp, no more than 256 or
// than the row needs at `each` vectors per thread.
int row_threads(long long h, int vec, int each) {
  int x = 32;
  while (x < 256 && static_cast<long long>(x) * vec * each < h) x *= 2;
  return x;
}

template <typename TI, typename TO, int VEC>
void embed_t(const EmbedArgs& a, cudaStream_t st) {
  // four vectors of a row in flight per thread; with few rows all threads of a block on one row
  const int x = row_threads(a.h, VEC, a.n < 592 ? 1 : 4), y = 256 / x;
  embed_kernel<TI, TO, VEC><<<static_cast<unsigned>((a.n + y - 1) / y), dim3(x, y), 0, st>>>(
      static_cast<const TI*>(a.table), a.ld, a.v, a.h, a.ids, a.n, a.scale, static_cast<TO*>(a.out), a.ldo, a.bad);
}

template <typename TI, typename TO, int VEC>
cudaError_t grad_t(const GradArgs& a, cudaStream_t st) {
  const int x = row_threads(a.h, VEC, 1), y = 256 / x;
  auto groups = [&a](long long cols) { return static_cast<unsigned>((a.h + cols - 1) / cols); };
  cudaError_t e = launch_pdl(grad_tiles_kernel<TI, TO, VEC>,
                             dim3((a.tiles + y - 1) / y, groups(static_cast<long long>(x) * VEC)), dim3(x, y), 0, st, a);
  if (e != cudaSuccess || a.tiles < 2) return e;
  return launch_pdl(grad_runs_kernel<TO, VEC>, dim3(a.tiles - 1, groups(kRunX * VEC)), dim3(kRunX, kRunY), 0, st, a);
}

template <typename TI, typename TO, int VEC>
cudaError_t few_t(const EmbedGradArgs& a, bool after_clear, cudaStream_t st) {
  const int x = row_threads(a.h, VEC, 1);
  const long long cols = static_cast<long long>(x) * VEC;
  const dim3 grid(static_cast<unsigned>(a.n), static_cast<unsigned>((a.h + cols - 1) / cols)), block(x, 256 / x);
  if (after_clear) return launch_pdl(grad_few_kernel<TI, TO, VEC>, grid, block, 0, st, a);
  grad_few_kernel<TI, TO, VEC><<<grid, block, 0, st>>>(a);
  return cudaGetLastError();
}

template <typename F>
void by_types(int in_bf16, int out_bf16, int vec, const F& f) {
  auto go = [&](auto ti, auto to) {
    using TI = decltype(ti);
    using TO = decltype(to);
    if constexpr (sizeof(TI) == 2) {  // 16 bytes of the first matrix at most (pick_vec)
      if (vec == 8) return f.template operator()<TI, TO, 8>();
    }
    if (vec == 4) f.template operator()<TI, TO, 4>();
    else if (vec == 2) f.template operator()<TI, TO, 2>();
    else f.template operator()<TI, TO, 1>();
  };
  if (in_bf16 && out_bf16) go(uint16_t{}, uint16_t{});
  else if (in_bf16) go(uint16_t{}, float{});
  else if (out_bf16) go(float{}, uint16_t{});
  else go(float{}, float{});
}

struct EmbedCall {
  const EmbedArgs& a;
  cudaStream_t st;
  template <typename TI, typename TO, int VEC>
  void operator()() const {
    embed_t<TI, TO, VEC>(a, st);
  }
};
struct GradCall {
  const GradArgs& a;
  cudaStream_t st;
  cudaError_t* e;
  template <typename TI, typename TO, int VEC>
  void operator()() const {
    *e = grad_t<TI, TO, VEC>(a, st);
  }
};

// Sorted positions per tile: long tiles leave fewer partial sums and fewer
// blocks that look for runs, so the longest that gives the SMs 24 warps each
// (8192 x 4096 bf16: 32, 200 us with the clearing; 16 and 64 204 us), and no more
// than 2048 tiles where longer ones can be had (65536 x 256: 32, 82 us; 16 90 us).
int tile_len(long long n, long long h, int vec) {
  const long long warps = (h + 32 * vec - 1) / (32 * vec);  // per tile
  int len = 64;
  while (len > 8 && (n + len - 1) / len * warps < 148 * 24 && (n + len / 2 - 1) / (len / 2) <= 2048) len /= 2;
  return len;
}

struct EmbedGradLayout {
  size_t buf0, buf1, part, total;
  long long ldp;
  int tiles, len, vec;
};
EmbedGradLayout grad_layout(const EmbedGradArgs& a) {
  EmbedGradLayout L;
  const long long n = a.n, h = a.h;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  L.vec = pick_vec(h, a.g, a.ldg, a.in_bf16 ? 2 : 4, a.out, a.ldo, a.out_bf16 ? 2 : 4);
  L.len = tile_len(n, h, L.vec);
  L.tiles = static_cast<int>((n + L.len - 1) / L.len);
  L.ldp = (h + 7) / 8 * 8;
  L.buf0 = 0;
  L.buf1 = up(n * sizeof(int2));
  L.part = L.buf1 + up(n * sizeof(int2));
  L.total = L.part + up(static_cast<size_t>(L.tiles) * 2 * L.ldp * sizeof(float));
  return L;
}

// Which of the two gradients takes the call.
bool few_tokens(const EmbedGradArgs& a, int vec) {
  return a.n <= kFewTokens / 2 || (a.n <= kFewTokens && row_threads(a.h, vec, 1) <= 128);
}

}  // namespace

void launch_embed(const EmbedArgs& a, cudaStream_t st) {
  if (a.n == 0 || a.h == 0) return;
  const int vec = pick_vec(a.h, a.table, a.ld, a.in_bf16 ? 2 : 4, a.out, a.ldo, a.out_bf16 ? 2 : 4);
  by_types(a.in_bf16, a.out_bf16, vec, EmbedCall{a, st});
}

struct FewCall {
  const EmbedGradArgs& a;
  bool after_clear;
  cudaStream_t st;
  cudaError_t* e;
  template <typename TI, typename TO, int VEC>
  void operator()() const {
    *e = few_t<TI, TO, VEC>(a, after_clear, st);
  }
};

// beside_clear: next to the clearing kernel, which reads and writes none of the sort's data.
template <int THREADS>
cudaError_t launch_sort(const SortArgs& s, bool beside_clear, cudaStream_t st) {
  static std::mutex mu;
  static uint64_t ready = 0;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!(ready >> (dev & 63) & 1)) {
      e = cudaFuncSetAttribute(sort_kernel<THREADS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               static_cast<int>(sort_smem_bytes(THREADS, kMaxDigitBits)));
      if (e != cudaSuccess) return e;
      ready |= 1ull << (dev & 63);
    }
  }
  const size_t smem = sort_smem_bytes(THREADS, s.digit_bits);
  if (beside_clear) return launch_pdl(sort_kernel<THREADS>, dim3(kSortCtas), dim3(THREADS), smem, st, s);
  sort_kernel<THREADS><<<kSortCtas, THREADS, smem, st>>>(s);
  return cudaGetLastError();
}

size_t embed_grad_workspace(const EmbedGradArgs& a) {
  const EmbedGradLayout L = grad_layout(a);
  return few_tokens(a, L.vec) ? 0 : L.total;
}

cudaError_t launch_embed_grad(const EmbedGradArgs& a, void* ws, int num_sms, cudaStream_t st, int* launches) {
  if (a.n == 0 && a.accumulate) return cudaSuccess;
  const int es_out = a.out_bf16 ? 2 : 4;
  if (!a.accumulate) {
    const long long bytes = a.v * a.h * es_out;
    const long long blocks = std::max<long long>(1, std::min<long long>((bytes + 8191) / 8192, num_sms * kClearBlocks));
    clear_kernel<<<static_cast<unsigned>(blocks), 256, 0, st>>>(static_cast<uint8_t*>(a.out), a.v, a.h * es_out,
                                                                a.ldo * es_out);
    *launches += 1;
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || a.n == 0) return e;
  }
  const EmbedGradLayout L = grad_layout(a);
  if (few_tokens(a, L.vec)) {
    cudaError_t e = cudaSuccess;
    by_types(a.in_bf16, a.out_bf16, L.vec, FewCall{a, !a.accumulate, st, &e});
    *launches += 1;
    return e;
  }
  uint8_t* w = static_cast<uint8_t*>(ws);
  SortArgs s{};
  s.ids = a.ids;
  s.n = static_cast<int>(a.n);
  s.v = static_cast<int>(a.v);
  s.padding_id = a.padding_id;
  s.has_padding = a.has_padding;
  int bits = 1;
  while ((a.v >> bits) != 0) ++bits;  // keys 0..v
  s.passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
  s.digit_bits = (bits + s.passes - 1) / s.passes;
  s.buf0 = reinterpret_cast<int2*>(w + L.buf0);
  s.buf1 = reinterpret_cast<int2*>(w + L.buf1);
  s.bad = a.bad;
  cudaError_t e = a.n <= kFewIds ? launch_sort<512>(s, !a.accumulate, st) : launch_sort<1024>(s, !a.accumulate, st);
  if (e != cudaSuccess) return e;
  *launches += 1;
  GradArgs g{};
  g.sorted = s.passes & 1 ? s.buf1 : s.buf0;
  g.n = s.n;
  g.v = s.v;
  g.len = L.len;
  g.tiles = L.tiles;
  g.g = a.g;
  g.ldg = a.ldg;
  g.h = a.h;
  g.scale = a.scale;
  g.out = a.out;
  g.ldo = a.ldo;
  g.accumulate = a.accumulate;
  g.part = reinterpret_cast<float*>(w + L.part);
  g.ldp = L.ldp;
  by_types(a.in_bf16, a.out_bf16, L.vec, GradCall{g, st, &e});
  *launches += L.tiles > 1 ? 2 : 1;
  return e;
}

}  // namespace orda
