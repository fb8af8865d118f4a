// linear_ce.cu -- row kernels of the linear softmax cross entropy
// (orda_linear_cross_entropy_device); its products run in gemm_sm100.cu.
//
// With z = h W^T, y the label, a the label smoothing and g the loss scale:
//   lse = log sum_v e^{z_v}
//   nll = (1 - a) (lse - z_y) + a (lse - mean_v z_v)
//   dz_v = e^{z_v - lse} - (1 - a) [v = y] - a / V,  dh = g dz W,  dW = g dz^T h
// (g after the products: in dz it would round one factor of every row, 1 / the
// count of tokens, to bf16)
// The label's logit is the reference of its row: the logits product sums
// Z_o = sum_{v != y} e^{z_v - z_y} per 64-column part, so that
//   lse - z_y = log(1 + Z_o),  1 - p_y = Z_o / (1 + Z_o)
// lose nothing to cancellation when the label's probability nears 1. A label's
// logit below -2.36e38 (a masked entry), whose base-2 exponent fp32 does not hold,
// is held as -FLT_MAX: an infinite reference would turn the parts that keep it
// into NaN. The loss of such a row comes from the logit itself.
//
// The label's logit is a rounded fp32 sum; the other logits are the tensor cores'
// fp32 sums over at most 2048 of K at a time, added in fp32: exact where fp32 holds
// the sums, else too small by up to 2e-6 of themselves on average (see kCeKBlocks in
// gemm_sm100.cu). No factor undoes that average: it would be an error of its own
// size wherever nothing was cut. The recomputed pieces' gradients, which are
// rounded to bf16, sum K in one.
//
// Between the logits product and the two gradient products the logits of a
// piece are kept as 16-bit fixed point, t = log2 e^{z - z_y} in steps of
// 2^-9 over (-64, 64), and 0 below (a part whose own sum is under 2^-40 is
// kept against its own maximum, so 0 stands for less than 2^-16 of a part's
// largest probability): an error of at most 2^-10 ln 2 = 6.8e-4 (3.9e-4 rms) of
// each probability, where the bf16 rounding of the gradient operand that
// follows is at most 2^-8 = 3.9e-3 (1.6e-3 rms). It takes half the bytes of
// fp32 logits; the statistics are fp32 and come from the accumulators.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cstdint>

#include "kernels.h"
#include "ptx.cuh"

namespace orda {
namespace {

constexpr float kLog2E = 1.4426950408889634f;
constexpr double kLn2 = 0.6931471805599453;
constexpr float kLn2f = 0.6931471805599453f;

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// One block per token: the label's logit (fp32 products and sums of the bf16
// operands) and a copy of the hidden state in which an ignored token is zero,
// so that whatever an ignored row holds (NaN and infinities of padding
// included) reaches no product. Bound by bandwidth: 3 rows of H bf16 each.
constexpr int kPrepThreads = 128;

__global__ void __launch_bounds__(kPrepThreads) ce_prep_kernel(const CeArgs a) {
  const long long row = blockIdx.x;
  pdl_trigger();
  const bool token = row < a.bt;
  const int64_t y = token ? a.labels[row] : a.ignore_index;
  bool live = token && y != a.ignore_index;
  if (row == 0 && threadIdx.x == 0) {
    const int old = *a.status;
    if (old != DEV_OK && !(old & kStatusReported)) *(old == DEV_LABEL_RANGE ? a.bad_label : a.earlier) = old;
    *a.status = DEV_OK;
  }
  if (live && (y < 0 || y >= a.v)) {
    if (threadIdx.x == 0) *a.bad_label = DEV_LABEL_RANGE;
    live = false;
  }
  const uint16_t* h = static_cast<const uint16_t*>(a.h) + row * a.ldh;
  const uint16_t* w = static_cast<const uint16_t*>(a.w) + (live ? y : 0) * a.ldw;
  uint16_t* out = a.h_clean + row * a.ld_clean;
  const int nvec = static_cast<int>(a.hd / 8);
  float s = 0.f;
  if (live) {
#pragma unroll 4
    for (int i = threadIdx.x; i < nvec; i += kPrepThreads) {
      const uint4 p = __ldcs(reinterpret_cast<const uint4*>(h) + i);
      const uint4 q = *(reinterpret_cast<const uint4*>(w) + i);
      reinterpret_cast<uint4*>(out)[i] = p;
      const uint32_t pw[4] = {p.x, p.y, p.z, p.w}, qw[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        s = fmaf(bf16_lo(pw[k]), bf16_lo(qw[k]), s);
        s = fmaf(bf16_hi(pw[k]), bf16_hi(qw[k]), s);
      }
    }
    for (long long i = 8ll * nvec + threadIdx.x; i < a.hd; i += kPrepThreads) {
      out[i] = h[i];
      s = fmaf(bf16_lo(h[i]), bf16_lo(w[i]), s);
    }
  } else {
    for (int i = threadIdx.x; i < nvec; i += kPrepThreads) reinterpret_cast<uint4*>(out)[i] = make_uint4(0, 0, 0, 0);
    for (long long i = 8ll * nvec + threadIdx.x; i < a.hd; i += kPrepThreads) out[i] = 0;
  }
  if (!token) return;
  s = warp_sum(s);
  __shared__ float part[kPrepThreads / 32];
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    float x = 0.f;
#pragma unroll
    for (int k = 0; k < kPrepThreads / 32; ++k) x += part[k];
    const float x2 = x * kLog2E;
    a.ref[row] = make_float2(!live ? 0.f : x2 < -FLT_MAX ? -FLT_MAX : x2, __int_as_float(live ? static_cast<int>(y) : -1));
    a.nll[row] = x;
    if (live) atomicAdd(a.count, 1);
  }
}

__global__ void mark_reported_kernel(int* word, int status) { atomicCAS(word, status, status | kStatusReported); }

// Sum of 2^(r_i) * d_i with a running maximum of the references r_i.
struct Acc {
  double d;
  float r;
};
__device__ __forceinline__ void acc_add(Acc& a, double d, float r) {
  // equal references, the usual case, add without a factor
  if (r == a.r) {
    a.d += d;
  } else if (d != 0.0) {
    if (!(r <= a.r)) {
      a.d = (a.d == 0.0 ? 0.0 : a.d * exp2(static_cast<double>(a.r) - static_cast<double>(r))) + d;
      a.r = r;
    } else {
      a.d += d * exp2(static_cast<double>(r) - static_cast<double>(a.r));
    }
  }
}

// The row's loss and gradient constants from its parts' sum m; every block of
// the row does the same. Results are fp32, and so is the arithmetic where no
// two large numbers cancel.
struct RowResult {
  float4 c;  // -lse log2 e, label, a / V, the label's gradient
  float nll, lse;
};

__device__ __forceinline__ RowResult row_result(const CeArgs& a, float2 ref, float zy, const Acc& m, float sx) {
  RowResult r;
  float gap, miss, l;  // lse - z_y, 1 - p_y and lse
  if (m.r == ref.x && ref.x <= -FLT_MAX) {
    // every logit lies below -2.36e38: the exponents do not hold their differences
    gap = miss = l = NAN;
  } else if (m.r == ref.x) {
    const float z = static_cast<float>(m.d);
    gap = log1pf(z);
    miss = z < INFINITY ? z / (1.f + z) : 1.f;
    l = fmaf(ref.x, kLn2f, gap);
  } else {
    const double up = static_cast<double>(m.r) - static_cast<double>(ref.x);
    const double own = exp2(-up);  // the label's term next to m.d
    const double lg = log(m.d + own);
    const double lse = static_cast<double>(m.r) * kLn2 + lg;
    gap = static_cast<float>(ref.x > -FLT_MAX ? up * kLn2 + lg : lse - static_cast<double>(zy));
    miss = static_cast<float>(m.d / (m.d + own));
    l = static_cast<float>(lse);
  }
  const float uni = a.alpha / static_cast<float>(a.v);
  r.nll = a.alpha > 0.f ? (1.f - a.alpha) * gap + a.alpha * (l - sx / static_cast<float>(a.v)) : gap;
  r.lse = l;
  r.c.x = -l * kLog2E;
  r.c.y = ref.y;
  r.c.z = uni;
  r.c.w = a.alpha - uni - miss;
  return r;
}

// The count of tokens that the mean divides by (1 for a sum).
__device__ __forceinline__ double loss_denominator(const CeArgs& a) {
  if (a.reduction_sum) return 1.0;
  return static_cast<double>(a.denom_override > 0 ? a.denom_override : max(*static_cast<volatile int*>(a.count), 1));
}

// One block per row, or several along the columns where the rows are few:
//   * the row's records (coalesced, 8 bytes per 64 columns) -> constants;
//   * 16-bit logits -> bf16 logit gradients, in place: 2^(t + off) - a / V with
//     off = (the part's reference - lse) log2 e. Bound by bandwidth, 4 bytes
//     per element; a thread holds 8 neighbouring columns, and the first loads
//     are under way while the constants are formed.
// The block that ends last sums the losses in row order.
constexpr int kRowThreads = 256;
constexpr int kRowSteps = 4;
constexpr int kRowChunk = kRowThreads * 8 * kRowSteps;

__global__ void __launch_bounds__(kRowThreads) ce_rows_kernel(const CeArgs a, uint16_t* piece, long long ld, long long n,
                                                              int segs, long long seg_cols) {
  __shared__ Acc acc_s[kRowThreads];
  __shared__ double d_s[kRowThreads / 32], x_s[kRowThreads / 32];
  __shared__ float4 const_s;
  __shared__ bool last;
  pdl_trigger();
  pdl_wait();
  const long long row = blockIdx.x / segs;
  const int seg = static_cast<int>(blockIdx.x - row * segs);
  const long long c0 = seg * seg_cols, c1 = min(n, c0 + seg_cols);
  uint16_t* base = piece + row * ld;
  const float2* rec = a.rec + row * a.rec_ld;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  uint4 v[kRowSteps];
  auto load = [&](long long at) {
#pragma unroll
    for (int i = 0; i < kRowSteps; ++i) {
      const long long col = at + i * (kRowThreads * 8) + threadIdx.x * 8;
      if (col < c1) v[i] = __ldcs(reinterpret_cast<const uint4*>(base + col));
    }
  };
  if (c0 < c1) load(c0);

  const float2 ref = a.ref[row];
  const bool live = __float_as_int(ref.y) >= 0;
  // parts against the row's reference, the usual case, are a plain sum
  double d = 0.0, sx = 0.0;
  bool other = false;
  if (live) {
#pragma unroll 4
    for (int p = threadIdx.x; p < a.n_parts; p += kRowThreads) {
      const float2 c = rec[p];
      d += static_cast<double>(c.x);
      other |= c.y != ref.x;
    }
    if (a.alpha > 0.f) {
#pragma unroll 4
      for (int p = threadIdx.x; p < a.n_parts; p += kRowThreads) sx += static_cast<double>(a.sx[row * a.rec_ld + p]);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    d += __shfl_xor_sync(0xffffffffu, d, o);
    if (a.alpha > 0.f) sx += __shfl_xor_sync(0xffffffffu, sx, o);
  }
  if (lane == 0) {
    d_s[warp] = d;
    x_s[warp] = sx;
  }
  const bool mixed = __syncthreads_or(other);
  if (mixed) {
    Acc acc{0.0, ref.x};
    for (int p = threadIdx.x; p < a.n_parts; p += kRowThreads) {
      const float2 c = rec[p];
      acc_add(acc, static_cast<double>(c.x), c.y);
    }
    acc_s[threadIdx.x] = acc;
    __syncthreads();
    for (int o = kRowThreads / 2; o > 0; o >>= 1) {
      if (static_cast<int>(threadIdx.x) < o) {
        Acc m = acc_s[threadIdx.x];
        acc_add(m, acc_s[threadIdx.x + o].d, acc_s[threadIdx.x + o].r);
        acc_s[threadIdx.x] = m;
      }
      __syncthreads();
    }
  }
  if (threadIdx.x == 0) {
    RowResult r{make_float4(-INFINITY, __int_as_float(-1), 0.f, 0.f), 0.f, 0.f};
    if (live) {
      Acc m{0.0, ref.x};
      double x = 0.0;
#pragma unroll
      for (int w = 0; w < kRowThreads / 32; ++w) {
        m.d += d_s[w];
        x += x_s[w];
      }
      if (mixed) m = acc_s[0];
      // a.nll holds the label's logit until seg 0 replaces it; only that block's loss is used
      r = row_result(a, ref, seg == 0 ? a.nll[row] : 0.f, m, static_cast<float>(x));
    }
    const_s = r.c;
    if (seg == 0) {
      a.row_const[row] = r.c;
      a.nll[row] = r.nll;
      if (a.lse) a.lse[row] = r.lse;
      if (row == 0) *a.scale = static_cast<float>(1.0 / loss_denominator(a));
      __threadfence();
    }
  }
  __syncthreads();
  const float4 c = const_s;

  if (c0 < c1) {
    const int label = __float_as_int(c.y);  // -1: none
    const int label8 = label < 0 ? -1 : label & ~7, label_in = label & 7;
    for (long long at = c0; at < c1; at += kRowChunk) {
      if (at > c0) load(at);
#pragma unroll
      for (int i = 0; i < kRowSteps; ++i) {
        const long long col = at + i * (kRowThreads * 8) + threadIdx.x * 8;
        if (col >= c1) continue;
        // 2^(t + off) = 2^(t - 62.5) 2^(off + 62.5): the first factor is an exact
        // argument from u's bits (2^23 + u as a float, over 512, less the bias), and
        // flushes to zero for code 0, so the code needs no test of its own
        const float up = ex2(rec[col >> a.part_shift].y + (c.x + 62.5f));
        uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          constexpr float kBias = -(8388608.0f + kCeQBias) / kCeQScale - 62.5f;
          const float x0 = fmaf(__uint_as_float(__byte_perm(w[k], 0x4B000000u, 0x7610)), 1.0f / kCeQScale, kBias);
          const float x1 = fmaf(__uint_as_float(__byte_perm(w[k], 0x4B000000u, 0x7632)), 1.0f / kCeQScale, kBias);
          const __nv_bfloat162 b = __floats2bfloat162_rn(fmaf(ex2(x0), up, -c.z), fmaf(ex2(x1), up, -c.z));
          w[k] = *reinterpret_cast<const uint32_t*>(&b);
        }
        if (col == label8) {
          const uint32_t dy = __bfloat16_as_ushort(__float2bfloat16_rn(c.w));
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (2 * k == label_in) w[k] = (w[k] & 0xffff0000u) | dy;
            if (2 * k + 1 == label_in) w[k] = (w[k] & 0xffffu) | (dy << 16);
          }
        }
        *reinterpret_cast<uint4*>(base + col) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }

  // every block has read the count of live tokens when the last one is here
  if (threadIdx.x == 0) last = atomicAdd(a.done, 1) == static_cast<int>(gridDim.x) - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double s = 0.0;
#pragma unroll 4
  for (long long i = threadIdx.x; i < a.bt; i += kRowThreads) s += static_cast<double>(__ldcg(a.nll + i));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) d_s[warp] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int w = 0; w < kRowThreads / 32; ++w) s += d_s[w];
    *a.loss = static_cast<float>(s / loss_denominator(a));
    *a.count = 0;
    *a.done = 0;
  }
}

// scale times the sum over K slabs, in slab order, and the output's type.
template <bool BF16>
__global__ void __launch_bounds__(256)
    slab_sum_kernel(const float* __restrict__ buf, int slabs, long long slab_rows, long long ldb, long long rows,
                    long long cols, const float* scale, void* out, long long ldo, int vec_ok) {
  pdl_trigger();
  pdl_wait();
  const float g = *scale;
  const long long groups = (cols + 3) / 4;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < rows * groups; i += gridDim.x * 256ll) {
    const long long r = i / groups, c = (i - r * groups) * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int k = 0; k < slabs; ++k) {
      const float4 x = *reinterpret_cast<const float4*>(buf + (k * slab_rows + r) * ldb + c);
      s.x += x.x;
      s.y += x.y;
      s.z += x.z;
      s.w += x.w;
    }
    s = make_float4(g * s.x, g * s.y, g * s.z, g * s.w);
    const float f[4] = {s.x, s.y, s.z, s.w};
    if (BF16) {
      __nv_bfloat16* o = static_cast<__nv_bfloat16*>(out) + r * ldo + c;
      if (vec_ok && c + 4 <= cols) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(f[0], f[1]), hi = __floats2bfloat162_rn(f[2], f[3]);
        *reinterpret_cast<uint2*>(o) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
      } else {
        for (int k = 0; k < 4 && c + k < cols; ++k) o[k] = __float2bfloat16_rn(f[k]);
      }
    } else {
      float* o = static_cast<float*>(out) + r * ldo + c;
      if (vec_ok && c + 4 <= cols) *reinterpret_cast<float4*>(o) = s;
      else
        for (int k = 0; k < 4 && c + k < cols; ++k) o[k] = f[k];
    }
  }
}

}  // namespace

cudaError_t launch_ce_prep(const CeArgs& a, cudaStream_t stream) {
  ce_prep_kernel<<<static_cast<unsigned>(a.clean_rows), kPrepThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_mark_reported(int* word, int status, cudaStream_t stream) {
  mark_reported_kernel<<<1, 1, 0, stream>>>(word, status);
  return cudaGetLastError();
}

// Several blocks per row, of 8192 columns at least, while that gives the SMs up to eight blocks each.
cudaError_t launch_ce_rows(const CeArgs& a, uint16_t* piece, long long ld, long long n, cudaStream_t stream) {
  long long segs = std::max<long long>(1, std::min((148 * 8) / a.bt, n / kRowChunk));
  const long long seg_cols = ((n + segs - 1) / segs + kRowThreads * 8 - 1) / (kRowThreads * 8) * (kRowThreads * 8);
  return launch_pdl(ce_rows_kernel, dim3(static_cast<unsigned>(a.bt * segs)), dim3(kRowThreads), 0, stream, a, piece,
                    ld, n, static_cast<int>(segs), seg_cols);
}

cudaError_t launch_slab_sum(const float* buf, int slabs, long long slab_rows, long long ldb, long long rows,
                            long long cols, const float* scale, void* out, long long ldo, int out_bf16,
                            cudaStream_t stream) {
  const long long n = rows * ((cols + 3) / 4);
  const unsigned blocks = static_cast<unsigned>(std::min<long long>((n + 255) / 256, 148 * 16));
  const int esz = out_bf16 ? 2 : 4;
  const int vec_ok = reinterpret_cast<uintptr_t>(out) % (4 * esz) == 0 && ldo % 4 == 0;
  return launch_pdl(out_bf16 ? slab_sum_kernel<true> : slab_sum_kernel<false>, dim3(blocks), dim3(256), 0, stream, buf,
                    slabs, slab_rows, ldb, rows, cols, scale, out, ldo, vec_ok);
}

}  // namespace orda
