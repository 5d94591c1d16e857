// Layer norm over rows of C channels, with a scale and shift per contiguous segment of
// rows (the DiT's adaLN modulation of a packed sequence), forward and backward.
//
//   xhat = (x - mean) * rstd,  y = xhat * w + b,   w = weight, or 1 + weight (modulate)
//   a = dy * w,  dx = rstd * (a - mean(a) - xhat * mean(a * xhat))
//   dw = sum over the segment's rows of dy * xhat,  db = sum of dy
//
// Bound by HBM: every row is read once and written once.  A row is held in registers by
// one wave (short rows) or one workgroup, 8 consecutive channels per thread and step;
// a workgroup walks consecutive rows of one segment, so that the segment's weights, and
// in the backward pass the sums of dw and db, stay in registers (past 8192 channels the
// backward pass keeps 50 to 249 of them in scratch memory).  Those sums leave as
// one fp32 partial row per workgroup and are added by a second kernel in a fixed order.
// Statistics and sums are fp32; the variance is taken about the row's own mean.
#include "h3a_device.h"
#include "h3a_internal.h"

namespace h3a {

namespace {

// 8 channels of a row, as they are in memory, and as floats.
template <int DT>
struct Row8 {
  static constexpr int kBytes = DT == H3A_FP32 ? 4 : 2;
  u32x4 v[DT == H3A_FP32 ? 2 : 1];
};

template <int DT>
__device__ __forceinline__ float element(const char *p, int64_t i) {
  if constexpr (DT == H3A_FP32) return reinterpret_cast<const float *>(p)[i];
  else if constexpr (DT == H3A_FP16) return (float)reinterpret_cast<const _Float16 *>(p)[i];
  else return __uint_as_float((uint32_t)reinterpret_cast<const uint16_t *>(p)[i] << 16);
}

template <int DT>
__device__ __forceinline__ void unpack(const Row8<DT> &r, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == H3A_FP32) {
      x[i] = __uint_as_float(r.v[0][i]);
      x[i + 4] = __uint_as_float(r.v[1][i]);
    } else if constexpr (DT == H3A_FP16) {
      typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
      const f16x2 h = __builtin_bit_cast(f16x2, (uint32_t)r.v[0][i]);
      x[2 * i] = (float)h.x;
      x[2 * i + 1] = (float)h.y;
    } else {
      x[2 * i] = bf16_lo(r.v[0][i]);
      x[2 * i + 1] = bf16_hi(r.v[0][i]);
    }
  }
}

// Channels c .. c+7 of a row of C; those past the end are 0.  VEC: C is a multiple of 8
// and rows are 16-byte aligned; otherwise whole eights are read and written as 16-byte
// accesses off their grid (which global memory takes) and a row's end one by one (60000
// rows of 1001 bf16 channels, forward: 136 us with every channel by itself).
template <int DT>
__device__ __forceinline__ int64_t byte_of(int c) { return (int64_t)c * Row8<DT>::kBytes; }
template <int DT, bool VEC>
__device__ __forceinline__ Row8<DT> load8(const char *row, int c, int C) {
  Row8<DT> r;
  constexpr int kVecs = sizeof(r.v) / sizeof(r.v[0]);
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
      r.v[i] = c < C ? *reinterpret_cast<const u32x4 *>(row + byte_of<DT>(c) + 16 * i) : u32x4{0, 0, 0, 0};
  } else if (c + 8 <= C) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) __builtin_memcpy(&r.v[i], row + byte_of<DT>(c) + 16 * i, 16);
  } else if constexpr (DT == H3A_FP32) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      r.v[i >> 2][i & 3] = c + i < C ? reinterpret_cast<const uint32_t *>(row)[c + i] : 0u;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t *p = reinterpret_cast<const uint16_t *>(row) + c + 2 * i;
      const uint32_t lo = c + 2 * i < C ? p[0] : 0u, hi = c + 2 * i + 1 < C ? p[1] : 0u;
      r.v[0][i] = lo | hi << 16;
    }
  }
  return r;
}

template <int DT, bool VEC>
__device__ __forceinline__ void store8(char *row, int c, int C, const float (&x)[8]) {
  Row8<DT> r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == H3A_FP32) {
      r.v[0][i] = __float_as_uint(x[i]);
      r.v[1][i] = __float_as_uint(x[i + 4]);
    } else if constexpr (DT == H3A_FP16) {
      typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
      r.v[0][i] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)x[2 * i], (_Float16)x[2 * i + 1]});
    } else {
      r.v[0][i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
    }
  }
  constexpr int kVecs = sizeof(r.v) / sizeof(r.v[0]);
  if constexpr (VEC) {
    if (c < C) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i) *reinterpret_cast<u32x4 *>(row + byte_of<DT>(c) + 16 * i) = r.v[i];
    }
  } else if (c + 8 <= C) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) __builtin_memcpy(row + byte_of<DT>(c) + 16 * i, &r.v[i], 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (c + i >= C) break;
      if constexpr (DT == H3A_FP32) reinterpret_cast<uint32_t *>(row)[c + i] = r.v[i >> 2][i & 3];
      else reinterpret_cast<uint16_t *>(row)[c + i] = (uint16_t)(r.v[0][i >> 1] >> (16 * (i & 1)));
    }
  }
}

// A weight or bias row (bf16, fp16 or fp32, any alignment) as floats; it is read once
// per workgroup and segment.
__device__ __forceinline__ void load_affine(const void *p, int dt, int64_t row, int c, int C, float otherwise,
                                            float add, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (!p || c + i >= C) {
      x[i] = otherwise;
    } else {
      const char *b = static_cast<const char *>(p);
      const int64_t at = row * C + c + i;
      x[i] = add + (dt == H3A_FP32 ? element<H3A_FP32>(b, at)
                                   : dt == H3A_FP16 ? element<H3A_FP16>(b, at) : element<H3A_BF16>(b, at));
    }
  }
}

// Sums of two values over the TPR threads of a row, on all of them.  `slot` alternates
// between rows, so that one barrier per row suffices.
template <int TPR>
__device__ __forceinline__ float2 row_sum(float2 v, float2 (*xch)[4], int slot) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    v.x += __shfl_xor(v.x, o);
    v.y += __shfl_xor(v.y, o);
  }
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) xch[slot][threadIdx.x >> 6] = v;
    __syncthreads();
    v = xch[slot][0];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      v.x += xch[slot][w].x;
      v.y += xch[slot][w].y;
    }
  }
  return v;
}

// The workgroup's segment, and its rows [r0, r1) in it.
struct Share {
  int seg, r0, r1;
};
__device__ __forceinline__ Share share_of(const NormArgs &a) {
  const int w = blockIdx.x;
  int s = 0;
  while (s + 1 < a.segments && w >= a.first_wg[s + 1]) ++s;
  const int r0 = a.bounds[s] + (w - a.first_wg[s]) * a.rows_per_wg;
  const int r1 = r0 + a.rows_per_wg;
  return {s, r0, r1 < a.bounds[s + 1] ? r1 : a.bounds[s + 1]};
}

template <int DT, int TPR, int NV, bool VEC>
__global__ void __launch_bounds__(256) layer_norm_fwd_kernel(NormArgs a) {
  constexpr int kRowsAtOnce = 256 / TPR;
  __shared__ float2 xch[4][4];
  const int t = threadIdx.x % TPR;
  const Share sh = share_of(a);
  float w[NV][8], b[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = 8 * (t + i * TPR);
    load_affine(a.w, a.w_dtype, a.seg0 + sh.seg, c, a.C, 1.f, a.w_add, w[i]);
    load_affine(a.b, a.w_dtype, a.seg0 + sh.seg, c, a.C, 0.f, 0.f, b[i]);
  }
  const float inv_c = 1.f / (float)a.C;
  int slot = 0;
  for (int r = sh.r0 + (int)threadIdx.x / TPR; r < sh.r1; r += kRowsAtOnce) {
    const char *xr = a.x + (int64_t)r * a.x_stride;
    float x[NV][8];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      unpack<DT>(load8<DT, VEC>(xr, 8 * (t + i * TPR), a.C), x[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += x[i][e];
    }
    const float mean = row_sum<TPR>(float2{sum, 0.f}, xch, slot).x * inv_c;
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[i][e] -= mean;
        if (8 * (t + i * TPR) + e < a.C) sq = fmaf(x[i][e], x[i][e], sq);
      }
    const float rstd = rsqrtf(row_sum<TPR>(float2{sq, 0.f}, xch, slot + 1).x * inv_c + a.eps);
    slot ^= 2;
    if (t == 0 && a.mean) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
    }
    char *yr = a.y + (int64_t)r * a.y_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = fmaf(x[i][e] * rstd, w[i][e], b[i][e]);
      store8<DT, VEC>(yr, 8 * (t + i * TPR), a.C, y);
    }
  }
}

template <int DT, int TPR, int NV, bool VEC>
__global__ void __launch_bounds__(256) layer_norm_bwd_kernel(NormArgs a) {
  constexpr int kRowsAtOnce = 256 / TPR;
  __shared__ float2 xch[2][4];
  __shared__ float fold[TPR > 64 ? 1 : 3 * 64 * 8];
  const int t = threadIdx.x % TPR;
  const Share sh = share_of(a);
  float w[NV][8], dw[NV][8], db[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    load_affine(a.w, a.w_dtype, a.seg0 + sh.seg, 8 * (t + i * TPR), a.C, 1.f, a.w_add, w[i]);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[i][e] = db[i][e] = 0.f;
  }
  const float inv_c = 1.f / (float)a.C;
  // The next row's loads are in flight while a row is reduced and stored, where
  // registers allow; a row itself stays as it came from memory and is unpacked twice, so
  // the loads fit (42120 rows of 5376 bf16 channels: 427 us without the loads ahead, 388
  // with them and floats kept, 335 so).
  constexpr bool kAhead = NV * sizeof(Row8<DT>) <= 48;
  Row8<DT> xn[NV], gn[NV];
  float mean_n = 0.f, rstd_n = 0.f;
  auto load = [&](int r) __attribute__((always_inline)) {
    const char *xr = a.x + (int64_t)r * a.x_stride, *gr = a.dy + (int64_t)r * a.dy_stride;
    mean_n = a.mean[r];
    rstd_n = a.rstd[r];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      xn[i] = load8<DT, VEC>(xr, 8 * (t + i * TPR), a.C);
      gn[i] = load8<DT, VEC>(gr, 8 * (t + i * TPR), a.C);
    }
  };
  int slot = 0, r = sh.r0 + (int)threadIdx.x / TPR;
  if (kAhead && r < sh.r1) load(r);
  for (; r < sh.r1; r += kRowsAtOnce) {
    if (!kAhead) load(r);
    const float mean = mean_n, rstd = rstd_n;
    Row8<DT> xc[NV], gc[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      xc[i] = xn[i];
      gc[i] = gn[i];
    }
    if (kAhead && r + kRowsAtOnce < sh.r1) load(r + kRowsAtOnce);
    float2 s = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float x[8], g[8];
      unpack<DT>(xc[i], x);
      unpack<DT>(gc[i], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = (x[e] - mean) * rstd;
        dw[i][e] = fmaf(g[e], x[e], dw[i][e]);
        db[i][e] += g[e];
        g[e] *= w[i][e];
        s.x += g[e];
        s.y = fmaf(g[e], x[e], s.y);
      }
    }
    s = row_sum<TPR>(s, xch, slot);
    slot ^= 1;
    const float m1 = s.x * inv_c, m2 = s.y * inv_c;
    char *dr = a.y + (int64_t)r * a.y_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (u32x4 &v : xc[i].v) asm volatile("" : "+v"(v));  // unpacked again, not kept
#pragma unroll
      for (u32x4 &v : gc[i].v) asm volatile("" : "+v"(v));
      float x[8], g[8];
      unpack<DT>(xc[i], x);
      unpack<DT>(gc[i], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = rstd * (g[e] * w[i][e] - m1 - (x[e] - mean) * rstd * m2);
      store8<DT, VEC>(dr, 8 * (t + i * TPR), a.C, x);
    }
  }
  if (!a.partial) return;
  float *out = a.partial + (int64_t)(a.wg0 + blockIdx.x) * 2 * a.C;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      float(&v)[8] = which ? db[i] : dw[i];
      if constexpr (TPR == 64) {  // the other waves' rows
        const int wave = threadIdx.x >> 6;
        __syncthreads();
        if (wave > 0) {
#pragma unroll
          for (int e = 0; e < 8; ++e) fold[((wave - 1) * 8 + e) * 64 + t] = v[e];
        }
        __syncthreads();
        if (wave > 0) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (v[e] + fold[e * 64 + t]) + (fold[(8 + e) * 64 + t] + fold[(16 + e) * 64 + t]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = 8 * (t + i * TPR) + e;
        if (c < a.C) out[which * a.C + c] = v[e];
      }
    }
  }
}

// Sums of the partial rows of each segment's workgroups: 64 channels of dw or db per
// workgroup, its waves in turn.  Sixteen waves where segments have over 128 partial rows on
// average (512 rows of 5376 channels: 10.7 us with four, 4.8 with sixteen), four where they
// have fewer (39: 6.4 and 8.6).
template <int kSumWaves>
__global__ void __launch_bounds__(64 * kSumWaves) layer_norm_param_grad_kernel(NormArgs a) {
  __shared__ float fold[kSumWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane, seg = blockIdx.y, which = blockIdx.z;
  const int w0 = a.wg0 + a.first_wg[seg], w1 = a.wg0 + a.first_wg[seg + 1];
  float sum = 0.f;
  if (c < a.C) {
    constexpr int kFlight = 8;  // loads in flight
    for (int w = w0 + wave; w < w1; w += kSumWaves * kFlight) {
      float v[kFlight];
#pragma unroll
      for (int i = 0; i < kFlight; ++i)
        v[i] = w + kSumWaves * i < w1 ? a.partial[((int64_t)(w + kSumWaves * i) * 2 + which) * a.C + c] : 0.f;
#pragma unroll
      for (int i = 0; i < kFlight; ++i) sum += v[i];
    }
  }
  fold[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && c < a.C) {
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < kSumWaves; ++w) sum += fold[w][lane];
    (which ? a.db : a.dw)[(int64_t)(a.seg0 + seg) * a.C + c] = sum;
  }
}

typedef void (*NormKernel)(NormArgs);

// Rows up to 1024 channels take one wave, longer ones a workgroup.
template <int DT, bool VEC>
NormKernel pick_fwd(int C, int *rows_at_once) {
  *rows_at_once = C <= 1024 ? 4 : 1;
  if (C <= 512) return layer_norm_fwd_kernel<DT, 64, 1, VEC>;
  if (C <= 1024) return layer_norm_fwd_kernel<DT, 64, 2, VEC>;
  if (C <= 2048) return layer_norm_fwd_kernel<DT, 256, 1, VEC>;
  if (C <= 4096) return layer_norm_fwd_kernel<DT, 256, 2, VEC>;
  if (C <= 6144) return layer_norm_fwd_kernel<DT, 256, 3, VEC>;
  if (C <= 8192) return layer_norm_fwd_kernel<DT, 256, 4, VEC>;
  return layer_norm_fwd_kernel<DT, 256, 8, VEC>;
}
template <int DT, bool VEC>
NormKernel pick_bwd(int C, int *rows_at_once) {
  *rows_at_once = C <= 1024 ? 4 : 1;
  if (C <= 512) return layer_norm_bwd_kernel<DT, 64, 1, VEC>;
  if (C <= 1024) return layer_norm_bwd_kernel<DT, 64, 2, VEC>;
  if (C <= 2048) return layer_norm_bwd_kernel<DT, 256, 1, VEC>;
  if (C <= 4096) return layer_norm_bwd_kernel<DT, 256, 2, VEC>;
  if (C <= 6144) return layer_norm_bwd_kernel<DT, 256, 3, VEC>;
  if (C <= 8192) return layer_norm_bwd_kernel<DT, 256, 4, VEC>;
  return layer_norm_bwd_kernel<DT, 256, 8, VEC>;
}
template <bool BWD, bool VEC>
NormKernel pick(int dtype, int C, int *rows_at_once) {
  switch (dtype) {
    case H3A_FP32: return BWD ? pick_bwd<H3A_FP32, VEC>(C, rows_at_once) : pick_fwd<H3A_FP32, VEC>(C, rows_at_once);
    case H3A_FP16: return BWD ? pick_bwd<H3A_FP16, VEC>(C, rows_at_once) : pick_fwd<H3A_FP16, VEC>(C, rows_at_once);
    default: return BWD ? pick_bwd<H3A_BF16, VEC>(C, rows_at_once) : pick_fwd<H3A_BF16, VEC>(C, rows_at_once);
  }
}

}  // namespace

// Rows per workgroup, in whole steps of the rows it takes at once: as many as make the
// grid per_cu workgroups on each of the chip's 256 CUs, each segment adding at most one (13
// more than fit took 408 us for 335 at 42120 rows of 5376 channels, backward).  per_cu is by
// width alone, and what fits goes by type and alignment too: backward, one workgroup fewer
// fits from 1025 to 2048 and from 6145 channels on, and up to 512 in fp32 and at odd widths
// of bf16, forward half as many past 8192; these run the rest of the grid as a second round
// (bf16 backward: 3.9 TB/s at 2048 and 8192 channels, 4.2 to 4.8 at 512, 1024, 4096 and 5376).
int norm_rows_per_wg(int64_t rows, int C, int segments, bool bwd) {
  const int per_cu = bwd ? (C <= 512 || (C > 1024 && C <= 2048) ? 5 : (C <= 1024 ? 3 : 2)) : (C <= 2048 ? 8 : 4);
  const int wgs = 256 * per_cu - (segments < 128 ? segments : 0);
  const int step = C <= 1024 ? 4 : 1;
  // Backward, four rows at least: a workgroup leaves as many bytes of partial sums as a row and
  // a half has to read and write.
  const int64_t n = (rows + wgs - 1) / wgs, least = bwd ? 4 : 1;
  return (int)((n < least ? least : n) + step - 1) / step * step;
}

int norm_wgs(const int *bounds, int segments, int rows_per_wg) {
  int64_t n = 0;
  for (int s = 0; s < segments; ++s) n += (bounds[s + 1] - bounds[s] + rows_per_wg - 1) / rows_per_wg;
  return (int)n;
}

int launch_layer_norm(NormArgs a, const int *bounds, int segments, int dtype, bool bwd, bool vec, hipStream_t s) {
  int at_once = 1;
  const NormKernel kernel = bwd ? (vec ? pick<true, true>(dtype, a.C, &at_once) : pick<true, false>(dtype, a.C, &at_once))
                                : (vec ? pick<false, true>(dtype, a.C, &at_once) : pick<false, false>(dtype, a.C, &at_once));
  a.wg0 = 0;
  for (a.seg0 = 0; a.seg0 < segments; a.seg0 += kNormSegments) {
    a.segments = segments - a.seg0 < kNormSegments ? segments - a.seg0 : kNormSegments;
    int wgs = 0;
    for (int i = 0; i <= a.segments; ++i) {
      a.bounds[i] = bounds[a.seg0 + i];
      a.first_wg[i] = wgs;
      if (i < a.segments) wgs += (bounds[a.seg0 + i + 1] - a.bounds[i] + a.rows_per_wg - 1) / a.rows_per_wg;
    }
    if (wgs > 0) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)wgs), dim3(256), 0, s, a);
      const int rc = check_launch(bwd ? "layer_norm_bwd_kernel" : "layer_norm_fwd_kernel");
      if (rc) return rc;
    }
    if (bwd && a.partial) {
      const bool many = wgs > 128 * a.segments;
      hipLaunchKernelGGL((many ? layer_norm_param_grad_kernel<16> : layer_norm_param_grad_kernel<4>),
                         dim3((unsigned)((a.C + 63) / 64), (unsigned)a.segments, 2), dim3(many ? 1024 : 256), 0, s, a);
      const int rc = check_launch("layer_norm_param_grad_kernel");
      if (rc) return rc;
    }
    a.wg0 += wgs;
  }
  return H3A_OK;
}

}  // namespace h3a
