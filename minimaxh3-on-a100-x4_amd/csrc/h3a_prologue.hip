// Fused per-head qk-RMSNorm + split-half RoPE, in place, for gfx950.
//
// Replaces comfy_kitchen's rms_rope_split_half_(q, k, rope_freqs, qw, kw,
// epsilon, rot_dim) as called by the DiT attention (harness/sp_runtime.py:93-99,
// custom_nodes/h3_profiler/__init__.py:99-106) on [1,S,H,128] strided views of
// the fused QKV projection output.  It is HBM-bound: every q/k row is read
// once and written once (4*S*H*D*2 bytes) plus one rope row per token.
//
// Layout of the work: one wave owns one (b,s) token and a chunk of HPW heads
// (28 or 16, chosen per launch).  Its four 16-lane groups walk the chunk
// one head each per step; within a group each lane holds 8 consecutive dims
// (one 128-bit access), so one wave access moves four whole 256-byte head rows
// (1 KB contiguous in the fused QKV layout).  The token's RoPE matrices and
// the two weight vectors are loaded into registers once per wave and reused
// for all 2 x HPW rows; the chunk's row loads are issued before any math.  The sum of squares
// is reduced across the 16 lanes with DPP moves; the RoPE partner dims
// (i, i+rot/2) sit rot/16 lanes apart: a DPP rotation at rot = 128, else one
// shuffle each.
#include "h3a_device.h"
#include "h3a_internal.h"

namespace h3a {

constexpr int kRopeD = 128;

// v of another lane of the same 16-lane row, in the VALU (no LDS round trip as
// a shuffle takes).
template <int CTRL>
__device__ __forceinline__ float dpp_row(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
constexpr int kDppXor1 = 0xB1;         // quad_perm [1,0,3,2]
constexpr int kDppXor2 = 0x4E;         // quad_perm [2,3,0,1]
constexpr int kDppHalfMirror = 0x141;  // lane i of 8 <- 7 - i
constexpr int kDppMirror = 0x140;      // lane i of 16 <- 15 - i
constexpr int kDppRor8 = 0x128;        // lane i of 16 <- i ^ 8

// Sum over the 16 lanes of a row, on all of them.  Once the lanes of a quad (of
// 8) hold the same sum, a mirror pairs them as an xor with 4 (8) would.
__device__ __forceinline__ float group16_sum(float v) {
  v += dpp_row<kDppXor1>(v);
  v += dpp_row<kDppXor2>(v);
  v += dpp_row<kDppHalfMirror>(v);
  v += dpp_row<kDppMirror>(v);
  return v;
}

__device__ __forceinline__ void unpack8(const u32x4 &w, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16_lo(w[i]);
    x[2 * i + 1] = bf16_hi(w[i]);
  }
}

__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
  return u32x4{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
               pack_bf16x2(x[6], x[7])};
}

// Heads per wave (HPW, a multiple of 4: four 16-lane groups): 28 when it
// divides H, otherwise 16.  At H=56, 28 gives two full waves per token, each
// reading the token's RoPE row once (same box: 5.41 TB/s against 5.15 with 16
// heads, of which the fourth wave per token has 8; 4.80 with 8 full waves and
// 5.00 with one wave of all 56, whose 201 VGPRs halve the waves in flight);
// non-temporal stores changed nothing.
__host__ __device__ constexpr int rope_heads_per_wave(int H) { return H % 28 == 0 ? 28 : 16; }

// The lane's half of its token's 2x2 matrices: lanes of the first rotated half
// (c < nh) apply the first row (R00, R01), their partners the second (R10, R11).
// Lanes past the rotated dims hold nothing.
// kRot128: every dim is rotated (nh = 8), so neither this nor the row needs a
// branch: branches between a token's loads and its use make the compiler wait
// for more loads than the token's own.
template <bool kRot128>
__device__ __forceinline__ void load_rope(float2 (&R)[8], const float *rope_row, int c, int nh) {
  if (kRot128) {
    const float *p = rope_row + (c & 7) * 32 + (c >> 3) * 2;
#pragma unroll
    for (int e = 0; e < 8; ++e) R[e] = *(const float2 *)(p + 4 * e);
  } else if (c < 2 * nh) {
    const float *p = rope_row + (c < nh ? c * 32 : (c - nh) * 32 + 2);
#pragma unroll
    for (int e = 0; e < 8; ++e) R[e] = *(const float2 *)(p + 4 * e);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) R[e] = float2{0.f, 1.f};
  }
}

// y = rmsnorm(x) * w, then rotate pairs (i, i+rot/2) with the lane's matrix rows.
template <bool kRot128>
__device__ __forceinline__ void norm_rope_row(float (&x)[8], const float (&w)[8], float eps,
                                              const float2 (&R)[8], int c, int nh) {
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
  ss = group16_sum(ss);
  const float r = rsqrtf(ss * (1.0f / kRopeD) + eps);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = x[e] * r * w[e];

  const bool first = c < nh;
  const bool rotated = c < 2 * nh;
  float xp[8];
  if (kRot128) {  // the partner is 8 lanes away
#pragma unroll
    for (int e = 0; e < 8; ++e) xp[e] = dpp_row<kDppRor8>(x[e]);
  } else {
    const int partner = first ? c + nh : (rotated ? c - nh : c);
#pragma unroll
    for (int e = 0; e < 8; ++e) xp[e] = __shfl(x[e], partner, 16);
  }
  if (kRot128 || rotated) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf(R[e].x, first ? x[e] : xp[e], R[e].y * (first ? xp[e] : x[e]));
  }
}

template <int kHeadsPerWave, bool kRot128>
__global__ void __launch_bounds__(256) qk_rmsnorm_rope_kernel(RopeArgs a) {
  static_assert(kHeadsPerWave % 4 == 0, "four 16-lane groups per wave");
  constexpr int kSteps = kHeadsPerWave / 4;  // heads per 16-lane group
  const int tid = threadIdx.x, lane = tid & 63, grp = lane >> 4, c = lane & 15;
  const int nchunk = (a.H + kHeadsPerWave - 1) / kHeadsPerWave;
  const int64_t item = (int64_t)blockIdx.x * 4 + (tid >> 6);  // (token, head chunk)
  if (item >= (int64_t)a.B * a.S * nchunk) return;            // whole waves leave together
  const int chunk = (int)(item % nchunk);
  const int64_t bs = item / nchunk;
  const int s = (int)(bs % a.S), b = (int)(bs / a.S);

  float wq[8], wk[8];
  unpack8(*(const u32x4 *)(a.qw + c * 8), wq);
  unpack8(*(const u32x4 *)(a.kw + c * 8), wk);
  float2 R[8];
  const int nh = a.rot >> 4;
  load_rope<kRot128>(R, a.rope + b * a.rsb + s * a.rss, c, nh);

  uint16_t *qrow = a.q + b * a.qsb + s * a.qss + c * 8;
  uint16_t *krow = a.k + b * a.ksb + s * a.kss + c * 8;
  int heads[kSteps];
  u32x4 qv[kSteps], kv[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int h = chunk * kHeadsPerWave + i * 4 + grp;
    heads[i] = h;
    const int hc = h < a.H ? h : a.H - 1;  // past-the-end groups recompute the last head, store nothing
    qv[i] = *(const u32x4 *)(qrow + hc * a.qsh);
    kv[i] = *(const u32x4 *)(krow + hc * a.ksh);
  }
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    float xq[8], xk[8];
    unpack8(qv[i], xq);
    unpack8(kv[i], xk);
    norm_rope_row<kRot128>(xq, wq, a.eps, R, c, nh);
    norm_rope_row<kRot128>(xk, wk, a.eps, R, c, nh);
    if (heads[i] < a.H) {
      *(u32x4 *)(qrow + heads[i] * a.qsh) = pack8(xq);
      *(u32x4 *)(krow + heads[i] * a.ksh) = pack8(xk);
    }
  }
}

// The prologue with the block pooling of SLA's block map fused in (the
// means block_pool_kernel takes of the stored q and k).  One workgroup per
// (b, block of blk tokens, chunk of kHeadsPerWave heads); wave w normalises
// and rotates tokens w, w+4, w+8, ... of the block as qk_rmsnorm_rope_kernel
// does and sums, per (head, dim), the bf16 values it stores, in token order.
// The waves' sums S0..S3 are combined as (S0 + S1) + (S2 + S3) through LDS and
// scaled by 1/rows: block_pool_kernel's lane rg sums rows rg, rg+4, ... in
// order and combines the four lane groups in that association, so the means
// are equal to its output bit for bit, and the selection made from them is
// the same.  Bound by HBM at full size and by the latency of a wave's serial
// tokens at small ones.  A ring holds kDepth tokens' loads; a slot is refilled
// after its token's stores (the compiler cannot move loads above them), so
// with kDepth = 2 one token's loads are in flight while the other is computed, and
// with 1 none are: there the gain is from cross-lane steps in the VALU and, at
// rot = 128, a row without branches.  Per call, against LDS shuffles and branches
// token by token: H=14 S=4104 44.8 -> 24.1 us (4 heads, kDepth = 2), H=56 S=4104
// 66.9 -> 55.2, H=28 S=42120 (blocks of 96) 299 -> 264, H=56 S=42120 510 -> 499 (4.9
// TB/s; a 2 GiB copy moves 5.0 on the same card); longer by more than 1 % (to 3 %)
// only at rot = 64 with 14 or 28 heads of S=42120.
template <int kHeadsPerWave, int kDepth, bool kRot128>
__global__ void __launch_bounds__(256) qk_rmsnorm_rope_pool_kernel(RopeArgs a, int blk, int nb, float *pq,
                                                                   float *pk) {
  static_assert(kHeadsPerWave % 4 == 0, "four 16-lane groups per wave");
  constexpr int kSteps = kHeadsPerWave / 4;
  // Partial sums of waves 1 and 3 (slots 0 and 1), then of wave 2 (slot 0):
  // [slot][step][q,k][lane] of 8 floats.
  __shared__ __attribute__((aligned(16))) float xch[2][kSteps][2][64][8];
  const int tid = threadIdx.x, lane = tid & 63, grp = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nchunk = (a.H + kHeadsPerWave - 1) / kHeadsPerWave;
  const int chunk = (int)(blockIdx.x % nchunk);
  const int64_t bj = blockIdx.x / nchunk;
  const int j = (int)(bj % nb), b = (int)(bj / nb);
  const int r0 = j * blk;
  const int rows = a.S - r0 < blk ? a.S - r0 : blk;

  float wq[8], wk[8];
  unpack8(*(const u32x4 *)(a.qw + c * 8), wq);
  unpack8(*(const u32x4 *)(a.kw + c * 8), wk);
  const int nh = a.rot >> 4;
  int heads[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) heads[i] = chunk * kHeadsPerWave + i * 4 + grp;
  float sq[kSteps][8], sk[kSteps][8];
#pragma unroll
  for (int i = 0; i < kSteps; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) sq[i][e] = sk[i][e] = 0.f;

  // This wave's tokens wave, wave + 4, ...: a ring of kDepth tokens' loads in
  // flight, each slot refilled once its token is done.  With two slots, loads
  // past the wave's last token repeat it (its own rows): a branch there would
  // make the compiler wait for both slots (H=14 S=4104: 24.1 us, 30.6 with it).  With
  // one, the branch costs nothing and the repeated load up to 17 % (blocks of 32).
  const int mine = (rows - wave + 3) / 4;
  struct Token {
    float2 R[8];
    u32x4 q[kSteps], k[kSteps];
  };
  Token ring[kDepth];
  auto token_of = [&](int n) __attribute__((always_inline)) { return r0 + wave + 4 * (n < mine ? n : mine - 1); };
  auto load = [&](Token &in, int n) __attribute__((always_inline)) {
    const int s = token_of(n);
    load_rope<kRot128>(in.R, a.rope + b * a.rsb + s * a.rss, c, nh);
    const uint16_t *qrow = a.q + b * a.qsb + s * a.qss + c * 8;
    const uint16_t *krow = a.k + b * a.ksb + s * a.kss + c * 8;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int hc = heads[i] < a.H ? heads[i] : a.H - 1;  // past-the-end groups store nothing
      in.q[i] = *(const u32x4 *)(qrow + hc * a.qsh);
      in.k[i] = *(const u32x4 *)(krow + hc * a.ksh);
    }
  };
  auto process = [&](const Token &in, int n) __attribute__((always_inline)) {
    const int s = token_of(n);
    uint16_t *qrow = a.q + b * a.qsb + s * a.qss + c * 8;
    uint16_t *krow = a.k + b * a.ksb + s * a.kss + c * 8;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      float xq[8], xk[8];
      unpack8(in.q[i], xq);
      unpack8(in.k[i], xk);
      norm_rope_row<kRot128>(xq, wq, a.eps, in.R, c, nh);
      norm_rope_row<kRot128>(xk, wk, a.eps, in.R, c, nh);
      const u32x4 oq = pack8(xq), ok = pack8(xk);
      if (heads[i] < a.H) {
        *(u32x4 *)(qrow + heads[i] * a.qsh) = oq;
        *(u32x4 *)(krow + heads[i] * a.ksh) = ok;
      }
      float yq[8], yk[8];  // the stored values
      unpack8(oq, yq);
      unpack8(ok, yk);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sq[i][e] += yq[e];
        sk[i][e] += yk[e];
      }
    }
  };
  if (mine > 0) {
#pragma unroll
    for (int d = 0; d < kDepth; ++d) load(ring[d], d);
    for (int n = 0; n < mine; n += kDepth) {
#pragma unroll
      for (int d = 0; d < kDepth; ++d) {
        if (n + d < mine) process(ring[d], n + d);
        if (kDepth > 1 || n + 1 < mine) load(ring[d], n + d + kDepth);
      }
    }
  }

  auto put = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      *(float4 *)&xch[slot][i][0][lane][0] = float4{sq[i][0], sq[i][1], sq[i][2], sq[i][3]};
      *(float4 *)&xch[slot][i][0][lane][4] = float4{sq[i][4], sq[i][5], sq[i][6], sq[i][7]};
      *(float4 *)&xch[slot][i][1][lane][0] = float4{sk[i][0], sk[i][1], sk[i][2], sk[i][3]};
      *(float4 *)&xch[slot][i][1][lane][4] = float4{sk[i][4], sk[i][5], sk[i][6], sk[i][7]};
    }
  };
  auto add = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sq[i][e] += xch[slot][i][0][lane][e];
        sk[i][e] += xch[slot][i][1][lane][e];
      }
  };
  if (wave & 1) put(wave >> 1);  // S1 -> slot 0, S3 -> slot 1
  __syncthreads();
  if (!(wave & 1)) add(wave >> 1);  // wave 0: S0 + S1, wave 2: S2 + S3
  __syncthreads();
  if (wave == 2) put(0);
  __syncthreads();
  if (wave != 0) return;  // no barrier follows
  add(0);  // (S0 + S1) + (S2 + S3)
  const float inv = 1.f / (float)rows;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    if (heads[i] >= a.H) continue;
    const int64_t o = (((int64_t)b * a.H + heads[i]) * nb + j) * kRopeD + c * 8;
    *(float4 *)(pq + o) = float4{sq[i][0] * inv, sq[i][1] * inv, sq[i][2] * inv, sq[i][3] * inv};
    *(float4 *)(pq + o + 4) = float4{sq[i][4] * inv, sq[i][5] * inv, sq[i][6] * inv, sq[i][7] * inv};
    *(float4 *)(pk + o) = float4{sk[i][0] * inv, sk[i][1] * inv, sk[i][2] * inv, sk[i][3] * inv};
    *(float4 *)(pk + o + 4) = float4{sk[i][4] * inv, sk[i][5] * inv, sk[i][6] * inv, sk[i][7] * inv};
  }
}

// Heads per workgroup.  A workgroup's waves walk their share of the block's
// tokens one after another, so with fewer 8-head workgroups than CUs the launch
// takes as long as one walk: 4-head chunks double the workgroups and shorten each
// step.  Measured with 8 / 4 heads: 24.5 / 19.5 us at H=4 S=1024 (16 workgroups of
// 8 heads), 29.3 / 24.1 at H=14 S=4104 (130), but 55.2 / 73.9 at H=56 S=4104 (455)
// and 499 / 626 at H=56 S=42120 (4613), where 2 KiB per access of a token's q or k
// against 1 KiB decides.
constexpr int64_t kPoolWideWgs = 256;
int launch_qk_rmsnorm_rope_pool(const RopeArgs &a, int blk, float *pq, float *pk, hipStream_t s) {
  const int nb = (a.S + blk - 1) / blk;
  const int64_t blocks = (int64_t)a.B * nb, wide = blocks * ((a.H + 7) / 8);
  const bool full = a.rot == kRopeD, wide_heads = wide >= kPoolWideWgs;
  auto *kernel = wide_heads
                     ? (full ? qk_rmsnorm_rope_pool_kernel<8, 1, true> : qk_rmsnorm_rope_pool_kernel<8, 1, false>)
                     : (full ? qk_rmsnorm_rope_pool_kernel<4, 2, true> : qk_rmsnorm_rope_pool_kernel<4, 2, false>);
  const int64_t wgs = wide_heads ? wide : blocks * ((a.H + 3) / 4);
  hipLaunchKernelGGL(kernel, dim3((unsigned)wgs), dim3(256), 0, s, a, blk, nb, pq, pk);
  return check_launch("qk_rmsnorm_rope_pool_kernel");
}

int launch_qk_rmsnorm_rope(const RopeArgs &a, hipStream_t s) {
  const int hpw = rope_heads_per_wave(a.H);
  const int64_t items = (int64_t)a.B * a.S * ((a.H + hpw - 1) / hpw);
  const int64_t blocks = (items + 3) / 4;
  const bool full = a.rot == kRopeD;
  auto *kernel = hpw == 28 ? (full ? qk_rmsnorm_rope_kernel<28, true> : qk_rmsnorm_rope_kernel<28, false>)
                           : (full ? qk_rmsnorm_rope_kernel<16, true> : qk_rmsnorm_rope_kernel<16, false>);
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, s, a);
  return check_launch("qk_rmsnorm_rope_kernel");
}

// ---------------------------------------------------------------------------
// The prologue from positions on several axes (time, height, width), out of place or in
// place, and its backward pass.  Pair i of a token turns by pos[axis(i)] * turns[i]
// revolutions; with y' = R(angle) (x * r * w), r = rsqrt(mean(x^2) + eps):
//   g = R(angle)^T dy',  dw = sum over rows of g * x * r,
//   dx = r * (g * w - x * r^2 * mean(x * g * w))
// HBM-bound as the kernel above, and laid out like it: 16 lanes per head row, 8 dims per
// lane.  The angles of four tokens are taken once per workgroup, one pair per lane, and
// shared through LDS: the product with the position in fp64 (exact to 2^-53 of the
// angle: far positions lose nothing), its fraction of a revolution in fp32.
__device__ __forceinline__ void token_angles(const RopeAxesArgs &a, int64_t bs, int lane, float (*cs)[64]) {
  if (2 * lane < a.rot) {
    const int64_t at = bs / a.S * a.pos_b + bs % a.S * a.axes + a.axis[lane];
    const double pos = a.pos_float ? (double)static_cast<const float *>(a.pos)[at]
                                   : (double)static_cast<const int32_t *>(a.pos)[at];
    double t = pos * a.turns[lane];
    t -= __builtin_rint(t);
    float s, c;
    sincospif((float)(2.0 * t), &s, &c);
    cs[0][lane] = c;
    cs[1][lane] = s;
  }
}

// The lane's 8 cosines and sines; its dims are 8c .. 8c+7, nh lanes hold a half.  The
// second half's sine is the first's negated: y'_c = cos y_c - sgn sin y_partner.
__device__ __forceinline__ void lane_angles(const float (*cs)[64], int c, int nh, float (&co)[8], float (&si)[8]) {
  const int f = c < nh ? c : c - nh;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    co[e] = c < 2 * nh ? cs[0][8 * f + e] : 1.f;
    si[e] = c < 2 * nh ? (c < nh ? -cs[1][8 * f + e] : cs[1][8 * f + e]) : 0.f;
  }
}

// x[e] of the lane that holds the other dim of each pair.
template <bool kRot128>
__device__ __forceinline__ void partner8(const float (&x)[8], float (&xp)[8], int c, int nh) {
  if (kRot128) {
#pragma unroll
    for (int e = 0; e < 8; ++e) xp[e] = dpp_row<kDppRor8>(x[e]);
  } else {
    const int partner = c < nh ? c + nh : (c < 2 * nh ? c - nh : c);
#pragma unroll
    for (int e = 0; e < 8; ++e) xp[e] = __shfl(x[e], partner, 16);
  }
}

constexpr int kAxesTokens = 4;  // tokens per workgroup and step

// kSteps: head rows per lane group in flight, so kSteps * 4 heads per item; items of a
// step are (token, tensor, chunk of heads), dealt to the workgroup's four waves.
template <int kSteps, bool kRot128, bool kBwd>
__global__ void __launch_bounds__(256) rope_axes_kernel(RopeAxesArgs a) {
  __shared__ float angles[2][kAxesTokens][2][64];
  __shared__ float fold[kBwd ? 4 : 1][2][128];
  const int tid = threadIdx.x, lane = tid & 63, grp = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nh = a.rot >> 4;
  const int64_t tokens = (int64_t)a.B * a.S;
  const int chunks[2] = {(a.H[0] + 4 * kSteps - 1) / (4 * kSteps), (a.H[1] + 4 * kSteps - 1) / (4 * kSteps)};
  const int per_token = chunks[0] + chunks[1];
  float dw[2][8];
#pragma unroll
  for (int e = 0; e < 8; ++e) dw[0][e] = dw[1][e] = 0.f;
  int slot = 0;
  for (int64_t t0 = (int64_t)blockIdx.x * kAxesTokens; t0 < tokens; t0 += (int64_t)gridDim.x * kAxesTokens) {
    if (t0 + wave < tokens) token_angles(a, t0 + wave, lane, angles[slot][wave]);
    __syncthreads();
    for (int item = wave; item < kAxesTokens * per_token; item += 4) {
      const int64_t bs = t0 + item / per_token;
      if (bs >= tokens) break;
      int chunk = item % per_token;
      const int which = chunk < chunks[0] ? 0 : 1;
      chunk -= which ? chunks[0] : 0;
      const int H = which ? a.H[1] : a.H[0], h0 = chunk * 4 * kSteps;
      const int64_t b = bs / a.S, s = bs % a.S;
      const int64_t *xs = which ? a.xs[1] : a.xs[0], *ys = which ? a.ys[1] : a.ys[0];
      const uint16_t *xrow = (which ? a.x[1] : a.x[0]) + b * xs[0] + s * xs[1] + 8 * c;
      uint16_t *yrow = (which ? a.y[1] : a.y[0]) + b * ys[0] + s * ys[1] + 8 * c;
      u32x4 xv[kSteps], gv[kBwd ? kSteps : 1];
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int h = h0 + 4 * i + grp < H ? h0 + 4 * i + grp : H - 1;
        xv[i] = *(const u32x4 *)(xrow + h * xs[2]);
        if constexpr (kBwd) {
          const int64_t *gs = which ? a.dys[1] : a.dys[0];
          gv[i] = *(const u32x4 *)((which ? a.dy[1] : a.dy[0]) + b * gs[0] + s * gs[1] + 8 * c + h * gs[2]);
        }
      }
      float w[8], co[8], si[8];
      unpack8(*(const u32x4 *)((which ? a.w[1] : a.w[0]) + 8 * c), w);
      lane_angles(angles[slot][item / per_token], c, nh, co, si);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        if (h0 + 4 * i >= H) break;
        const int h = h0 + 4 * i + grp;
        float x[8], p[8], y[8];
        unpack8(xv[i], x);
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
        const float r = rsqrtf(group16_sum(ss) * (1.0f / kRopeD) + a.eps);
        if constexpr (!kBwd) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = x[e] * r * w[e];
          partner8<kRot128>(x, p, c, nh);
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = fmaf(co[e], x[e], si[e] * p[e]);
        } else {
          float g[8], m = 0.f;
          unpack8(gv[i], g);
          partner8<kRot128>(g, p, c, nh);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            g[e] = fmaf(co[e], g[e], -si[e] * p[e]);
            const float gx = g[e] * x[e];
            if (h < H) {
              if (which) dw[1][e] = fmaf(gx, r, dw[1][e]);
              else dw[0][e] = fmaf(gx, r, dw[0][e]);
            }
            m = fmaf(gx, w[e], m);
          }
          m = group16_sum(m) * (1.0f / kRopeD) * r * r;
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = r * fmaf(-x[e], m, g[e] * w[e]);
        }
        if (h < H) *(u32x4 *)(yrow + h * ys[2]) = pack8(y);
      }
    }
    slot ^= 1;
  }
  if constexpr (kBwd) {
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float v = dw[which][e];
        v += __shfl_xor(v, 16);
        v += __shfl_xor(v, 32);
        if (grp == 0) fold[wave][which][8 * c + e] = v;
      }
    __syncthreads();
    const int which = tid >> 7, d = tid & 127;
    a.partial[(int64_t)blockIdx.x * 256 + tid] =
        (fold[0][which][d] + fold[1][which][d]) + (fold[2][which][d] + fold[3][which][d]);
  }
}

// Sums of the workgroups' partial rows in a fixed order: 4 columns per workgroup, 64
// threads to a column, each taking every 64th row, all in flight.
constexpr int kAxesBwdWgs = 768;  // 3 workgroups of the backward kernel per CU at a time
__global__ void __launch_bounds__(256) rope_axes_param_grad_kernel(RopeAxesArgs a, int wgs) {
  __shared__ float fold[4][4];
  const int col = threadIdx.x & 3, part = threadIdx.x >> 2, at = blockIdx.x * 4 + col;
  constexpr int kPer = kAxesBwdWgs / 64;
  float v[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int row = part + 64 * i;
    v[i] = row < wgs ? a.partial[(int64_t)row * 256 + at] : 0.f;
  }
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) sum += v[i];
#pragma unroll
  for (int o = 4; o < 64; o <<= 1) sum += __shfl_xor(sum, o);
  if ((threadIdx.x & 63) < 4) fold[threadIdx.x >> 6][col] = sum;
  __syncthreads();
  if (threadIdx.x < 4) a.dw[at >> 7][at & 127] = (fold[0][col] + fold[1][col]) + (fold[2][col] + fold[3][col]);
}

// Forward: workgroups at most (a launch has fewer than 2^32 threads; the kernel walks on).
constexpr int64_t kAxesMaxWgs = 1 << 22;
// Backward: workgroups that each leave a partial row of the weights' gradients.
int rope_axes_bwd_wgs(int B, int S) {
  const int64_t n = ((int64_t)B * S + kAxesTokens - 1) / kAxesTokens;
  return (int)(n < kAxesBwdWgs ? n : kAxesBwdWgs);
}

template <bool kBwd>
static int launch_rope_axes_as(const RopeAxesArgs &a, hipStream_t s) {
  const int64_t groups = ((int64_t)a.B * a.S + kAxesTokens - 1) / kAxesTokens;
  const int64_t wgs = kBwd ? rope_axes_bwd_wgs(a.B, a.S) : (groups < kAxesMaxWgs ? groups : kAxesMaxWgs);
  const bool full = a.rot == kRopeD;
  const int h = a.H[0] > a.H[1] ? a.H[0] : a.H[1];
  void (*kernel)(RopeAxesArgs) =
      h > 16 ? (full ? rope_axes_kernel<7, true, kBwd> : rope_axes_kernel<7, false, kBwd>)
             : (full ? rope_axes_kernel<2, true, kBwd> : rope_axes_kernel<2, false, kBwd>);
  hipLaunchKernelGGL(kernel, dim3((unsigned)wgs), dim3(256), 0, s, a);
  int rc = check_launch("rope_axes_kernel");
  if (rc || !kBwd) return rc;
  hipLaunchKernelGGL(rope_axes_param_grad_kernel, dim3(64), dim3(256), 0, s, a, (int)wgs);
  return check_launch("rope_axes_param_grad_kernel");
}
int launch_rope_axes(const RopeAxesArgs &a, bool bwd, hipStream_t s) {
  return bwd ? launch_rope_axes_as<true>(a, s) : launch_rope_axes_as<false>(a, s);
}

int rope_kernel_attrs(double out[6]) {
  hipFuncAttributes fa;
  const void *fn = reinterpret_cast<const void *>(&qk_rmsnorm_rope_kernel<28, true>);  // the H=56 width
  if (hipFuncGetAttributes(&fa, fn) != hipSuccess) return fail(H3A_ERR_HIP, "hipFuncGetAttributes failed");
  int blocks = 0, dev = 0, clk = 0, max_threads = 0;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, fn, 256, 0) != hipSuccess ||
      hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&clk, hipDeviceAttributeClockRate, dev) != hipSuccess ||
      hipDeviceGetAttribute(&max_threads, hipDeviceAttributeMaxThreadsPerMultiProcessor, dev) != hipSuccess)
    return fail(H3A_ERR_HIP, "occupancy query failed");
  out[0] = fa.numRegs;
  out[1] = (double)fa.sharedSizeBytes;
  out[2] = blocks;
  out[3] = clk;
  out[4] = max_threads > 0 ? (double)(blocks * 256) / max_threads : 0.0;
  out[5] = 256;
  return H3A_OK;
}

}  // namespace h3a
