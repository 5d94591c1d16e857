// Attention over a sliding window with a few first keys that stay visible (sinks),
// forward and backward, for gfx950: head_dim 128, bf16 in and out, fp32 sums.
//
// Query row i of sequence b sits at position pos = q_start + i and sees key j iff
//   j < len  and  (pos - left <= j <= pos + right  or  j < sinks)  and, if causal, j <= pos.
// Rows at positions outside [0, len) belong to no token: O = 0, lse = -inf, no gradient.
//   p_ij = exp(scale q_i.k_j - lse_i),  O_i = sum_j p_ij v_j
//   delta_i = dO_i.O_i,  ds_ij = p_ij (dO_i.v_j - delta_i)
//   dQ_i = scale sum_j ds_ij k_j,  dK_j = scale sum_i ds_ij q_i,  dV_j = sum_i p_ij dO_i
//
// Every product runs on v_mfma_f32_32x32x16_bf16 in the transposed form of the dense
// kernel: a wave holds 32 rows of one operand in registers as columns, streams the
// other side's rows through LDS, and finds the score tile in the layout in which it
// is the next product's operand.  P and dS are rounded to bf16 for that product (as
// the dense kernel rounds P); scores, softmax statistics and all sums are fp32.
#include "h3a_device.h"
#include "h3a_internal.h"
#include "h3a_queue.h"
#include "h3a_tile.h"

namespace h3a {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kRows = 128;  // rows (queries or keys) per workgroup, 32 per wave

// One LDS tile read both ways: whole rows as an MFMA operand (16 consecutive rows,
// one 16-byte chunk) and transposed (4 rows x 4 chunks).  Chunk c of row r sits in
// slot c ^ swz(r), swz(r) = 4 * (r % 4) + (r / 4) % 4: 16 different values over 16
// rows for the first kind, 4 values that are multiples of 4 apart over 4 rows for the
// second, so neither has bank conflicts.
struct DualLayout {
  static constexpr int kKRow = 256, kVRow = 256;  // bytes
  static constexpr int kKSlots = 16, kVSlots = 16;
  __device__ __forceinline__ static int swz(int r) { return 4 * (r & 3) + ((r >> 2) & 3); }
  __device__ __forceinline__ static int k_chunk(int r, int slot) { return slot ^ swz(r); }
  __device__ __forceinline__ static int v_chunk(int r, int slot) { return slot ^ swz(r); }
  __device__ __forceinline__ static int k_base(int l32, int g) { return l32 * kKRow + 16 * (g ^ swz(l32)); }
  __device__ __forceinline__ static int k_off(int kb, int ks) { return kb ^ (32 * ks); }
  // Transposed read of rows 4*(lane/32) + (lane%16)/4, columns as SwzLayout::v_base;
  // the rows 8 further on differ in swz by 2: offset ^ 32.
  __device__ __forceinline__ static int v_base(int lane) {
    const int i = (lane & 15) >> 2, g = lane >> 5;
    const int c = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    return (4 * g + i) * kVRow + 16 * (c ^ (4 * i + g)) + 8 * (lane & 1);
  }
};

// acc (128 dims x 32 columns) += X^T P over NKS sixteen-row steps of tile X, P in the
// score accumulator's order (pack_p).
template <int NKS>
__device__ __forceinline__ void transposed_product(const uint16_t *buf, const u32x4 (&pf)[NKS], int v_rd,
                                                   f32x16 (&acc)[4]) {
  const char *vb = reinterpret_cast<const char *>(buf);
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) {
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) {
      const int off = v_rd ^ (64 * dt);
      const u32x2 lo = lds_read_tr16_b64(reinterpret_cast<const uint16_t *>(vb + off + 16 * ks * 256));
      const u32x2 hi = lds_read_tr16_b64(reinterpret_cast<const uint16_t *>(vb + (off ^ 32) + (16 * ks + 8) * 256));
      acc[dt] = mfma_32x32x16(u32x4{lo.x, lo.y, hi.x, hi.y}, pf[ks], acc[dt]);
    }
  }
}

// A wave's 32 rows as columns of an MFMA operand, straight from global memory; rows
// past `rows` are zeros.
__device__ __forceinline__ void load_columns(u32x4 (&f)[8], const uint16_t *base, int64_t stride, int row, int rows,
                                             int g) {
  const uint16_t *p = base + (int64_t)(row < rows ? row : 0) * stride + 8 * g;
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) {
    const u32x4 v = *(const u32x4 *)(p + 16 * ks);
    f[ks] = row < rows ? v : u32x4{0, 0, 0, 0};
  }
}

// acc * mul, rounded to bf16, to rows row0 .. row0 + nrows - 1: through a wave-private
// LDS tile, so that every store writes four whole rows.  Columns whose `live` is false
// store zeros.
__device__ __forceinline__ void store_columns(const f32x16 (&acc)[4], float mul, bool live, uint8_t *tile,
                                              uint16_t *base, int64_t stride, int nrows, int lane) {
  const int g = lane >> 5, l32 = lane & 31;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) {
#pragma unroll
    for (int rr = 0; rr < 4; ++rr) {
      u32x2 val = {pack_bf16x2(acc[dt][4 * rr + 0] * mul, acc[dt][4 * rr + 1] * mul),
                   pack_bf16x2(acc[dt][4 * rr + 2] * mul, acc[dt][4 * rr + 3] * mul)};
      if (!live) val = u32x2{0, 0};
      const int c = 4 * dt + rr;
      *(u32x2 *)(tile + l32 * 256 + ((c ^ (l32 & 15)) << 4) + 8 * g) = val;
    }
  }
  const int ch = lane & 15;
  const __amdgpu_buffer_rsrc_t res = stage_rsrc(base, stride, nrows < 32 ? nrows : 32);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 4 * i + (lane >> 4);
    const u32x4 val = *(const u32x4 *)(tile + r * 256 + ((ch ^ (r & 15)) << 4));
    __builtin_amdgcn_raw_buffer_store_b128(val, res, (int)((uint32_t)r * (uint32_t)stride * 2u + 16u * ch), 0, 0);
  }
}

// A sequence of the batch: first query's position, keys, and the rows that are tokens.
struct Span {
  int qs, len, i_lo, i_hi;  // rows i_lo <= i < i_hi sit at positions 0 <= qs + i < len
};
constexpr int kPosLimit = 1 << 29;  // positions, window sides and lengths stay below it
__device__ __forceinline__ Span span_of(const WindowArgs &a, int b) {
  Span s;
  s.len = a.kv_lens ? a.kv_lens[b] : a.Skv;
  s.len = s.len < 0 ? 0 : (s.len > a.Skv ? a.Skv : s.len);
  s.qs = a.q_starts ? a.q_starts[b] : a.q_start;
  s.qs = s.qs < -kPosLimit ? -kPosLimit : (s.qs > kPosLimit ? kPosLimit : s.qs);
  s.i_lo = s.qs < 0 ? -s.qs : 0;
  s.i_hi = s.len - s.qs < a.Sq ? s.len - s.qs : a.Sq;
  s.len = __builtin_amdgcn_readfirstlane(s.len);
  s.qs = __builtin_amdgcn_readfirstlane(s.qs);
  s.i_lo = __builtin_amdgcn_readfirstlane(s.i_lo);
  s.i_hi = __builtin_amdgcn_readfirstlane(s.i_hi);
  return s;
}

// First keys that stay visible to position pos.
__device__ __forceinline__ int first_keys(const WindowArgs &a, const Span &s, int pos) {
  int n = a.sinks < s.len ? a.sinks : s.len;
  return a.causal && n > pos + 1 ? pos + 1 : n;
}

// The key stages of a run of positions p0 .. p1: [0, first) and then [lo, hi), or one
// range [0, hi) where the two meet.
struct KeyStages {
  int n_first, n, lo, first, hi;
  __device__ __forceinline__ void init(const WindowArgs &a, const Span &s, int p0, int p1) {
    first = first_keys(a, s, p1);
    lo = p0 - a.left > 0 ? p0 - a.left : 0;
    hi = (p1 + a.right < s.len - 1 ? p1 + a.right : s.len - 1) + 1;
    n_first = 0;
    if (first >= lo) {
      lo = 0;
      hi = hi > first ? hi : first;
    } else {
      n_first = (first + kBN - 1) / kBN;
    }
    n = n_first + (hi - lo + kBN - 1) / kBN;
  }
  __device__ __forceinline__ int key0(int j) const { return j < n_first ? j * kBN : lo + (j - n_first) * kBN; }
  __device__ __forceinline__ int limit(int j) const { return j < n_first ? first : hi; }
};

// What a wave at positions p0 .. p1 sees of a 64-key stage: nothing, all of it, or a part.
enum Cover { kNone, kAll, kPart };
__device__ __forceinline__ Cover cover_of(const WindowArgs &a, const Span &s, const KeyStages &ks, int j, int p0,
                                          int p1) {
  const int k0 = ks.key0(j), k1 = k0 + kBN - 1;
  const int f0 = first_keys(a, s, p0), f1 = first_keys(a, s, p1);
  if (k1 < f0) return kAll;
  if (j < ks.n_first) return k0 < f1 ? kPart : kNone;
  const int end0 = p0 + a.right < s.len - 1 ? p0 + a.right : s.len - 1;
  const int end1 = p1 + a.right < s.len - 1 ? p1 + a.right : s.len - 1;
  if (k0 >= p1 - a.left && k1 <= end0) return kAll;
  if (k0 >= f1 && (k0 > end1 || k1 < p0 - a.left)) return kNone;
  return kPart;
}

// Scores the lane's row does not see -> `hidden`.  Keys lo .. hi and those below first
// are seen; a stage of the first keys alone (only_first) ends at `first`.
__device__ __forceinline__ void mask_band(f32x16 (&s)[2], int key0, int g, int lo, int hi, int first, bool only_first,
                                          float hidden) {
  const int l = only_first ? 1 << 30 : lo;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int j = key0 + 32 * u + 8 * (r >> 2) + 4 * g + (r & 3);
      if (!((j >= l && j <= hi) || j < first)) s[u][r] = hidden;
    }
}

// Work item -> (tile, head, batch), consecutive tiles of a head on one XCD.
struct Item {
  int tile, h, b;
};
__device__ __forceinline__ Item item_of(int total, int tiles, int heads) {
  const int w = xcd_remap((int)blockIdx.x, total);
  const int bh = w / tiles;
  return {w % tiles, bh % heads, bh / heads};
}

// Forward.  A workgroup takes 128 query rows of one head, a wave 32 of them; the
// 64-key stages of their window are double-buffered in LDS by DMA, two workgroups to a
// CU, so that one's softmax overlaps the other's MFMAs.
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) window_fwd_kernel(WindowArgs a) {
  using L = SwzLayout;
  __shared__ __attribute__((aligned(16))) uint16_t kbuf[2][StageBytes<L>::kK / 2], vbuf[2][StageBytes<L>::kV / 2];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Item it = item_of(a.total, a.nqt, a.H);
  const Span sp = span_of(a, it.b);
  const int q0 = it.tile * kRows, wq0 = q0 + 32 * wave, row = wq0 + l32;
  const int r0 = q0 > sp.i_lo ? q0 : sp.i_lo, r1 = (q0 + kRows < sp.i_hi ? q0 + kRows : sp.i_hi) - 1;
  const bool live = row >= sp.i_lo && row < sp.i_hi;
  const uint16_t *Kb = a.k + it.b * a.ksb + (it.h / a.rep) * a.ksh;
  const uint16_t *Vb = a.v + it.b * a.vsb + (it.h / a.rep) * a.vsh;

  f32x16 o[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) o[dt] = f32x16{0.f};
  float m = kNegInf, lsum = 0.f;
  if (r1 >= r0) {
    // The wave's rows that are tokens; a wave without one takes the tile's nearest.
    auto clamp_row = [&](int i) __attribute__((always_inline)) { return i < r0 ? r0 : (i > r1 ? r1 : i); };
    const int p0 = sp.qs + clamp_row(wq0), p1 = sp.qs + clamp_row(wq0 + 31), pos = sp.qs + clamp_row(row);
    KeyStages st;
    st.init(a, sp, sp.qs + r0, sp.qs + r1);
    const int lo = pos - a.left, first = first_keys(a, sp, pos);
    const int hi = pos + a.right < sp.len - 1 ? pos + a.right : sp.len - 1;
    TileDma<4, L, false> kdma;
    TileDma<4, L, true> vdma;
    kdma.init(a.kss, wave, lane);
    vdma.init(a.vss, wave, lane);
    auto fetch = [&](int j) __attribute__((always_inline)) {
      kdma.issue(Kb, a.kss, st.key0(j), st.limit(j), kbuf[j & 1]);
      vdma.issue(Vb, a.vss, st.key0(j), st.limit(j), vbuf[j & 1]);
    };
    fetch(0);
    u32x4 qf[8];
    load_columns(qf, a.q + it.b * a.qsb + it.h * a.qsh, a.qss, row, a.Sq, g);
    const int k_rd = L::k_base(l32, g), v_rd = L::v_base(lane);
    wait_vmem_all();
    __syncthreads();
    for (int j = 0; j < st.n; ++j) {
      if (j + 1 < st.n) fetch(j + 1);
      const Cover c = cover_of(a, sp, st, j, p0, p1);
      if (c != kNone) {
        f32x16 s[2];
        u32x4 pf[4];
        score_tile<L, 2>(kbuf[j & 1], qf, k_rd, s);
        if (c == kPart) mask_band(s, st.key0(j), g, lo, hi, first, j < st.n_first, kNegInf);
        softmax_stage<2>(s, 0, kBN, g, a.sl2, m, lsum, o, pf);
        pv_tile<L, 4>(vbuf[j & 1], pf, v_rd, o);
      }
      wait_vmem_all();
      __syncthreads();
    }
  }
  const float ltot = half_swap_sum(lsum);
  const float inv = ltot > 0.f ? 1.f / ltot : 0.f;
  if (a.lse && g == 0 && row < a.Sq)
    a.lse[((int64_t)it.b * a.H + it.h) * a.Sq + row] = live && ltot > 0.f ? (m + log2f(ltot)) * kLn2 : kNegInf;
  if (wq0 < a.Sq)
    store_columns(o, inv, live, reinterpret_cast<uint8_t *>(&kbuf[0][0]) + wave * 8192,
                  a.o + it.b * a.osb + it.h * a.osh + (int64_t)wq0 * a.oss, a.oss, a.Sq - wq0, lane);
}

// Backward, dQ: tiles and stages as forward, with P from the stored lse.  The tile's
// delta = dO.O goes to a.delta for the second kernel.
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) window_dq_kernel(WindowArgs a) {
  using L = DualLayout;
  __shared__ __attribute__((aligned(16))) uint16_t kbuf[2][StageBytes<L>::kK / 2], vbuf[2][StageBytes<L>::kK / 2];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Item it = item_of(a.total, a.nqt, a.H);
  const Span sp = span_of(a, it.b);
  const int q0 = it.tile * kRows, wq0 = q0 + 32 * wave, row = wq0 + l32;
  const int r0 = q0 > sp.i_lo ? q0 : sp.i_lo, r1 = (q0 + kRows < sp.i_hi ? q0 + kRows : sp.i_hi) - 1;
  const bool live = row >= sp.i_lo && row < sp.i_hi;
  const uint16_t *Kb = a.k + it.b * a.ksb + (it.h / a.rep) * a.ksh;
  const uint16_t *Vb = a.v + it.b * a.vsb + (it.h / a.rep) * a.vsh;

  f32x16 dq[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) dq[dt] = f32x16{0.f};
  if (r1 >= r0) {
    auto clamp_row = [&](int i) __attribute__((always_inline)) { return i < r0 ? r0 : (i > r1 ? r1 : i); };
    const int p0 = sp.qs + clamp_row(wq0), p1 = sp.qs + clamp_row(wq0 + 31), pos = sp.qs + clamp_row(row);
    KeyStages st;
    st.init(a, sp, sp.qs + r0, sp.qs + r1);
    const int lo = pos - a.left, first = first_keys(a, sp, pos);
    const int hi = pos + a.right < sp.len - 1 ? pos + a.right : sp.len - 1;
    TileDma<4, L, false> kdma, vdma;
    kdma.init(a.kss, wave, lane);
    vdma.init(a.vss, wave, lane);
    auto fetch = [&](int j) __attribute__((always_inline)) {
      kdma.issue(Kb, a.kss, st.key0(j), st.limit(j), kbuf[j & 1]);
      vdma.issue(Vb, a.vss, st.key0(j), st.limit(j), vbuf[j & 1]);
    };
    fetch(0);
    u32x4 qf[8], df[8];
    load_columns(qf, a.q + it.b * a.qsb + it.h * a.qsh, a.qss, row, a.Sq, g);
    load_columns(df, a.dout + it.b * a.gsb + it.h * a.gsh, a.gss, row, a.Sq, g);
    float delta = 0.f;
    {
      u32x4 of[8];
      load_columns(of, a.o + it.b * a.osb + it.h * a.osh, a.oss, row, a.Sq, g);
#pragma unroll
      for (int ks = 0; ks < 8; ++ks)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          delta = fmaf(bf16_hi(of[ks][i]), bf16_hi(df[ks][i]), fmaf(bf16_lo(of[ks][i]), bf16_lo(df[ks][i]), delta));
      delta = half_swap_sum(delta);
    }
    const int64_t stat = ((int64_t)it.b * a.H + it.h) * a.Sq + (row < a.Sq ? row : a.Sq - 1);
    if (g == 0 && row < a.Sq) a.delta[stat] = delta;
    // A row without a finite lse saw nothing: p = exp2(-inf) = 0.
    const float l2 = a.lse[stat] == kNegInf ? -kNegInf : a.lse[stat] * kLog2e;
    const int k_rd = L::k_base(l32, g), t_rd = L::v_base(lane);
    wait_vmem_all();
    __syncthreads();
    for (int j = 0; j < st.n; ++j) {
      if (j + 1 < st.n) fetch(j + 1);
      const Cover c = cover_of(a, sp, st, j, p0, p1);
      if (c != kNone) {
        f32x16 s[2], dp[2];
        u32x4 dsf[4];
        score_tile<L, 2>(kbuf[j & 1], qf, k_rd, s);
        if (c == kPart) mask_band(s, st.key0(j), g, lo, hi, first, j < st.n_first, kNegInf);
        score_tile<L, 2>(vbuf[j & 1], df, k_rd, dp);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[u][r] = fast_exp2(fmaf(s[u][r], a.sl2, -l2)) * (dp[u][r] - delta);
        // (0 * dP is not 0 where a hidden value row holds an infinity or NaN.)
        if (c == kPart) mask_band(s, st.key0(j), g, lo, hi, first, j < st.n_first, 0.f);
        pack_p<2>(s, dsf);
        transposed_product<4>(kbuf[j & 1], dsf, t_rd, dq);
      }
      wait_vmem_all();
      __syncthreads();
    }
  }
  if (wq0 < a.Sq)
    store_columns(dq, a.scale, live, reinterpret_cast<uint8_t *>(&kbuf[0][0]) + wave * 8192,
                  a.dq + it.b * a.dqsb + it.h * a.dqsh + (int64_t)wq0 * a.dqss, a.dqss, a.Sq - wq0, lane);
}

// Backward, dK and dV: a workgroup takes 128 keys of one key head, a wave 32 of them as
// columns, and streams the queries that see them, of every head that shares the keys,
// in 64-row stages of Q and dO.  A key's queries are one interval of positions, so the
// sums run in a fixed order with no atomics.
//
// The first keys are seen by every query, the others by a window's: tiles that hold
// first keys are cut into a.pieces equal runs of stages, which leave fp32 partial sums
// in a.part for window_dkdv_sum_kernel.
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) window_dkdv_kernel(WindowArgs a) {
  using L = DualLayout;
  constexpr int kQ = 64;  // queries per stage
  __shared__ __attribute__((aligned(16))) uint16_t qbuf[2][kQ * 128], dbuf[2][kQ * 128];
  __shared__ __attribute__((aligned(16))) float stats[2][2][kQ];  // lse (log2 units), delta
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int first_items = a.first_tiles * a.pieces, per_bh = a.nkt - a.first_tiles + first_items;
  Item it = item_of(a.total, per_bh, a.Hkv);
  int piece = -1;  // of tile it.tile
  if (it.tile < first_items) {
    piece = it.tile % a.pieces;
    it.tile /= a.pieces;
  } else {
    it.tile -= first_items - a.first_tiles;
  }
  const Span sp = span_of(a, it.b);
  const int j0 = it.tile * kRows, wj0 = j0 + 32 * wave, key = wj0 + l32;
  const int j1 = (j0 + kRows < sp.len ? j0 + kRows : sp.len) - 1;

  f32x16 dk[4], dv[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) dk[dt] = dv[dt] = f32x16{0.f};
  // Rows [i_a, i_b) see some key of the tile.
  int i_a = sp.i_lo, i_b = sp.i_hi;
  if (j0 >= a.sinks) {
    i_a = j0 - a.right - sp.qs > i_a ? j0 - a.right - sp.qs : i_a;
    i_b = j1 + a.left + 1 - sp.qs < i_b ? j1 + a.left + 1 - sp.qs : i_b;
  } else if (a.causal) {
    i_a = j0 - sp.qs > i_a ? j0 - sp.qs : i_a;
  }
  // Stage t: rows i0 .. of head h; stages t_a .. t_b - 1 are this piece's.
  const int per_head = j1 >= j0 && i_b > i_a ? (i_b - i_a + kQ - 1) / kQ : 0;
  const int64_t stages = (int64_t)per_head * a.rep;
  const int64_t t_a = piece < 0 ? 0 : stages * piece / a.pieces;
  const int64_t t_b = piece < 0 ? stages : stages * (piece + 1) / a.pieces;
  if (t_b > t_a) {
    // Positions that see the lane's key.
    int plo = key - a.right, phi = key + a.left;
    if (key < a.sinks) {
      plo = a.causal ? key : -(1 << 30);
      phi = 1 << 30;
    }
    if (key >= sp.len) phi = -(1 << 30), plo = 1 << 30;
    const bool keys_whole = wj0 + 31 < sp.len;
    u32x4 kf[8], vf[8];
    load_columns(kf, a.k + it.b * a.ksb + it.h * a.ksh, a.kss, key, sp.len, g);
    load_columns(vf, a.v + it.b * a.vsb + it.h * a.vsh, a.vss, key, sp.len, g);
    TileDma<4, L, false, kQ> qdma, ddma;
    qdma.init(a.qss, wave, lane);
    ddma.init(a.gss, wave, lane);
    int h = it.h * a.rep + (int)(t_a / per_head), i0 = i_a + (int)(t_a % per_head) * kQ;
    float st_next = 0.f;
    auto fetch = [&](int buf) __attribute__((always_inline)) {
      qdma.issue(a.q + it.b * a.qsb + h * a.qsh, a.qss, i0, i_b, qbuf[buf]);
      ddma.issue(a.dout + it.b * a.gsb + h * a.gsh, a.gss, i0, i_b, dbuf[buf]);
      // Waves 0 and 1 take the rows' lse and delta; rows past the end get p = 0.
      if (wave < 2) {
        const int i = i0 + lane;
        const int64_t at = ((int64_t)it.b * a.H + h) * a.Sq + (i < i_b ? i : i_b - 1);
        const float x = wave == 0 ? a.lse[at] : a.delta[at];
        if (wave == 0) st_next = i < i_b && x != kNegInf ? x * kLog2e : -kNegInf;
        else st_next = i < i_b ? x : 0.f;
      }
    };
    fetch(0);
    if (wave < 2) stats[0][wave][lane] = st_next;
    const int k_rd = L::k_base(l32, g), t_rd = L::v_base(lane);
    wait_vmem_all();
    __syncthreads();
    const int total = (int)(t_b - t_a);
    for (int t = 0; t < total; ++t) {
      const int buf = t & 1, p_stage = sp.qs + i0, rows = i_b - i0;
      i0 += kQ;
      if (i0 >= i_b) {
        i0 = i_a;
        ++h;
      }
      if (t + 1 < total) fetch(buf ^ 1);
#pragma unroll 1  // one 32-row half's registers at a time
      for (int u = 0; u < kQ / 32; ++u) {
        const int p0 = p_stage + 32 * u, p1 = p0 + 31;
        bool none = rows <= 32 * u, all = keys_whole && rows >= 32 * u + 32;
        if (wj0 < a.sinks) {
          none = none || (a.causal && p1 < wj0);
          if (wj0 + 31 >= a.sinks) all = all && p0 >= wj0 + 31 - a.right && p1 <= a.sinks + a.left;
          else all = all && (!a.causal || p0 >= wj0 + 31);
        } else {
          none = none || p1 < wj0 - a.right || p0 > wj0 + 31 + a.left;
          all = all && p0 >= wj0 + 31 - a.right && p1 <= wj0 + a.left;
        }
        if (none) continue;
        const uint16_t *qt = qbuf[buf] + u * 32 * 128, *dt = dbuf[buf] + u * 32 * 128;
        f32x16 s[1], dp[1];
        u32x4 pf[2], dsf[2];
        score_tile<L, 1>(qt, kf, k_rd, s);
        score_tile<L, 1>(dt, vf, k_rd, dp);
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const float4 l2 = *(const float4 *)&stats[buf][0][32 * u + 8 * r4 + 4 * g];
          const float4 de = *(const float4 *)&stats[buf][1][32 * u + 8 * r4 + 4 * g];
          const float lv[4] = {l2.x, l2.y, l2.z, l2.w}, dl[4] = {de.x, de.y, de.z, de.w};
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int pos = p0 + 8 * r4 + 4 * g + r;
            float p = fast_exp2(fmaf(s[0][4 * r4 + r], a.sl2, -lv[r]));
            float ds = p * (dp[0][4 * r4 + r] - dl[r]);
            if (!all && !(pos >= plo && pos <= phi)) p = ds = 0.f;
            s[0][4 * r4 + r] = p;
            dp[0][4 * r4 + r] = ds;
          }
        }
        pack_p<1>(s, pf);
        pack_p<1>(dp, dsf);
        transposed_product<2>(dt, pf, t_rd, dv);
        transposed_product<2>(qt, dsf, t_rd, dk);
      }
      if (t + 1 < total && wave < 2) stats[buf ^ 1][wave][lane] = st_next;
      wait_vmem_all();
      __syncthreads();
    }
  }
  if (piece >= 0) {
    const int64_t bh = (int64_t)it.b * a.Hkv + it.h;
    float *part = a.part + ((bh * a.first_tiles + it.tile) * a.pieces + piece) * (2 * kRows * 128) +
                  (32 * wave + l32) * 128 + 4 * g;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int rr = 0; rr < 4; ++rr) {
        *(float4 *)(part + dt * 32 + 8 * rr) =
            float4{dk[dt][4 * rr], dk[dt][4 * rr + 1], dk[dt][4 * rr + 2], dk[dt][4 * rr + 3]};
        *(float4 *)(part + kRows * 128 + dt * 32 + 8 * rr) =
            float4{dv[dt][4 * rr], dv[dt][4 * rr + 1], dv[dt][4 * rr + 2], dv[dt][4 * rr + 3]};
      }
  } else if (wj0 < a.Skv) {
    const bool live = key < sp.len;
    uint8_t *tile = reinterpret_cast<uint8_t *>(&qbuf[0][0]) + wave * 8192;
    store_columns(dk, a.scale, live, tile, a.dk + it.b * a.dksb + it.h * a.dksh + (int64_t)wj0 * a.dkss, a.dkss,
                  a.Skv - wj0, lane);
    store_columns(dv, 1.f, live, tile, a.dv + it.b * a.dvsb + it.h * a.dvsh + (int64_t)wj0 * a.dvss, a.dvss,
                  a.Skv - wj0, lane);
  }
}

// dK and dV of the tiles that were cut: the pieces' partial sums in order.  A thread
// takes 4 dims of a key.
__global__ void __launch_bounds__(256) window_dkdv_sum_kernel(WindowArgs a) {
  const int rows = a.first_tiles * kRows, d = 4 * (threadIdx.x & 31);
  const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);  // ((b, h), dk or dv, key)
  const int key = (int)(item % rows), which = (int)(item / rows & 1);
  const int64_t bh = item / rows / 2;
  if (key >= a.Skv || bh >= (int64_t)a.B * a.Hkv) return;
  const int b = (int)(bh / a.Hkv), h = (int)(bh % a.Hkv);
  const float *p = a.part + ((bh * a.first_tiles + key / kRows) * a.pieces * 2 + which) * (kRows * 128) +
                   (key % kRows) * 128 + d;
  float4 sum = *(const float4 *)p;
  for (int i = 1; i < a.pieces; ++i) {
    const float4 x = *(const float4 *)(p + (int64_t)i * 2 * kRows * 128);
    sum.x += x.x;
    sum.y += x.y;
    sum.z += x.z;
    sum.w += x.w;
  }
  const float mul = which ? 1.f : a.scale;
  uint16_t *out = which ? a.dv + b * a.dvsb + h * a.dvsh + (int64_t)key * a.dvss
                        : a.dk + b * a.dksb + h * a.dksh + (int64_t)key * a.dkss;
  *(u32x2 *)(out + d) = u32x2{pack_bf16x2(sum.x * mul, sum.y * mul), pack_bf16x2(sum.z * mul, sum.w * mul)};
}

// Tiles that hold first keys, and the runs each is cut into: as many as make a run no
// longer than a window tile's.
static void plan_dkdv(WindowArgs &a) {
  const int64_t range = (int64_t)kRows + a.left + a.right;
  a.nkt = (a.Skv + kRows - 1) / kRows;
  a.first_tiles = (a.sinks + kRows - 1) / kRows;
  a.pieces = (int)((a.Sq + range - 1) / range);
  if (a.first_tiles == 0 || a.pieces == 1) a.first_tiles = 0, a.pieces = 1;
}

size_t window_bwd_bytes(WindowArgs a) {
  plan_dkdv(a);
  const size_t delta = ((size_t)a.B * a.H * a.Sq * sizeof(float) + 255) / 256 * 256;
  return delta + (size_t)a.B * a.Hkv * a.first_tiles * a.pieces * 2 * kRows * 128 * sizeof(float);
}

int launch_window_fwd(WindowArgs a, hipStream_t s) {
  a.nqt = (a.Sq + kRows - 1) / kRows;
  a.total = a.B * a.H * a.nqt;
  hipLaunchKernelGGL(window_fwd_kernel, dim3((unsigned)a.total), dim3(256), 0, s, a);
  return check_launch("window_fwd_kernel");
}

int launch_window_bwd(WindowArgs a, void *ws, hipStream_t s) {
  a.delta = static_cast<float *>(ws);
  a.nqt = (a.Sq + kRows - 1) / kRows;
  a.total = a.B * a.H * a.nqt;
  hipLaunchKernelGGL(window_dq_kernel, dim3((unsigned)a.total), dim3(256), 0, s, a);
  int rc = check_launch("window_dq_kernel");
  if (rc) return rc;
  plan_dkdv(a);
  a.part = a.delta + ((size_t)a.B * a.H * a.Sq + 63) / 64 * 64;
  a.total = a.B * a.Hkv * (a.nkt + a.first_tiles * (a.pieces - 1));
  hipLaunchKernelGGL(window_dkdv_kernel, dim3((unsigned)a.total), dim3(256), 0, s, a);
  rc = check_launch("window_dkdv_kernel");
  if (rc || a.first_tiles == 0) return rc;
  const int64_t rows = (int64_t)a.B * a.Hkv * a.first_tiles * kRows * 2;
  hipLaunchKernelGGL(window_dkdv_sum_kernel, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, s, a);
  return check_launch("window_dkdv_sum_kernel");
}

}  // namespace h3a
