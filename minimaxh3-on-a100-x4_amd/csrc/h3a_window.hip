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
  __device__ __forceinline__ static int v_off(int vb, int dt) { return vb ^ (64 * dt); }
  __device__ __forceinline__ static int v_off8(int off) { return off ^ 32; }  // 8 rows on, less 8 * kVRow
};
struct ValueLayout : SwzLayout {
  __device__ __forceinline__ static int v_off8(int off) { return off; }
};

// MFMAs fed from LDS in a fixed order: an operand is read kAhead instructions before the
// MFMA that takes it (left to itself the compiler reads one or two ahead and every MFMA
// waits for LDS: 40-55 % of the matrix cores' cycles).  pin_order() keeps what is written
// before it before what is written after it.
__device__ __forceinline__ void pin_order() { __builtin_amdgcn_sched_barrier(0); }

// Operand i of the scores of a 64-row stage X: rows 32 * (i % 2) .., k-step i / 2.
template <class L>
__device__ __forceinline__ u32x4 stage_operand(const uint16_t *x, int k_rd, int i) {
  return *(const u32x4 *)(reinterpret_cast<const char *>(x) + L::k_off(k_rd, i >> 1) + (i & 1) * 32 * 256);
}
// The transposed operand of acc[i % 4] for 16-row step i / 4 of tile X.
template <class L>
__device__ __forceinline__ u32x4 transposed_operand(const uint16_t *x, int t_rd, int i) {
  const char *p = reinterpret_cast<const char *>(x) + 16 * (i >> 2) * 256;
  const int off = L::v_off(t_rd, i & 3);
  const u32x2 lo = lds_read_tr16_b64(reinterpret_cast<const uint16_t *>(p + off));
  const u32x2 hi = lds_read_tr16_b64(reinterpret_cast<const uint16_t *>(p + L::v_off8(off) + 8 * 256));
  return u32x4{lo.x, lo.y, hi.x, hi.y};
}

constexpr int kAhead = 6, kAheadT = 3;

// acc += X^T F for a wave's 32 columns, where F = weigh(s) of the scores s = X xf over the
// 64 rows of a stage; the product is with Y.
template <class LX, class LY, class Weigh>
__device__ __forceinline__ void stage_single(const uint16_t *x, const uint16_t *y, const u32x4 (&xf)[8], int k_rd,
                                             int t_rd, f32x16 (&acc)[4], Weigh weigh) {
  f32x16 s[2] = {f32x16{0.f}, f32x16{0.f}};
  u32x4 a[kAhead], b[kAheadT], f[4];
  pin_order();
#pragma unroll
  for (int i = 0; i < kAhead; ++i) a[i] = stage_operand<LX>(x, k_rd, i);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    pin_order();
    s[i & 1] = mfma_32x32x16(a[i % kAhead], xf[i >> 1], s[i & 1]);
    if (i + kAhead < 16) a[i % kAhead] = stage_operand<LX>(x, k_rd, i + kAhead);
  }
#pragma unroll
  for (int i = 0; i < kAheadT; ++i) b[i] = transposed_operand<LY>(y, t_rd, i);
  pin_order();
  weigh(s, f);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    pin_order();
    acc[i & 3] = mfma_32x32x16(b[i % kAheadT], f[i >> 2], acc[i & 3]);
    if (i + kAheadT < 16) b[i % kAheadT] = transposed_operand<LY>(y, t_rd, i + kAheadT);
  }
  pin_order();
}

// The same with F = weigh(s, dp) of two scores, s = X xf and dp = Y yf, and the product
// with X: 32 rows at a time, the two chains of MFMAs side by side.
template <class L, class Weigh>
__device__ __forceinline__ void stage_pair(const uint16_t *x, const uint16_t *y, const u32x4 (&xf)[8],
                                           const u32x4 (&yf)[8], int k_rd, int t_rd, f32x16 (&acc)[4], Weigh weigh) {
  auto operand = [&](int u, int i) __attribute__((always_inline)) {
    return *(const u32x4 *)(reinterpret_cast<const char *>(i & 1 ? y : x) + L::k_off(k_rd, i >> 1) + u * 32 * 256);
  };
  u32x4 a[kAhead];
  pin_order();
#pragma unroll
  for (int i = 0; i < kAhead; ++i) a[i] = operand(0, i);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    f32x16 s = {0.f}, dp = {0.f};
    u32x4 b[kAheadT], f[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      pin_order();
      if (i & 1) dp = mfma_32x32x16(a[i % kAhead], yf[i >> 1], dp);
      else s = mfma_32x32x16(a[i % kAhead], xf[i >> 1], s);
      if (i + kAhead < 16) a[i % kAhead] = operand(u, i + kAhead);
    }
#pragma unroll
    for (int i = 0; i < kAheadT; ++i) b[i] = transposed_operand<L>(x + u * 32 * 128, t_rd, i);
    pin_order();
    weigh(u, s, dp, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      pin_order();
      acc[i & 3] = mfma_32x32x16(b[i % kAheadT], f[i >> 2], acc[i & 3]);
      if (i + kAheadT < 8) {
        b[i % kAheadT] = transposed_operand<L>(x + u * 32 * 128, t_rd, i + kAheadT);
      } else if (u == 0) {  // the other half's first operands
        a[2 * (i + kAheadT - 8)] = operand(1, 2 * (i + kAheadT - 8));
        a[2 * (i + kAheadT - 8) + 1] = operand(1, 2 * (i + kAheadT - 8) + 1);
      }
    }
  }
  pin_order();
}
static_assert(kAhead == 2 * kAheadT, "stage_pair: the last products fetch the next scores' operands");

// Stages 0 .. n-1 of two LDS buffers in turn, as code of their own, so that every LDS
// address is a register and a constant.
template <int P>
using C = std::integral_constant<int, P>;
template <class Stage>
__device__ __forceinline__ void two_buffers(int n, Stage stage) {
  for (int j = 0; j < n; j += 2) {
    stage(C<0>{}, j);
    if (j + 1 < n) stage(C<1>{}, j + 1);
  }
}

// A wave's 32 rows as columns of an MFMA operand, straight from global memory; rows
// past `rows` are zeros: the loads (row 0 for those), and what makes them zeros.
__device__ __forceinline__ void issue_columns(u32x4 (&f)[8], const uint16_t *base, int64_t stride, int row, int rows,
                                              int g) {
  const uint16_t *p = base + (int64_t)(row < rows ? row : 0) * stride + 8 * g;
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) f[ks] = *(const u32x4 *)(p + 16 * ks);
}
__device__ __forceinline__ void clear_past(u32x4 (&f)[8], int row, int rows) {
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) f[ks] = row < rows ? f[ks] : u32x4{0, 0, 0, 0};
}
__device__ __forceinline__ void load_columns(u32x4 (&f)[8], const uint16_t *base, int64_t stride, int row, int rows,
                                             int g) {
  issue_columns(f, base, stride, row, rows, g);
  clear_past(f, row, rows);
}

// The same products 32 rows at a time, in the compiler's order: scores of the rows of X, and
// acc += Y^T F.
template <class L>
__device__ __forceinline__ f32x16 scores_32(const uint16_t *x, const u32x4 (&xf)[8], int k_rd) {
  f32x16 s[1];
  score_tile<L, 1>(x, xf, k_rd, s);
  return s[0];
}
template <class L>
__device__ __forceinline__ void product_32(f32x16 (&acc)[4], const uint16_t *y, const f32x16 &w, int t_rd) {
  const f32x16 ws[1] = {w};
  u32x4 f[2];
  pack_p<1>(ws, f);
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i & 3] = mfma_32x32x16(transposed_operand<L>(y, t_rd, i), f[i >> 2], acc[i & 3]);
}
__device__ __forceinline__ void clear(f32x16 (&acc)[4]) {
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) acc[dt] = f32x16{0.f};
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

// The kernels' products multiply a hidden pair's weight, 0, with what the hidden row holds,
// which is not 0 where that is an infinity or NaN.  So where a sum of a tile is not finite,
// its stages are walked a second time: the values that are not finite are taken out of the
// LDS tile that the product reads, once their places are noted, and every column is told
// which of its sums a row that it sees makes infinite or NaN.  That is a second pass over the
// same matrix products, whatever the values are and whoever sees them; its loops are simple
// ones, one buffer and 32 rows at a time, so that they need no more registers than the first
// pass's.  At H=16 S=4096, 511 keys to either side: forward 0.053 ms, with one bad row of V
// 0.135 (each spoiled column summed again by itself: 6.0), with a bad channel of V 0.49 (6.4);
// backward 0.20 ms, with one bad row of V 0.30 (8.8), with dO all infinite 0.81.

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// Whether one of the wave's sums that count is not finite (the same on all lanes).
__device__ __forceinline__ bool spoiled(const f32x16 (&acc)[4], bool counts) {
  bool bad = false;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) bad |= !finite(acc[dt][r]);
  return __builtin_amdgcn_ballot_w64(bad && counts) != 0;
}

// Whether a flag is set in one of a workgroup's four waves.
__device__ __forceinline__ bool any_wave(bool flag, int (&flags)[4], int wave, int lane) {
  if (lane == 0) flags[wave] = flag;
  __syncthreads();
  return (flags[0] | flags[1] | flags[2] | flags[3]) != 0;
}

// Where a stage's values are not finite: bit e of [row][c] is element 8*c + e; `up` for
// +infinity, `down` for -infinity, both for NaN.
template <int ROWS>
struct BadValues {
  __attribute__((aligned(16))) uint8_t up[ROWS][16], down[ROWS][16];
};

// Takes the values that are not finite out of a stage, and notes them: zeros in their
// place, or (kWhole) in that of their whole row.  By NT threads.
template <class L, bool kIsV, int ROWS, int NT, bool kWhole>
__device__ __forceinline__ void take_out(uint16_t *tile, BadValues<ROWS> &bad, int thread) {
#pragma unroll 1
  for (int at = thread; at < ROWS * 16; at += NT) {
    const int row = at >> 4, slot = at & 15, chunk = kIsV ? L::v_chunk(row, slot) : L::k_chunk(row, slot);
    u32x4 x = *(const u32x4 *)(tile + 8 * at);
    uint32_t up = 0, down = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t v = x[e >> 1] >> (16 * (e & 1)) & 0xffffu;
      if ((v & 0x7f80u) != 0x7f80u) continue;
      if (v & 0x7fu || !(v & 0x8000u)) up |= 1u << e;
      if (v & 0x7fu || v & 0x8000u) down |= 1u << e;
      x[e >> 1] &= e & 1 ? 0x0000ffffu : 0xffff0000u;
    }
    bad.up[row][chunk] = (uint8_t)up;
    bad.down[row][chunk] = (uint8_t)down;
    const uint64_t lanes = __builtin_amdgcn_ballot_w64((up | down) != 0);  // a row's 16 chunks: 16 lanes
    if (kWhole && lanes >> (thread & 48) & 0xffffu) x = u32x4{0, 0, 0, 0};
    if (lanes) *(u32x4 *)(tile + 8 * at) = x;
  }
}

// The rows of a stage that hold such values, and 0 for the weights of those rows (32 of
// them, in the accumulators' order).
template <int ROWS>
__device__ __forceinline__ uint64_t bad_rows(const BadValues<ROWS> &bad, int lane) {
  const u32x4 any = *(const u32x4 *)bad.up[lane % ROWS] | *(const u32x4 *)bad.down[lane % ROWS];
  return __builtin_amdgcn_ballot_w64(lane < ROWS && (any[0] | any[1] | any[2] | any[3]) != 0);
}
__device__ __forceinline__ void drop_rows(f32x16 &w, uint32_t rows, int g) {
#pragma unroll
  for (int r = 0; r < 16; ++r)
    if (rows >> (8 * (r >> 2) + 4 * g + (r & 3)) & 1) w[r] = 0.f;
}

// The sums of a lane's column that rows it sees make infinite or NaN: bit 16*dt + r is
// acc[dt][r].  kSigns: the weights are probabilities, and an infinity keeps its sign; the
// others' are 0 or NaN, and so NaN is what either makes.
template <bool kSigns>
struct BadSums {
  uint64_t up = 0, down = 0;
  // Bits 4*c .. 4*c + 3: the lane half's four bits of byte c.
  __device__ __forceinline__ static uint64_t half_bits(u32x4 row, int g) {
    uint64_t bits = 0;
#pragma unroll
    for (int k = 3; k >= 0; --k) {
      uint32_t x = row[k] >> (4 * g) & 0x0f0f0f0fu;
      x = (x | x >> 4) & 0x00ff00ffu;
      bits = bits << 16 | ((x | x >> 8) & 0xffffu);
    }
    return bits;
  }
  // A stage's: sees(i), whether the lane's column sees row i, all(i), whether that makes all
  // of its sums NaN (the row's weight being that).
  template <int ROWS, class Sees, class All>
  __device__ __forceinline__ void add(const BadValues<ROWS> &bad, int lane, Sees sees, All all) {
    for (uint64_t rows = bad_rows(bad, lane); rows; rows &= rows - 1) {
      const int i = __builtin_ctzll(rows);
      const bool seen = sees(i);
      if (__builtin_amdgcn_ballot_w64(seen && (kSigns ? up & down : up) != ~0ull) == 0) continue;
      if (seen) {
        const u32x4 u = *(const u32x4 *)bad.up[i], d = *(const u32x4 *)bad.down[i];
        const uint64_t every = all(i) ? ~0ull : 0;
        up |= half_bits(kSigns ? u : u | d, lane >> 5) | every;
        if (kSigns) down |= half_bits(d, lane >> 5) | every;
      }
    }
  }
  __device__ __forceinline__ void put(f32x16 (&acc)[4]) const {
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const bool u = up >> (16 * dt + r) & 1, d = kSigns ? down >> (16 * dt + r) & 1 : u;
        if (u || d) acc[dt][r] += u && d ? __builtin_nanf("") : (u ? -kNegInf : kNegInf);
      }
  }
};

// Natural logarithm of l * 2^m: -inf for an empty sum, l where that is not finite.
__device__ __forceinline__ float log_sum(float m, float l) {
  return !finite(l) ? l : (l > 0.f ? (m + log2f(l)) * kLn2 : kNegInf);
}

// DMA of the rows of [row0, limit) that a tile holds, the rest as zeros.
template <class Dma>
__device__ __forceinline__ void fetch_tile(const Dma &dma, const uint16_t *base, int64_t stride, int row0, int limit,
                                           uint16_t *tile) {
  dma.template issue_desc<0, Dma::kInst>(dma.desc(base, stride, row0, limit), tile);
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
template <int BN = kBN>
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
      n_first = (first + BN - 1) / BN;
    }
    n = n_first + (hi - lo + BN - 1) / BN;
  }
  __device__ __forceinline__ int key0(int j) const { return j < n_first ? j * BN : lo + (j - n_first) * BN; }
  __device__ __forceinline__ int limit(int j) const { return j < n_first ? first : hi; }
};

// What a wave at positions p0 .. p1 sees of a stage: nothing, all of it, or a part.
enum Cover { kNone, kAll, kPart };
template <int BN>
__device__ __forceinline__ Cover cover_of(const WindowArgs &a, const Span &s, const KeyStages<BN> &ks, int j, int p0,
                                          int p1) {
  const int k0 = ks.key0(j), k1 = k0 + BN - 1;
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
template <int NSUB>
__device__ __forceinline__ void mask_band(f32x16 (&s)[NSUB], int key0, int g, int lo, int hi, int first, bool only_first,
                                          float hidden) {
  const int l = only_first ? 1 << 30 : lo;
#pragma unroll
  for (int u = 0; u < NSUB; ++u)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int j = key0 + 32 * u + 8 * (r >> 2) + 4 * g + (r & 3);
      if (!((j >= l && j <= hi) || j < first)) s[u][r] = hidden;
    }
}

// Work items: `tiles` per head, dealt to the XCDs in runs of `chunk` consecutive ones, so
// that neighbours, which read nearly the same keys, share an L2.  Workgroup i runs on
// XCD i % 8; which of a round's 8 runs an XCD gets is rotated by a hash of the round, so
// that no XCD is left with all the short ends of a padded batch, whatever the number of
// runs per head (B=2 H=56/8 S=8192, one sequence less than half as long: forward 1.03 ->
// 0.77 ms against one contiguous range per XCD).
struct Item {
  int tile, h, b;  // tile < 0: none
};
__device__ __forceinline__ Item item_of(const WindowArgs &a, int i, int chunk, int tiles, int heads) {
  const int x = i & 7, k = i >> 3;
  const int n = k / chunk, run = n * 8 + ((x + (int)((uint32_t)n * 2654435761u >> 29)) & 7);
  const int runs = (tiles + chunk - 1) / chunk, bh = run / runs;
  const int tile = (run % runs) * chunk + k % chunk;
  return {bh < a.B * heads && tile < tiles ? tile : -1, bh % heads, bh / heads};
}

// Forward.  A workgroup takes 128 query rows of one head, a wave 32 of them; the
// 64-key stages of their window are double-buffered in LDS by DMA, two workgroups to a
// CU, so that one's softmax overlaps the other's MFMAs.  The softmax runs against a stale
// maximum (a row's maximum per stage instead: 9.27 ms for 9.10 at H=56 S=42120 with 4096
// keys to either side and 512 first ones, 780 us for 763 at B=2 H=56 S=8192, 1024 and
// 256).  Bound by the MFMAs: 1.09 PFLOP/s of the visible pairs there, a large library
// matrix product reaching 1.21.  Two groups of four waves that take turns at the MFMAs
// and the softmax, a barrier after each turn: 1.21 ms for 0.73 at S=8192.
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) window_fwd_kernel(WindowArgs a) {
  using L = SwzLayout;
  __shared__ __attribute__((aligned(16))) uint16_t kbuf[2][StageBytes<L>::kK / 2], vbuf[2][StageBytes<L>::kV / 2];
  __shared__ BadValues<kBN> bad;
  __shared__ int flags[4];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Item it = item_of(a, (int)blockIdx.x, a.chunk, a.nqt, a.H);
  if (it.tile < 0) return;
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
    KeyStages<> st;
    st.init(a, sp, sp.qs + r0, sp.qs + r1);
    const int lo = pos - a.left, first = first_keys(a, sp, pos);
    const int hi = pos + a.right < sp.len - 1 ? pos + a.right : sp.len - 1;
    TileDma<4, L, false> kdma;
    TileDma<4, L, true> vdma;
    kdma.init(a.kss, wave, lane);
    vdma.init(a.vss, wave, lane);
    auto fetch = [&](int j, auto par) __attribute__((always_inline)) {
      constexpr int P = decltype(par)::value;
      fetch_tile(kdma, Kb, a.kss, st.key0(j), st.limit(j), kbuf[P]);
      fetch_tile(vdma, Vb, a.vss, st.key0(j), st.limit(j), vbuf[P]);
    };
    fetch(0, C<0>{});
    u32x4 qf[8];
    load_columns(qf, a.q + it.b * a.qsb + it.h * a.qsh, a.qss, row, a.Sq, g);
    const int k_rd = L::k_base(l32, g), v_rd = L::v_base(lane);
    wait_vmem_all();
    __syncthreads();
    two_buffers(st.n, [&](auto par, int j) __attribute__((always_inline)) {
      constexpr int P = decltype(par)::value;
      if (j + 1 < st.n) fetch(j + 1, C<P ^ 1>{});
      const Cover c = cover_of(a, sp, st, j, p0, p1);
      if (c != kNone)
        stage_single<L, ValueLayout>(kbuf[P], vbuf[P], qf, k_rd, v_rd, o,
                                     [&](f32x16(&s)[2], u32x4(&pf)[4]) __attribute__((always_inline)) {
                                       if (c == kPart) mask_band(s, st.key0(j), g, lo, hi, first, j < st.n_first, kNegInf);
                                       softmax_stage_stale<2, true>(s, 0, kBN, g, a.sl2, m, lsum, o, pf);
                                     });
      wait_vmem_all();
      __syncthreads();
    });
    // (A column whose own scores are not finite is NaN throughout, whatever V holds.)
    if (any_wave(spoiled(o, live && finite(half_swap_sum(lsum))), flags, wave, lane)) {
      BadSums<true> seen;
      clear(o);
      m = kNegInf, lsum = 0.f;
      for (int j = 0; j < st.n; ++j) {
        fetch(j, C<0>{});
        wait_vmem_all();
        __syncthreads();
        take_out<L, true, kBN, 256, false>(vbuf[0], bad, tid);
        __syncthreads();
#pragma unroll 1
        for (int u = 0; u < 2; ++u) {
          f32x16 s[1] = {scores_32<L>(kbuf[0] + u * 32 * 128, qf, k_rd)};
          u32x4 pf[2];
          mask_band(s, st.key0(j) + 32 * u, g, lo, hi, first, j < st.n_first, kNegInf);
          softmax_stage<1>(s, 0, 32, g, a.sl2, m, lsum, o, pf);
          pv_tile<L, 2>(vbuf[0] + u * 32 * 128, pf, v_rd, o);
        }
        seen.add(bad, lane, [&](int i) {
          const int key = st.key0(j) + i;
          return (j >= st.n_first && key >= lo && key <= hi) || key < first;
        }, [](int) { return false; });
        __syncthreads();
      }
      seen.put(o);
    }
  }
  const float ltot = half_swap_sum(lsum);
  const float inv = ltot > 0.f ? 1.f / ltot : 0.f;
  if (a.lse && g == 0 && row < a.Sq)
    a.lse[((int64_t)it.b * a.H + it.h) * a.Sq + row] = live ? log_sum(m, ltot) : kNegInf;
  if (wq0 < a.Sq)
    store_columns(o, inv, live, reinterpret_cast<uint8_t *>(&kbuf[0][0]) + wave * 8192,
                  a.o + it.b * a.osb + it.h * a.osh + (int64_t)wq0 * a.oss, a.oss, a.Sq - wq0, lane);
}

// Forward for few query rows (a new token, or a short chunk of them, against a cache).
// Bound by the bytes of K and V, so the rows of all heads that share a key head ride
// together as columns, 32 to a workgroup, and the keys are split: over a.pieces
// workgroups, and within one over its four waves, each with its own running softmax and
// its own double-buffered 32-key stages (no barrier until the end).  The waves merge
// through LDS, the workgroups through a.part and window_token_sum_kernel.
constexpr int kTokenStage = 32, kTokenRows = 32;
struct TokenLds {
  uint16_t k[4][2][kTokenStage * 128], v[4][2][kTokenStage * 128];  // by wave
  BadValues<kTokenStage> bad[4];
};

// Column c of a key head's group of 32 -> query row and head among those that share it
// (row >= Sq: none).  Sequences of 32 rows or more fill groups head by head, so that a
// group's rows are consecutive; shorter ones run on from head to head.
struct TokenColumn {
  int row, head;
};
__device__ __forceinline__ TokenColumn token_column(const WindowArgs &a, int group, int c) {
  if (a.Sq >= kTokenRows) {
    const int per_head = (a.Sq + kTokenRows - 1) / kTokenRows;
    return {group % per_head * kTokenRows + c, group / per_head};
  }
  const int col = group * kTokenRows + c;
  return {col < a.rep * a.Sq ? col % a.Sq : a.Sq, col / a.Sq};
}

__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) window_token_kernel(WindowArgs a) {
  using L = SwzLayout;
  __shared__ __attribute__((aligned(16))) TokenLds lds;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int piece = (int)blockIdx.x % a.pieces, unit = (int)blockIdx.x / a.pieces;
  const int group = unit % a.nqt, bh = unit / a.nqt, hk = bh % a.Hkv, b = bh / a.Hkv;
  const Span sp = span_of(a, b);
  const TokenColumn at = token_column(a, group, l32);
  const bool has = at.row < a.Sq;
  const int h = hk * a.rep + (has ? at.head : 0), row = has ? at.row : 0;
  // The rows the workgroup's keys are for: its 32, or all of a short sequence.
  const int c0 = a.Sq < kTokenRows ? 0 : __builtin_amdgcn_readfirstlane(token_column(a, group, 0).row);
  const int r0 = c0 > sp.i_lo ? c0 : sp.i_lo, r1 = (c0 + kTokenRows < sp.i_hi ? c0 + kTokenRows : sp.i_hi) - 1;
  const bool live = has && row >= r0 && row <= r1;

  f32x16 o[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) o[dt] = f32x16{0.f};
  float m = kNegInf, lsum = 0.f;
  if (r1 >= r0) {
    const int p0 = sp.qs + r0, p1 = sp.qs + r1;
    const int pos = sp.qs + (row < r0 ? r0 : (row > r1 ? r1 : row));
    KeyStages<kTokenStage> st;
    st.init(a, sp, p0, p1);
    const int lo = pos - a.left, first = first_keys(a, sp, pos);
    const int hi = pos + a.right < sp.len - 1 ? pos + a.right : sp.len - 1;
    const int j_a = (int)((int64_t)st.n * piece / a.pieces), j_b = (int)((int64_t)st.n * (piece + 1) / a.pieces);
    const uint16_t *Kb = a.k + b * a.ksb + hk * a.ksh, *Vb = a.v + b * a.vsb + hk * a.vsh;
    TileDma<1, L, false, kTokenStage> kdma;
    TileDma<1, L, true, kTokenStage> vdma;
    kdma.init(a.kss, 0, lane);
    vdma.init(a.vss, 0, lane);
    constexpr int kInst = decltype(kdma)::kInst + decltype(vdma)::kInst;
    auto fetch = [&](int j, int buf) __attribute__((always_inline)) {
      fetch_tile(kdma, Kb, a.kss, st.key0(j), st.limit(j), lds.k[wave][buf]);
      fetch_tile(vdma, Vb, a.vss, st.key0(j), st.limit(j), lds.v[wave][buf]);
    };
    int j = j_a + wave;
    if (j < j_b) fetch(j, 0);
    u32x4 qf[8];
    load_columns(qf, a.q + b * a.qsb + h * a.qsh, a.qss, row, a.Sq, g);
    const int k_rd = L::k_base(l32, g), v_rd = L::v_base(lane);
    for (int buf = 0; j < j_b; j += 4, buf ^= 1) {
      // The other buffer's last reads have returned; its next stage goes out before this
      // one is waited for.
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (j + 4 < j_b) {
        fetch(j + 4, buf ^ 1);
        wait_vmem_le<kInst>();
      } else {
        wait_vmem_all();
      }
      asm volatile("" ::: "memory");
      f32x16 s[1];
      u32x4 pf[2];
      score_tile<L, 1>(lds.k[wave][buf], qf, k_rd, s);
      if (cover_of(a, sp, st, j, p0, p1) != kAll)
        mask_band(s, st.key0(j), g, lo, hi, first, j < st.n_first, kNegInf);
      softmax_stage<1>(s, 0, kTokenStage, g, a.sl2, m, lsum, o, pf);
      pv_tile<L, 2>(lds.v[wave][buf], pf, v_rd, o);
    }
    if (spoiled(o, live && finite(half_swap_sum(lsum)))) {
      BadSums<true> seen;
      clear(o);
      m = kNegInf, lsum = 0.f;
      for (j = j_a + wave; j < j_b; j += 4) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        fetch(j, 0);
        wait_vmem_all();
        asm volatile("" ::: "memory");
        take_out<L, true, kTokenStage, 64, false>(lds.v[wave][0], lds.bad[wave], lane);
        f32x16 s[1] = {scores_32<L>(lds.k[wave][0], qf, k_rd)};
        u32x4 pf[2];
        mask_band(s, st.key0(j), g, lo, hi, first, j < st.n_first, kNegInf);
        softmax_stage<1>(s, 0, kTokenStage, g, a.sl2, m, lsum, o, pf);
        pv_tile<L, 2>(lds.v[wave][0], pf, v_rd, o);
        seen.add(lds.bad[wave], lane, [&](int i) {
          const int key = st.key0(j) + i;
          return (j >= st.n_first && key >= lo && key <= hi) || key < first;
        }, [](int) { return false; });
      }
      seen.put(o);
    }
  }
  // Merge the waves: wave u takes dims 32u .. 32u+31 of all four.
  __syncthreads();
  float *xch = reinterpret_cast<float *>(&lds.k[0][0][0]);           // [wave][dims / 32][register][lane]
  float2 *ml = reinterpret_cast<float2 *>(&lds.v[0][0][0]);          // [wave][lane]
  const float ltot = half_swap_sum(lsum);
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) xch[((wave * 4 + dt) * 16 + r) * 64 + lane] = o[dt][r];
  ml[wave * 64 + lane] = float2{m, ltot};
  __syncthreads();
  float top = kNegInf, l = 0.f, w[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) top = fmaxf(top, ml[u * 64 + lane].x);
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const float2 x = ml[u * 64 + lane];
    w[u] = x.x == kNegInf ? 0.f : fast_exp2(x.x - top);
    l = fmaf(x.y, w[u], l);
  }
  const float inv = a.pieces > 1 ? 1.f : (l > 0.f ? 1.f / l : 0.f);
  const int64_t slot = ((int64_t)unit * a.pieces + piece) * kTokenRows + l32;
#pragma unroll
  for (int r4 = 0; r4 < 4; ++r4) {
    float x[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < 4; ++u) sum = fmaf(w[u], xch[((u * 4 + wave) * 16 + 4 * r4 + r) * 64 + lane], sum);
      x[r] = live ? sum * inv : 0.f;
    }
    const int d = 32 * wave + 8 * r4 + 4 * g;
    if (a.pieces > 1) *(float4 *)(a.part + slot * 128 + d) = float4{x[0], x[1], x[2], x[3]};
    else if (has)
      *(u32x2 *)(a.o + b * a.osb + h * a.osh + row * a.oss + d) = u32x2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
  }
  if (wave == 0 && g == 0) {
    if (a.pieces > 1) {
      float *stat = a.part + (int64_t)gridDim.x * kTokenRows * 128 + slot * 2;
      *(float2 *)stat = live ? float2{top, l} : float2{kNegInf, 0.f};
    } else if (a.lse && has) {
      a.lse[((int64_t)b * a.H + h) * a.Sq + row] = live ? log_sum(top, l) : kNegInf;
    }
  }
}

// The pieces of a split key range: O = sum 2^(m_p - M) O_p / sum 2^(m_p - M) l_p.  A
// workgroup takes a row: 32 lanes of 4 dims, 8 groups of them over the pieces, each with
// all its loads in flight (28 rows of 33 pieces: 21 us as one walk per thread).
constexpr int kTokenPieces = 64;
__global__ void __launch_bounds__(256) window_token_sum_kernel(WindowArgs a, int units) {
  __shared__ float4 part[8][32];
  __shared__ float2 stat[8];
  constexpr int kPer = kTokenPieces / 8;
  const int unit = (int)(blockIdx.x / kTokenRows), c = (int)(blockIdx.x % kTokenRows);
  const int grp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = 4 * lane;
  const int group = unit % a.nqt, bh = unit / a.nqt, hk = bh % a.Hkv, b = bh / a.Hkv;
  const TokenColumn tc = token_column(a, group, c);
  if (tc.row >= a.Sq) return;
  const int h = hk * a.rep + tc.head, row = tc.row;
  const float *ml = a.part + (int64_t)units * a.pieces * kTokenRows * 128;
  const int64_t slot = (int64_t)unit * a.pieces * kTokenRows + c;
  float2 x[kPer];
  float4 v[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int p = grp + 8 * i;
    const int64_t at = slot + (int64_t)(p < a.pieces ? p : 0) * kTokenRows;
    x[i] = p < a.pieces ? *(const float2 *)(ml + at * 2) : float2{kNegInf, 0.f};
    v[i] = p < a.pieces ? *(const float4 *)(a.part + at * 128 + d) : float4{0.f, 0.f, 0.f, 0.f};
  }
  float top = kNegInf;
#pragma unroll
  for (int i = 0; i < kPer; ++i) top = fmaxf(top, x[i].x);
  float4 acc = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
  auto add = [&](float m, float lp, const float4 &o) __attribute__((always_inline)) {
    const float w = m == kNegInf ? 0.f : fast_exp2(m - top);
    acc.x = fmaf(w, o.x, acc.x);
    acc.y = fmaf(w, o.y, acc.y);
    acc.z = fmaf(w, o.z, acc.z);
    acc.w = fmaf(w, o.w, acc.w);
    l = fmaf(w, lp, l);
  };
#pragma unroll
  for (int i = 0; i < kPer; ++i) add(x[i].x, x[i].y, v[i]);
  part[grp][lane] = acc;
  if (lane == 0) stat[grp] = float2{top, l};
  __syncthreads();
  if (grp != 0) return;
  top = kNegInf;
  acc = {0.f, 0.f, 0.f, 0.f};
  l = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, stat[i].x);
#pragma unroll
  for (int i = 0; i < 8; ++i) add(stat[i].x, stat[i].y, part[i][lane]);
  const float inv = l > 0.f ? 1.f / l : 0.f;
  *(u32x2 *)(a.o + b * a.osb + h * a.osh + row * a.oss + d) =
      u32x2{pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv)};
  if (a.lse && d == 0) a.lse[((int64_t)b * a.H + h) * a.Sq + row] = log_sum(top, l);
}

// Whether a run of positions p0 .. p1 holds one that sees no more than a stage of keys (the
// window's part of the count is least at an end of the run).
__device__ __forceinline__ bool few_keys(const WindowArgs &a, const Span &s, int p0, int p1) {
  KeyStages<1> st0, st1;
  st0.init(a, s, p0, p0);
  st1.init(a, s, p1, p1);
  return st0.n <= kBN || st1.n <= kBN;
}

// Backward, dQ: tiles and stages as forward, with P from the stored lse.  The rows' lse
// (log2 units; +inf, so that p = 0, for a row that saw nothing) and delta = dO.O go to
// a.stats for the second kernel.  O's rounding to bf16 makes delta off by up to 2^-8 of what the
// few keys of a row near a sequence's start or under a narrow window give, which there is
// as much as dS itself (a row of one key has dS = 0): such tiles take sum p dP in a pass of
// their own instead (relative error of dQ and dK, S=100 causal: 0.0029 -> 0.0024, which is
// the rounding of dS and of the result; from 64 keys on delta's part is under a fifth).
// The pass takes 55 us of a backward's 319 at H=56/8 S=8192 with 17 keys to a row.
// Bound by the MFMAs: 0.99 ms for the 1.06 TFLOP of B=2 H=56/8 S=8192, 1024 keys to either
// side and 256 first ones, one sequence less than half as long.
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) window_dq_kernel(WindowArgs a) {
  using L = DualLayout;
  __shared__ __attribute__((aligned(16))) uint16_t kbuf[2][StageBytes<L>::kK / 2], vbuf[2][StageBytes<L>::kK / 2];
  __shared__ BadValues<kBN> bad;
  __shared__ int flags[4];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Item it = item_of(a, (int)blockIdx.x, a.chunk, a.nqt, a.H);
  if (it.tile < 0) return;
  const Span sp = span_of(a, it.b);
  const int q0 = it.tile * kRows, wq0 = q0 + 32 * wave, row = wq0 + l32;
  const int r0 = q0 > sp.i_lo ? q0 : sp.i_lo, r1 = (q0 + kRows < sp.i_hi ? q0 + kRows : sp.i_hi) - 1;
  const bool live = row >= sp.i_lo && row < sp.i_hi;
  const uint16_t *Kb = a.k + it.b * a.ksb + (it.h / a.rep) * a.ksh;
  const uint16_t *Vb = a.v + it.b * a.vsb + (it.h / a.rep) * a.vsh;

  f32x16 dq[4];
  float delta = 0.f, l2 = 0.f;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) dq[dt] = f32x16{0.f};
  if (r1 >= r0) {
    auto clamp_row = [&](int i) __attribute__((always_inline)) { return i < r0 ? r0 : (i > r1 ? r1 : i); };
    const int p0 = sp.qs + clamp_row(wq0), p1 = sp.qs + clamp_row(wq0 + 31), pos = sp.qs + clamp_row(row);
    KeyStages<> st;
    st.init(a, sp, sp.qs + r0, sp.qs + r1);
    const int lo = pos - a.left, first = first_keys(a, sp, pos);
    const int hi = pos + a.right < sp.len - 1 ? pos + a.right : sp.len - 1;
    TileDma<4, L, false> kdma, vdma;
    kdma.init(a.kss, wave, lane);
    vdma.init(a.vss, wave, lane);
    auto fetch = [&](int j, auto par) __attribute__((always_inline)) {
      constexpr int P = decltype(par)::value;
      fetch_tile(kdma, Kb, a.kss, st.key0(j), st.limit(j), kbuf[P]);
      fetch_tile(vdma, Vb, a.vss, st.key0(j), st.limit(j), vbuf[P]);
    };
    fetch(0, C<0>{});
    // All of them in flight at once.
    u32x4 qf[8], df[8], of[8];
    const int64_t stat = ((int64_t)it.b * a.H + it.h) * a.Sq + (row < a.Sq ? row : a.Sq - 1);
    issue_columns(qf, a.q + it.b * a.qsb + it.h * a.qsh, a.qss, row, a.Sq, g);
    issue_columns(df, a.dout + it.b * a.gsb + it.h * a.gsh, a.gss, row, a.Sq, g);
    issue_columns(of, a.o + it.b * a.osb + it.h * a.osh, a.oss, row, a.Sq, g);
    const float lse = a.lse[stat];
    pin_order();
    clear_past(qf, row, a.Sq);
    clear_past(df, row, a.Sq);
    clear_past(of, row, a.Sq);
    l2 = lse == kNegInf ? -kNegInf : lse * kLog2e;
    const int k_rd = L::k_base(l32, g), t_rd = L::v_base(lane);
    if (few_keys(a, sp, sp.qs + r0, sp.qs + r1)) {
      wait_vmem_all();
      __syncthreads();
      two_buffers(st.n, [&](auto par, int j) __attribute__((always_inline)) {
        constexpr int P = decltype(par)::value;
        if (j + 1 < st.n) fetch(j + 1, C<P ^ 1>{});
        f32x16 s[2], dp[2];
        score_tile<L, 2>(kbuf[P], qf, k_rd, s);
        score_tile<L, 2>(vbuf[P], df, k_rd, dp);
        const int key0 = st.key0(j) + 4 * g, low = j < st.n_first ? 1 << 30 : lo;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int at = key0 + 32 * u + 8 * (r >> 2) + (r & 3);
            if ((at >= low && at <= hi) || at < first)
              delta = fmaf(fast_exp2(fmaf(s[u][r], a.sl2, -l2)), dp[u][r], delta);
          }
        wait_vmem_all();
        __syncthreads();
      });
      if (st.n > 2) fetch(0, C<0>{});  // (two stages are both still there)
    } else {
#pragma unroll
      for (int ks = 0; ks < 8; ++ks)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          delta = fmaf(bf16_hi(of[ks][i]), bf16_hi(df[ks][i]), fmaf(bf16_lo(of[ks][i]), bf16_lo(df[ks][i]), delta));
    }
    delta = half_swap_sum(delta);
    if (g == 0 && row < a.Sq) {
      a.stats[stat] = l2;
      a.stats[a.stats_n + stat] = delta;
    }
    wait_vmem_all();
    __syncthreads();
    two_buffers(st.n, [&](auto par, int j) __attribute__((always_inline)) {
      constexpr int P = decltype(par)::value;
      if (j + 1 < st.n) fetch(j + 1, C<P ^ 1>{});
      const Cover c = cover_of(a, sp, st, j, p0, p1);
      if (c != kNone)
        stage_pair<L>(kbuf[P], vbuf[P], qf, df, k_rd, t_rd, dq,
                      [&](int u, f32x16 &s, const f32x16 &dp, u32x4 (&f)[2]) __attribute__((always_inline)) {
                        f32x16 ds[1];
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                          ds[0][r] = fast_exp2(fmaf(s[r], a.sl2, -l2)) * (dp[r] - delta);
                        if (c == kPart) {
                          const int key0 = st.key0(j) + 32 * u + 4 * g, low = j < st.n_first ? 1 << 30 : lo;
#pragma unroll
                          for (int r = 0; r < 16; ++r) {
                            const int at = key0 + 8 * (r >> 2) + (r & 3);
                            if (!((at >= low && at <= hi) || at < first)) ds[0][r] = 0.f;
                          }
                        }
                        pack_p<1>(ds, f);
                      });
      wait_vmem_all();
      __syncthreads();
    });
    // (A row whose own statistics are not finite is NaN throughout.)  Rows of K that are not
    // finite are taken out whole, with weight 0: K is also what the scores are from, and in a
    // row whose lse is finite the score of such a key is -inf.
    const bool own = !finite(delta) || l2 != l2;
    if (any_wave(spoiled(dq, live && !own), flags, wave, lane)) {
      BadSums<false> seen;
      clear(dq);
      for (int j = 0; j < st.n; ++j) {
        fetch(j, C<0>{});
        wait_vmem_all();
        __syncthreads();
        take_out<L, false, kBN, 256, true>(kbuf[0], bad, tid);
        __syncthreads();
        const uint64_t out = bad_rows(bad, lane);
#pragma unroll 1
        for (int u = 0; u < 2; ++u) {
          f32x16 s = scores_32<L>(kbuf[0] + u * 32 * 128, qf, k_rd);
          const f32x16 dp = scores_32<L>(vbuf[0] + u * 32 * 128, df, k_rd);
          const int key0 = st.key0(j) + 32 * u + 4 * g, low = j < st.n_first ? 1 << 30 : lo;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int at = key0 + 8 * (r >> 2) + (r & 3);
            s[r] = fast_exp2(fmaf(s[r], a.sl2, -l2)) * (dp[r] - delta);
            if (!((at >= low && at <= hi) || at < first)) s[r] = 0.f;
          }
          drop_rows(s, (uint32_t)(out >> 32 * u), g);
          product_32<L>(dq, kbuf[0] + u * 32 * 128, s, t_rd);
        }
        seen.add(bad, lane, [&](int i) {
          const int key = st.key0(j) + i;
          return (j >= st.n_first && key >= lo && key <= hi) || key < first;
        }, [](int) { return false; });
        __syncthreads();
      }
      if (own) seen.up = ~0ull;
      seen.put(dq);
    }
  }
  if (wq0 < a.Sq)
    store_columns(dq, a.scale, live, reinterpret_cast<uint8_t *>(&kbuf[0][0]) + wave * 8192,
                  a.dq + it.b * a.dqsb + it.h * a.dqsh + (int64_t)wq0 * a.dqss, a.dqss, a.Sq - wq0, lane);
}

// Backward, dK and dV: a workgroup sums one of them over 128 keys of one key head, a wave
// 32 of them as columns, and streams the queries that see them, of every head that
// shares the keys, in 64-row stages of Q and dO.  A key's queries are one interval of
// positions, so the sums run in a fixed order with no atomics.
//
// Both sums take the scores: 5 products for the 4 of one workgroup taking both.  But a
// wave's 192 registers of K, V and two sums leave nothing to read LDS ahead with (two
// waves per SIMD wait for every operand and spill: 2.7 ms at B=2 H=56/8 S=8192 with 1024
// keys to either side); alone on its SIMD it moves scores between register files for as
// long as it multiplies (3.5 ms); and waves of both kinds in one workgroup run their
// softmax at the same time (2.9 ms).  As it is: 1.7 to 1.8 ms there, 1.0 PFLOP/s of the five
// products, the rest being the tail of the grid (seven heads share a tile's keys, so an
// item is 238 stages and a place gets four or five of them) and the masked stages.
//
// The first keys are seen by every query, the others by a window's: tiles that hold
// first keys are cut into a.pieces equal runs of stages, which leave fp32 partial sums
// in a.part for window_dkdv_sum_kernel.  They come last in the grid, being short.  Where
// few tiles leave most of the chip idle (heads that share keys on a short sequence), the
// others are cut too, into a.rest_pieces.
constexpr int kQStage = 64;
struct DkdvLds {
  uint16_t q[2][kQStage * 128], dout[2][kQStage * 128];
  float stats[2][2][kQStage];  // lse (log2 units), delta
  BadValues<kQStage> bad;
  int flags[4];
};

// Where a piece's dK (which 0) or dV of 128 keys by 128 dims is in a.part: those of the first
// keys' tiles, then the others'.
__device__ __forceinline__ int64_t part_slot(const WindowArgs &a, int bh, int tile, int piece, int which) {
  const int64_t heads = (int64_t)a.B * a.Hkv, rest = a.nkt - a.first_tiles;
  const int64_t at = tile < a.first_tiles
                         ? ((int64_t)bh * a.first_tiles + tile) * a.pieces + piece
                         : heads * a.first_tiles * a.pieces + (bh * rest + tile - a.first_tiles) * a.rest_pieces + piece;
  return (at * 2 + which) * (kRows * 128);
}

template <bool kDk>
__device__ __forceinline__ void window_key_sums(const WindowArgs &a, const Item &it, int piece, int pieces, DkdvLds &lds) {
  using L = DualLayout;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Span sp = span_of(a, it.b);
  const int j0 = it.tile * kRows, wj0 = j0 + 32 * wave, key = wj0 + l32;
  const int j1 = (j0 + kRows < sp.len ? j0 + kRows : sp.len) - 1;

  f32x16 acc[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) acc[dt] = f32x16{0.f};
  // Rows [i_a, i_b) see some key of the tile.
  int i_a = sp.i_lo, i_b = sp.i_hi;
  if (j0 >= a.sinks) {
    i_a = j0 - a.right - sp.qs > i_a ? j0 - a.right - sp.qs : i_a;
    i_b = j1 + a.left + 1 - sp.qs < i_b ? j1 + a.left + 1 - sp.qs : i_b;
  } else if (a.causal) {
    i_a = j0 - sp.qs > i_a ? j0 - sp.qs : i_a;
  }
  // Stages t_a .. t_a + n - 1 are this piece's: kQStage rows of a head, head after head.
  const int per_head = j1 >= j0 && i_b > i_a ? (i_b - i_a + kQStage - 1) / kQStage : 0;
  const int64_t stages = (int64_t)per_head * a.rep;
  const int64_t t_a = stages * piece / pieces;
  const int n = (int)(stages * (piece + 1) / pieces - t_a);
  if (n > 0) {
    // Positions plo .. plo + span see the lane's key.
    int plo = key - a.right;
    uint32_t span = (uint32_t)(a.left + a.right);
    if (key < a.sinks) {
      plo = a.causal ? key : -(1 << 30);
      span = 0x7fffffffu;
    }
    if (key >= sp.len) plo = 1 << 30, span = 0;
    TileDma<4, L, false, kQStage> qdma, ddma;
    qdma.init(a.qss, wave, lane);
    ddma.init(a.gss, wave, lane);
    int fh = it.h * a.rep + (int)(t_a / per_head), frow = i_a + (int)(t_a % per_head) * kQStage;
    int crow = frow;  // rows of the stage that is computed
    auto fetch = [&](auto par) __attribute__((always_inline)) {
      constexpr int slot = decltype(par)::value;
      fetch_tile(qdma, a.q + it.b * a.qsb + fh * a.qsh, a.qss, frow, i_b, lds.q[slot]);
      fetch_tile(ddma, a.dout + it.b * a.gsb + fh * a.gsh, a.gss, frow, i_b, lds.dout[slot]);
      // Rows past i_b are zeros throughout: p = 1, but dO = dP = delta = 0.
      if (wave < (kDk ? 2 : 1)) {
        const int rows = i_b - frow < kQStage ? i_b - frow : kQStage;
        const float *st = a.stats + wave * a.stats_n + ((int64_t)it.b * a.H + fh) * a.Sq + frow;
        buffer_load_lds_b32(range_desc(st, rows * 4), 4 * lane, lds_address(lds.stats[slot][wave]));
      }
      frow += kQStage;
      if (frow >= i_b) {
        frow = i_a;
        ++fh;
      }
    };
    fetch(C<0>{});
    u32x4 kf[8], vf[8];
    load_columns(kf, a.k + it.b * a.ksb + it.h * a.ksh, a.kss, key, sp.len, g);
    if constexpr (kDk) load_columns(vf, a.v + it.b * a.vsb + it.h * a.vsh, a.vss, key, sp.len, g);
    const int k_rd = L::k_base(l32, g), t_rd = L::v_base(lane);
    const bool keys_whole = wj0 + 31 < sp.len;
    // What the wave's keys are to rows at positions p0 .. p0 + 63 (those past i_b give
    // nothing whatever p is).
    auto cover = [&](int p0) __attribute__((always_inline)) -> Cover {
      const int p1 = p0 + kQStage - 1;
      if (wj0 >= sp.len) return kNone;
      if (wj0 < a.sinks) {
        if (a.causal && p1 < wj0) return kNone;
        if (wj0 + 31 < a.sinks) return keys_whole && (!a.causal || p0 >= wj0 + 31) ? kAll : kPart;
      } else if (p1 < wj0 - a.right || p0 > wj0 + 31 + a.left) {
        return kNone;
      }
      return keys_whole && p0 >= wj0 + 31 - a.right && p1 <= (wj0 < a.sinks ? a.sinks : wj0) + a.left ? kAll : kPart;
    };
    // Statistic `which` of the rows of accumulator registers 4*r4 .. 4*r4+3 of half u.
    auto row_stats = [&](int slot, int which, int u, int r4, float(&x)[4]) __attribute__((always_inline)) {
      const float4 v = *(const float4 *)&lds.stats[slot][which][32 * u + 8 * r4 + 4 * g];
      x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    };
    wait_vmem_all();
    __syncthreads();
    two_buffers(n, [&](auto par, int j) __attribute__((always_inline)) {
      constexpr int slot = decltype(par)::value;
      const int p0 = sp.qs + crow;
      crow += kQStage;
      if (crow >= i_b) crow = i_a;
      if (j + 1 < n) fetch(C<slot ^ 1>{});
      const Cover c = cover(p0);
      // Half u's scores -> p, or (dK) ds; 0 where the row does not see the key.
      auto weigh = [&](int u, f32x16 &s, const f32x16 *dp) __attribute__((always_inline)) {
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          float l2[4], de[4];
          row_stats(slot, 0, u, r4, l2);
          if (kDk) row_stats(slot, 1, u, r4, de);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float p = fast_exp2(fmaf(s[4 * r4 + r], a.sl2, -l2[r]));
            s[4 * r4 + r] = kDk ? p * ((*dp)[4 * r4 + r] - de[r]) : p;
          }
        }
        if (c == kPart) {
          const uint32_t ahead = (uint32_t)(p0 + 32 * u + 4 * g - plo);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (ahead + 8 * (r >> 2) + (r & 3) > span) s[r] = 0.f;
        }
      };
      if (c != kNone) {
        if constexpr (kDk) {
          stage_pair<L>(lds.q[slot], lds.dout[slot], kf, vf, k_rd, t_rd, acc,
                        [&](int u, f32x16 &s, const f32x16 &dp, u32x4(&f)[2]) __attribute__((always_inline)) {
                          weigh(u, s, &dp);
                          const f32x16 ds[1] = {s};
                          pack_p<1>(ds, f);
                        });
        } else {
          stage_single<L, L>(lds.q[slot], lds.dout[slot], kf, k_rd, t_rd, acc,
                             [&](f32x16(&s)[2], u32x4(&f)[4]) __attribute__((always_inline)) {
                               weigh(0, s[0], nullptr);
                               weigh(1, s[1], nullptr);
                               pack_p<2>(s, f);
                             });
        }
      }
      wait_vmem_all();
      __syncthreads();
    });
    // For dK, rows of Q that are not finite are taken out whole, with weight 0 (as keys are in
    // window_dq_kernel): such a row's lse is NaN, and with it every sum of a key that it sees,
    // or -inf, and its weights are 0.
    if (any_wave(spoiled(acc, key < sp.len), lds.flags, wave, lane)) {
      BadSums<!kDk> seen;
      clear(acc);
      fh = it.h * a.rep + (int)(t_a / per_head), frow = i_a + (int)(t_a % per_head) * kQStage;
      for (int j = 0; j < n; ++j) {
        const int p0 = sp.qs + frow, rows = i_b - frow;
        fetch(C<0>{});
        wait_vmem_all();
        __syncthreads();
        take_out<L, false, kQStage, 256, kDk>(kDk ? lds.q[0] : lds.dout[0], lds.bad, tid);
        __syncthreads();
        const uint64_t out = kDk ? bad_rows(lds.bad, lane) : 0;
#pragma unroll 1
        for (int u = 0; u < 2; ++u) {
          f32x16 s = scores_32<L>(lds.q[0] + u * 32 * 128, kf, k_rd), dp = {0.f};
          if constexpr (kDk) dp = scores_32<L>(lds.dout[0] + u * 32 * 128, vf, k_rd);
          const uint32_t ahead = (uint32_t)(p0 + 32 * u + 4 * g - plo);
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int at = 32 * u + 8 * (r >> 2) + 4 * g + (r & 3);
            const float p = fast_exp2(fmaf(s[r], a.sl2, -lds.stats[0][0][at]));
            s[r] = kDk ? p * (dp[r] - lds.stats[0][1][at]) : p;
            // (Rows past i_b are zeros, but 0 times an infinity of the key's is not.)
            if (ahead + 8 * (r >> 2) + (r & 3) > span || at >= rows) s[r] = 0.f;
          }
          if (kDk) drop_rows(s, (uint32_t)(out >> 32 * u), g);
          product_32<L>(acc, (kDk ? lds.q[0] : lds.dout[0]) + u * 32 * 128, s, t_rd);
        }
        seen.add(lds.bad, lane, [&](int i) { return (uint32_t)(p0 + i - plo) <= span; }, [&](int i) {
          const float l2 = lds.stats[0][0][i];
          return kDk && (l2 != l2 || !finite(lds.stats[0][1][i]));
        });
        __syncthreads();
      }
      seen.put(acc);
    }
  }
  if (pieces > 1) {
    float *p = a.part + part_slot(a, it.b * a.Hkv + it.h, it.tile, piece, kDk ? 0 : 1) + (32 * wave + l32) * 128 + 4 * g;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int rr = 0; rr < 4; ++rr)
        *(float4 *)(p + dt * 32 + 8 * rr) =
            key < sp.len ? float4{acc[dt][4 * rr], acc[dt][4 * rr + 1], acc[dt][4 * rr + 2], acc[dt][4 * rr + 3]}
                         : float4{0.f, 0.f, 0.f, 0.f};
  } else if (wj0 < a.Skv) {
    uint8_t *tile = reinterpret_cast<uint8_t *>(&lds.q[0][0]) + wave * 8192;
    uint16_t *out = kDk ? a.dk + it.b * a.dksb + it.h * a.dksh + (int64_t)wj0 * a.dkss
                        : a.dv + it.b * a.dvsb + it.h * a.dvsh + (int64_t)wj0 * a.dvss;
    store_columns(acc, kDk ? a.scale : 1.f, key < sp.len, tile, out, kDk ? a.dkss : a.dvss, a.Skv - wj0, lane);
  }
}

__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) window_dkdv_kernel(WindowArgs a) {
  __shared__ __attribute__((aligned(16))) DkdvLds lds;
  // The grid: the window's tiles, then the first keys'; each run of tiles once for dK and then
  // for dV, which read the same rows.
  int i = (int)blockIdx.x;
  const bool whole = i < 2 * a.grid_whole;
  if (!whole) i -= 2 * a.grid_whole;
  const int chunk = whole ? a.chunk : a.chunk_pieces, k = i >> 3;
  const bool dv = (k / chunk) & 1;
  i = ((k / (2 * chunk) * chunk + k % chunk) << 3) | (i & 7);  // without the dK, dV pairing
  const int pieces = whole ? a.rest_pieces : a.pieces;
  Item it = item_of(a, i, chunk, (whole ? a.nkt - a.first_tiles : a.first_tiles) * pieces, a.Hkv);
  if (it.tile < 0) return;
  const int piece = it.tile % pieces;
  it.tile = it.tile / pieces + (whole ? a.first_tiles : 0);
  if (dv) window_key_sums<false>(a, it, piece, pieces, lds);
  else window_key_sums<true>(a, it, piece, pieces, lds);
}

// dK and dV of the tiles that were cut: the pieces' partial sums in order.  A thread
// takes 4 dims of a key.
__global__ void __launch_bounds__(256) window_dkdv_sum_kernel(WindowArgs a) {
  const int rows = (a.rest_pieces > 1 ? a.nkt : a.first_tiles) * kRows, d = 4 * (threadIdx.x & 31);
  const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);  // ((b, h), dk or dv, key)
  const int key = (int)(item % rows), which = (int)(item / rows & 1);
  const int64_t bh = item / rows / 2;
  if (key >= a.Skv || bh >= (int64_t)a.B * a.Hkv) return;
  const int b = (int)(bh / a.Hkv), h = (int)(bh % a.Hkv);
  const int tile = key / kRows, pieces = tile < a.first_tiles ? a.pieces : a.rest_pieces;
  const float *p = a.part + part_slot(a, (int)bh, tile, 0, which) + (key % kRows) * 128 + d;
  float4 sum = *(const float4 *)p;
  for (int i = 1; i < pieces; ++i) {
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
// longer than a window tile's, or than a quarter of what one of the chip's 512 places for
// workgroups has to do in all, if that is more (it also bounds the partial sums: 1024
// runs of 128 KB and one more per tile, and fewer than 1024 tiles are cut: 256 MB).  In stages of one query head.  Then, if the tiles' dK and dV
// fill less than half of the places, all of them may be cut into more runs, of four stages
// at least: the join costs about four stages, and ten if 512 runs leave partial sums
// (H=8/1 S=1568, 119 and 26 keys to the sides: 82 us in 26 workgroups, 27 with the join).
static void plan_dkdv(WindowArgs &a) {
  a.nkt = (a.Skv + kRows - 1) / kRows;
  a.first_tiles = (a.sinks + kRows - 1) / kRows;
  const int64_t all_rows = (a.Sq + kQStage - 1) / kQStage, heads = (int64_t)a.B * a.Hkv;
  int64_t run = ((int64_t)kRows + a.left + a.right + kQStage - 1) / kQStage;
  if (run > all_rows) run = all_rows;
  const int64_t share = 2 * heads * (a.first_tiles * all_rows + (a.nkt - a.first_tiles) * run) / (4 * 512);
  if (run < share) run = share;
  a.pieces = (int)((all_rows + run - 1) / run);
  if (a.first_tiles == 0 || a.pieces == 1) {
    a.first_tiles = 0;
    a.pieces = 1;
  }
  const int64_t items = 2 * heads * ((int64_t)a.first_tiles * a.pieces + a.nkt - a.first_tiles);
  int64_t best = run * a.rep;
  a.rest_pieces = 1;
  for (int64_t p = 2; p * items <= 512 && p * 4 <= run * a.rep; ++p) {
    const int64_t cost = (run * a.rep + p - 1) / p + 4 + 10 * items * p / 512;
    if (cost < best) {
      best = cost;
      a.rest_pieces = (int)p;
    }
  }
  a.pieces *= a.rest_pieces;
}

// Rows of each of the two statistics, padded to 256 bytes.
static size_t stat_rows(const WindowArgs &a) { return ((size_t)a.B * a.H * a.Sq + 63) / 64 * 64; }

size_t window_bwd_bytes(WindowArgs a) {
  plan_dkdv(a);
  const size_t cut = (size_t)a.first_tiles * a.pieces +
                     (a.rest_pieces > 1 ? (size_t)(a.nkt - a.first_tiles) * a.rest_pieces : 0);
  return (2 * stat_rows(a) + (size_t)a.B * a.Hkv * cut * 2 * kRows * 128) * sizeof(float);
}

// Grid of `tiles` work items for each of a batch's `heads` heads (item_of).  Runs are as long
// as they can be, up to 64 tiles, with a multiple of 8 to a sequence where the number of a
// head's tiles allows it: neighbours share more of
// what they read in an XCD's L2, and every XCD gets as many (dK and dV, against runs of a
// 128th of all tiles: 2.29 -> 2.01 ms at B=2 H=56/8 S=8192, 122 -> 111 us at H=14 S=4104;
// forward, runs of 16 tiles against 64: 10.0 -> 9.2 ms at H=56 S=42120).  Where sequences may
// end early, runs that are a part of a head may be empty, so there are at least `ragged_runs`.
static int deal(const WindowArgs &a, int tiles, int heads, int ragged_runs, int *chunk) {
  *chunk = 1;
  if (tiles == 0) return 0;
  int per_head = (tiles + 63) / 64;
  while (per_head < tiles && (int64_t)heads * per_head % 8) ++per_head;
  if (a.kv_lens && per_head > 1)
    while (per_head < tiles && ((int64_t)heads * per_head % 8 || (int64_t)a.B * heads * per_head < ragged_runs)) ++per_head;
  *chunk = (tiles + per_head - 1) / per_head;  // a head's runs alike
  const int64_t runs = (int64_t)a.B * heads * ((tiles + *chunk - 1) / *chunk);
  return (int)((runs + 7) / 8 * 8 * *chunk);
}

// Query rows up to which splitting the keys is weighed against the tiles.
constexpr int kTokenMaxRows = 8192;

// Whether the keys are split, and into how many workgroups per 32 rows.  In units of a
// token workgroup's step (four waves' stages of 32 keys, about 2 us of its CU): a round of
// workgroups costs three steps beside its own, the merge four, and a 64-key stage of the
// tiles 0.7 (two workgroups to a CU).
static bool plan_token(WindowArgs &a, int cus) {
  if (a.Sq > kTokenMaxRows) return false;
  const int per_head = (a.Sq + kTokenRows - 1) / kTokenRows;
  a.nqt = a.Sq >= kTokenRows ? a.rep * per_head : (a.rep * a.Sq + kTokenRows - 1) / kTokenRows;
  const int64_t units = (int64_t)a.B * a.Hkv * a.nqt;
  auto keys_of = [&](int rows) -> int64_t {  // of a workgroup with so many rows
    const int64_t n = (int64_t)a.left + a.right + a.sinks + (rows < a.Sq ? rows : a.Sq);
    return n < a.Skv ? n : a.Skv;
  };
  const int64_t steps = (keys_of(kTokenRows) + 4 * kTokenStage - 1) / (4 * kTokenStage);
  const int64_t tiles = (int64_t)a.B * a.H * ((a.Sq + kRows - 1) / kRows);
  int64_t best = (tiles + 2 * cus - 1) / (2 * cus) * ((keys_of(kRows) + kBN - 1) / kBN) * 7 / 10 + 3;
  a.pieces = 0;
  for (int p = 1; p <= kTokenPieces && p <= steps; ++p) {
    const int64_t rounds = (units * p + cus - 1) / cus;
    const int64_t cost = rounds * ((steps + p - 1) / p + 3) + (p > 1 ? 4 : 0);
    if (cost < best || (p == 1 && a.Sq == 1)) {  // (a lone row never takes a tile)
      best = cost;
      a.pieces = p;
    }
  }
  return a.pieces > 0;
}

static int cu_count(int *cus) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || *cus <= 0)
    return fail(H3A_ERR_HIP, "device query failed");
  return H3A_OK;
}

int plan_window_fwd(WindowArgs &a, bool *split, size_t *bytes) {
  *split = false;
  *bytes = 0;
  if (a.Sq > kTokenMaxRows) return H3A_OK;
  int cus = 0;
  const int rc = cu_count(&cus);
  if (rc) return rc;
  *split = plan_token(a, cus);
  if (*split && a.pieces > 1) *bytes = (size_t)a.B * a.Hkv * a.nqt * a.pieces * kTokenRows * (128 + 2) * sizeof(float);
  return H3A_OK;
}

int launch_window_fwd(WindowArgs a, bool split, void *ws, hipStream_t s) {
  if (!split) {
    a.nqt = (a.Sq + kRows - 1) / kRows;
    const int grid = deal(a, a.nqt, a.H, 256, &a.chunk);
    hipLaunchKernelGGL(window_fwd_kernel, dim3((unsigned)grid), dim3(256), 0, s, a);
    return check_launch("window_fwd_kernel");
  }
  a.part = static_cast<float *>(ws);
  const int units = a.B * a.Hkv * a.nqt;
  hipLaunchKernelGGL(window_token_kernel, dim3((unsigned)(units * a.pieces)), dim3(256), 0, s, a);
  const int rc = check_launch("window_token_kernel");
  if (rc || a.pieces == 1) return rc;
  hipLaunchKernelGGL(window_token_sum_kernel, dim3((unsigned)(units * kTokenRows)), dim3(256), 0, s, a, units);
  return check_launch("window_token_sum_kernel");
}

int launch_window_bwd(WindowArgs a, void *ws, hipStream_t s) {
  a.stats = static_cast<float *>(ws);
  a.stats_n = (int64_t)stat_rows(a);
  a.nqt = (a.Sq + kRows - 1) / kRows;
  const int grid = deal(a, a.nqt, a.H, 256, &a.chunk);
  hipLaunchKernelGGL(window_dq_kernel, dim3((unsigned)grid), dim3(256), 0, s, a);
  int rc = check_launch("window_dq_kernel");
  if (rc) return rc;
  plan_dkdv(a);
  a.part = a.stats + 2 * a.stats_n;
  a.grid_whole = deal(a, (a.nkt - a.first_tiles) * a.rest_pieces, a.Hkv, 128, &a.chunk);
  a.grid_pieces = deal(a, a.first_tiles * a.pieces, a.Hkv, 128, &a.chunk_pieces);
  hipLaunchKernelGGL(window_dkdv_kernel, dim3((unsigned)(2 * a.grid_whole + 2 * a.grid_pieces)), dim3(256), 0, s, a);
  rc = check_launch("window_dkdv_kernel");
  if (rc || (a.first_tiles == 0 && a.rest_pieces == 1)) return rc;
  const int64_t rows = (int64_t)a.B * a.Hkv * (a.rest_pieces > 1 ? a.nkt : a.first_tiles) * kRows * 2;
  hipLaunchKernelGGL(window_dkdv_sum_kernel, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, s, a);
  return check_launch("window_dkdv_sum_kernel");
}

}  // namespace h3a
