// Tiles of the attention kernels at head_dim 128: how a 64-key K or V stage lies
// in LDS and gets there, the score and PV products over it and the online
// softmax between them.  Device code shared by the dense, block-sparse and
// windowed kernels.
#pragma once

#include <type_traits>

#include "h3a_device.h"
#include "h3a_stale.h"

namespace h3a {

constexpr int kD = 128;
constexpr int kBN = 64;               // keys per pipeline stage
constexpr float kRescaleSlack = 8.f;  // log2 headroom before the running max is refreshed

// ---------------------------------------------------------------------------
// LDS layout of a 64-key K or V stage: the row pitch, which 16-byte global
// chunk each 16-byte LDS slot holds, and how the MFMA operand reads address
// the stage.  Bank-conflict free for the reads below (SQ_LDS_BANK_CONFLICT = 0
// measured).  The kernels take the layout as a template parameter L.
//
// SwzLayout: 256-byte rows; chunk c of row r sits in slot c ^ swz(r).
//   K: swz(r) = r & 15.  A 128-bit read of one chunk by 16 consecutive rows
//      (the A operand of the score MFMA) hits 16 distinct bank groups.
//   V: swz(r) = 4 * (r & 3).  A transpose read by 32 lanes covers 4 rows x
//      4 chunks, which land on 16 distinct bank groups: all 64 banks once.
//   Read offsets are base ^ const, held per lane.
struct SwzLayout {
  static constexpr int kKRow = 256, kVRow = 256;  // bytes
  static constexpr int kKSlots = 16, kVSlots = 16;
  __device__ __forceinline__ static int k_chunk(int r, int slot) { return slot ^ (r & 15); }
  __device__ __forceinline__ static int v_chunk(int r, int slot) { return slot ^ (4 * (r & 3)); }
  // Lane's A-operand chunk of k-step 0 (row l32, chunk g); k-step ks reads
  // chunk 2*ks + g, i.e. offset k_base ^ (32*ks).
  __device__ __forceinline__ static int k_base(int l32, int g) {
    return l32 * kKRow + 32 * ((l32 >> 1) & 7) + 16 * (g ^ (l32 & 1));
  }
  __device__ __forceinline__ static int k_off(int kb, int ks) { return kb ^ (32 * ks); }
  // Column block dt of the transpose reads is chunk 4*dt + c of the row,
  // stored in slot (4*dt + c) ^ 4*(row & 3): offset v_base ^ (64*dt).
  __device__ __forceinline__ static int v_base(int lane) {
    const int i = (lane & 15) >> 2;
    const int row = 4 * (lane >> 5) + i;
    const int c = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    return row * kVRow + 64 * i + 16 * c + 8 * (lane & 1);
  }
  __device__ __forceinline__ static int v_off(int vb, int dt) { return vb ^ (64 * dt); }
};

template <class L, int ROWS = kBN>
struct StageBytes {
  static constexpr int kK = ROWS * L::kKRow;
  static constexpr int kV = ROWS * L::kVRow;
};

// Global -> LDS staging of one ROWS-key K or V stage by LDS DMA.  Instruction
// t fills the 64 consecutive 16-byte slots 64t..64t+63 of the stage (1 KiB);
// each lane fetches the global chunk that its slot holds under the layout.
// The NW waves of the stream issue instructions t = wave, wave+NW, ...  The
// buffer resource is rebased on the stage's first key and covers exactly its
// valid rows, so rows >= Skv arrive as zeros (masked keys never carry
// NaN/Inf) and the per-lane offsets are loop-invariant.
template <int NW, class L, bool kIsV, int ROWS = kBN>
struct TileDma {
  static constexpr int kWaves = NW;
  static constexpr int kSlots = kIsV ? L::kVSlots : L::kKSlots;  // per row
  static constexpr int kInstTotal = ROWS * kSlots / 64;           // 64 lanes per instruction
  static constexpr int kInst = (kInstTotal + NW - 1) / NW;        // per wave (the last may be idle)
  static_assert(ROWS * kSlots % 64 == 0, "a stage is a whole number of DMA instructions");
  // With 16-slot rows and NW a multiple of 4, instruction i covers rows
  // 4*(wave + i*NW) + lane/16: the swizzle (row & 15 or row & 3) does not
  // depend on i, so the offsets are off[0] + i * 4*NW rows and one register
  // holds them all.
  static constexpr bool kAffine = kSlots == 16 && NW % 4 == 0;
  uint32_t off[kAffine ? 1 : kInst];
  uint32_t step;  // bytes between instructions when kAffine (wave-uniform)
  int wave;       // wave-uniform

  __device__ __forceinline__ void init(int64_t ss, int wave_uniform, int lane) {
    wave = wave_uniform;
    step = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(4 * NW * ss * 2));
#pragma unroll
    for (int i = 0; i < (kAffine ? 1 : kInst); ++i) {
      const int slot = 64 * (wave + i * NW) + lane;
      const int row = slot / kSlots, sl = slot % kSlots;
      const int chunk = kIsV ? L::v_chunk(row, sl) : L::k_chunk(row, sl);
      off[i] = (uint32_t)(((int64_t)(row < ROWS ? row : ROWS - 1) * ss + chunk * 8) * 2);
    }
  }
  // Offsets of instructions 0, 1, ... in issue order: `cur` starts at
  // first() and next() moves it on.  The add is opaque to the compiler, which
  // would otherwise hoist all kInst offsets out of the stage loop and keep
  // them in registers.  Without kAffine the cursor is the byte offset added
  // to every instruction's own offset (the stage's, for a descriptor of the
  // whole (b,h) slice).
  __device__ __forceinline__ uint32_t first() const { return kAffine ? off[0] : 0u; }
  __device__ __forceinline__ uint32_t next(uint32_t cur) const {
    if constexpr (kAffine) {
      uint32_t r;
      asm volatile("v_add_u32 %0, %1, %2" : "=v"(r) : "v"(cur), "s"(step));
      return r;
    } else {
      return cur;
    }
  }
  // Buffer descriptor of the stage that starts at key0 (valid rows only).
  __device__ __forceinline__ u32x4 desc(const uint16_t *base, int64_t ss, int key0, int Skv) const {
    const int rows = Skv - key0 >= ROWS ? ROWS : (Skv > key0 ? Skv - key0 : 0);
    return stage_desc(stage_ptr(base, key0, ss), ss, rows);
  }
  // Instruction i (0 <= i < kInst, a compile-time index) of this wave's
  // share; `cur` is its offset cursor (first(), then next() once per
  // instruction) and m0 the LDS address of its 1 KiB: that of instruction
  // 0, lds_address(tile) + 1024 * wave, plus 1024 * NW per instruction,
  // advanced by opaque_sadd so that the compiler does not keep every
  // instruction's address of both buffers live in SGPRs.
  __device__ __forceinline__ void issue_one(u32x4 d, int i, uint32_t cur, uint32_t m0) const {
    if (kInstTotal % NW == 0 || wave + i * NW < kInstTotal)
      buffer_load_lds_b128(d, kAffine ? cur : off[i] + cur, m0);
  }
  __device__ __forceinline__ void issue(const uint16_t *base, int64_t ss, int key0, int Skv,
                                        uint16_t *tile) const {
    issue_range<0, kInst>(base, ss, key0, Skv, tile);
  }
  // Instructions I0 .. I1-1 of this wave's share.
  template <int I0, int I1>
  __device__ __forceinline__ void issue_range(const uint16_t *base, int64_t ss, int key0, int Skv,
                                              uint16_t *tile) const {
    if constexpr (I1 > I0) issue_desc<I0, I1>(desc(base, ss, key0, Skv), tile);
  }
  // The same with the stage's descriptor given (StageCursor::desc).
  template <int I0, int I1>
  __device__ __forceinline__ void issue_desc(u32x4 d, uint16_t *tile) const {
    issue_desc_off<I0, I1>(d, tile, 0u);
  }
  // The same with a descriptor of the whole (b,h) slice and the stage's byte
  // offset in it, soff, added to every lane's offset (one v_add).
  template <int I0, int I1>
  __device__ __forceinline__ void issue_desc_off(u32x4 d, uint16_t *tile, uint32_t soff) const {
    if constexpr (I1 > I0) {
      uint32_t cur = first() + soff;
#pragma unroll
      for (int i = 0; i < I0; ++i) cur = next(cur);
      uint32_t m0 = lds_address(tile) + (uint32_t)(wave + I0 * NW) * 1024u;
#pragma unroll
      for (int i = I0; i < I1; ++i) {
        issue_one(d, i, cur, m0);
        if (i + 1 < I1) {
          cur = next(cur);
          m0 = opaque_sadd<1024u * NW>(m0);
        }
      }
    }
  }
  // Common staging interface: start() at the top of a stage, finish() at its
  // end; kAsync stagers need a vmcnt wait before the stage's barrier.
  static constexpr bool kAsync = true;
  __device__ __forceinline__ void start(const uint16_t *base, int64_t ss, int key0, int Skv,
                                        uint16_t *tile) {
    issue(base, ss, key0, Skv, tile);
  }
  __device__ __forceinline__ void finish(uint16_t *) const {}
};

// One wave's share of a stage's TileDma fetch issued one instruction at a
// time (issue_desc taken apart), to spread it over a matrix cluster.
template <class Dma>
struct DmaSeq {
  static constexpr int kCount = Dma::kInst;
  const Dma &dma;
  u32x4 d;
  uint32_t cur, m0;
  int i;
  // soff: the stage's byte offset when d describes the whole (b,h) slice.
  __device__ __forceinline__ DmaSeq(const Dma &dma_, u32x4 d_, uint16_t *tile, uint32_t soff)
      : dma(dma_), d(d_), cur(dma_.first() + soff), m0(lds_address(tile) + (uint32_t)dma_.wave * 1024u), i(0) {}
  __device__ __forceinline__ void issue() {
    dma.issue_one(d, i, cur, m0);
    ++i;
    if (i < Dma::kInst) {
      cur = dma.next(cur);
      m0 = opaque_sadd<1024u * Dma::kWaves>(m0);
    }
  }
};

// Wave-uniform position of a K or V stream in a contiguous range of key
// stages: the byte address of the next stage's first row and the number of
// valid rows from there on (it goes negative past the range's end, where the
// descriptor covers nothing and the DMA writes zeros).  advance() moves on by
// one stage with one opaque 64-bit scalar add; rebuilding the address as
// base + key0 * stride every stage costs a 64-bit multiply chain on the
// scalar unit in the middle of the issuing wave's DMA burst.
template <int ROWS>
struct StageCursor {
  uint32_t lo, hi, step_lo, step_hi, ss2;
  int rows_left;
  __device__ __forceinline__ void init(const uint16_t *base, int64_t ss, int key0, int key_end) {
    const uint64_t addr = reinterpret_cast<uint64_t>(base) + (uint64_t)((int64_t)key0 * ss * 2);
    const uint64_t step = (uint64_t)((int64_t)ROWS * ss * 2);
    lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)addr);
    hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(addr >> 32));
    step_lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)step);
    step_hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(step >> 32));
    ss2 = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(ss * 2));
    rows_left = __builtin_amdgcn_readfirstlane(key_end - key0);
    asm volatile("s_nop 4" : "+s"(lo), "+s"(hi), "+s"(ss2), "+s"(rows_left));  // as settled()
  }
  // The V# of the current stage, as stage_desc builds it: valid rows only.
  __device__ __forceinline__ u32x4 desc() const {
    const int rows = rows_left >= ROWS ? ROWS : (rows_left > 0 ? rows_left : 0);
    const uint32_t bytes = rows > 0 ? (uint32_t)(rows - 1) * ss2 + 256u : 0u;
    return u32x4{lo, hi & 0xffffu, bytes, (uint32_t)kBufferConfig};
  }
  __device__ __forceinline__ void advance() {
    asm volatile("s_add_u32 %0, %0, %2\n\ts_addc_u32 %1, %1, %3"
                 : "+s"(lo), "+s"(hi)
                 : "s"(step_lo), "s"(step_hi)
                 : "scc");
    rows_left -= ROWS;
  }
};

// A stage's scores live in NSUB accumulators of 32 keys: s[u] holds keys
// 32u..32u+31 of the stage.  In the S^T accumulator layout lane l owns query
// l%32; register r of s[u] holds key 32u + 8*(r/4) + 4*(l/32) + r%4.

// score_tile calls hook(k-step) after each k-step's MFMAs and pv_tile
// hook(4 * key step + dim tile) after each MFMA (by default nothing): where a
// matrix cluster's LDS DMA instructions go when they are spread over it.
struct NoHook {
  __device__ __forceinline__ void operator()(int) const {}
};

// S^T (32*NSUB keys x 32 queries of this wave) = K_stage Q^T.
template <class L, int NSUB, class Hook = NoHook>
__device__ __forceinline__ void score_tile(const uint16_t *kbuf, const u32x4 (&qf)[8], int k_rd,
                                           f32x16 (&s)[NSUB], Hook hook = Hook{}) {
#pragma unroll
  for (int u = 0; u < NSUB; ++u) s[u] = f32x16{0.f};
  const char *kb = reinterpret_cast<const char *>(kbuf);
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) {
    const char *p = kb + L::k_off(k_rd, ks);
#pragma unroll
    for (int u = 0; u < NSUB; ++u) {
      const u32x4 a = *(const u32x4 *)(p + 32 * u * L::kKRow);
      s[u] = mfma_32x32x16(a, qf[ks], s[u]);
    }
    hook(ks);
  }
}

// P^T fragments for the 2*NSUB sixteen-key steps, straight from the S^T
// registers.  Step ks, k-slot (g = lane/32, e) carries key
// 16*ks + 8*(e/4) + 4*g + e%4.
template <int NSUB>
__device__ __forceinline__ void pack_p(const f32x16 (&s)[NSUB], u32x4 (&pf)[2 * NSUB]) {
#pragma unroll
  for (int u = 0; u < NSUB; ++u)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      pf[2 * u + h] = u32x4{pack_bf16x2(s[u][8 * h + 0], s[u][8 * h + 1]),
                            pack_bf16x2(s[u][8 * h + 2], s[u][8 * h + 3]),
                            pack_bf16x2(s[u][8 * h + 4], s[u][8 * h + 5]),
                            pack_bf16x2(s[u][8 * h + 6], s[u][8 * h + 7])};
}

// V transpose reads.  Within each 16-lane group a ds_read_b64_tr_b16 gives
// lane j element j%4 of the 4 consecutive bf16 that lanes 4k + j/4 address
// (k = 0..3).  Lane i of group t points at row 4*(t/2) + i/4 (+16*ks, +8 for
// k-slots 4..7) and columns 16*(t%2) + 4*(i%4) (+32*dt), so lane l receives
// V[key][32*dt + l%32] for the 4 keys of its k-slots, in the score
// accumulator's key order.  L::v_base / L::v_off place that in the layout.
// O^T (128 dims x 32 queries) += V^T_stage P^T over NKS sixteen-key steps.
template <class L, int NKS, class Hook = NoHook>
__device__ __forceinline__ void pv_tile(const uint16_t *vbuf, const u32x4 (&pf)[NKS], int v_rd,
                                        f32x16 (&o)[4], Hook hook = Hook{}) {
  const char *vb = reinterpret_cast<const char *>(vbuf);
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) {
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) {
      const char *p = vb + L::v_off(v_rd, dt) + 16 * ks * L::kVRow;
      const u32x2 lo = lds_read_tr16_b64(reinterpret_cast<const uint16_t *>(p));
      const u32x2 hi = lds_read_tr16_b64(reinterpret_cast<const uint16_t *>(p + 8 * L::kVRow));
      o[dt] = mfma_32x32x16(u32x4{lo.x, lo.y, hi.x, hi.y}, pf[ks], o[dt]);
      hook(4 * ks + dt);
    }
  }
}

// Max of N values as a tree of v_max3 (depth log3 N), not a dependent chain:
// the softmax cluster is latency-bound.
template <int N>
__device__ __forceinline__ float max_tree(const float (&v)[N]) {
  if constexpr (N == 1) {
    return v[0];
  } else if constexpr (N == 2) {
    return fmaxf(v[0], v[1]);
  } else {
    constexpr int M = (N + 2) / 3;
    float t[M];
#pragma unroll
    for (int i = 0; i < M; ++i) {
      if (3 * i + 2 < N)
        t[i] = fmaxf(fmaxf(v[3 * i], v[3 * i + 1]), v[3 * i + 2]);
      else if (3 * i + 1 < N)
        t[i] = fmaxf(v[3 * i], v[3 * i + 1]);
      else
        t[i] = v[3 * i];
    }
    return max_tree<M>(t);
  }
}

// Row max of a masked score stage (all sub-tiles, both lane halves), in
// scale*log2(e) units.
template <int NSUB>
__device__ __forceinline__ float tile_max(const f32x16 (&s)[NSUB], float sl2) {
  float v[16 * NSUB];
#pragma unroll
  for (int u = 0; u < NSUB; ++u)
#pragma unroll
    for (int r = 0; r < 16; ++r) v[16 * u + r] = s[u][r];
  return half_swap_max(max_tree<16 * NSUB>(v)) * sl2;
}

// This lane's share of the row sum of a stage's p values (a tree of adds).
template <int NSUB>
__device__ __forceinline__ float tile_sum(const f32x16 (&s)[NSUB]) {
  float a[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    a[r] = s[0][r];
    if constexpr (NSUB >= 2) a[r] += s[1][r];
    if constexpr (NSUB == 4) a[r] += s[2][r] + s[3][r];
  }
#pragma unroll
  for (int w = 8; w >= 1; w >>= 1)
#pragma unroll
    for (int r = 0; r < w; ++r) a[r] += a[r + w];
  return a[0];
}

// Keys >= Skv of the stage starting at key0 -> -inf (tail stage only).
template <int NSUB>
__device__ __forceinline__ void mask_tail(f32x16 (&s)[NSUB], int key0, int Skv, int g) {
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int kk = key0 + 8 * (r >> 2) + 4 * g + (r & 3);
#pragma unroll
    for (int u = 0; u < NSUB; ++u)
      if (kk + 32 * u >= Skv) s[u][r] = kNegInf;
  }
}

// ---------------------------------------------------------------------------
// Softmax of one score stage (32*NSUB keys), in place: S -> P (bf16 pairs in
// pf), the running max m and this lane's share of the row sum of the
// unrounded p.  m is refreshed lazily: only when some row of the wave exceeds
// it by more than kRescaleSlack (p then stays <= 2^kRescaleSlack), and O and l
// are rescaled only then.  VALU work only.
template <int NSUB>
__device__ __forceinline__ void softmax_stage(f32x16 (&s)[NSUB], int key0, int Skv, int g, float sl2,
                                              float &m, float &lsum, f32x16 (&o)[4],
                                              u32x4 (&pf)[2 * NSUB]) {
  if (key0 + 32 * NSUB > Skv) mask_tail<NSUB>(s, key0, Skv, g);
  const float mx = tile_max<NSUB>(s, sl2);
  if (__builtin_amdgcn_ballot_w64(mx > m + kRescaleSlack) != 0) {
    const float mnew = fmaxf(m, mx);
    const float alpha = fast_exp2(m - ((mnew == kNegInf) ? 0.f : mnew));
    m = mnew;
    lsum *= alpha;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) o[dt] *= alpha;
  }
  const float muse = (m == kNegInf) ? 0.f : m;
#pragma unroll
  for (int u = 0; u < NSUB; ++u)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[u][r] = fast_exp2(fmaf(s[u][r], sl2, -muse));
  pack_p<NSUB>(s, pf);
  lsum += tile_sum<NSUB>(s);
}

// Softmax of one score stage against the running reference m without
// computing the stage's row max.  p = 2^(s*sl2 - m) is formed, packed and
// summed straight away; only if some lane's stage sum exceeds kStaleSumLimit
// or is not finite (stage_sum_needs_refresh; +inf when a score ran 128 or
// more above m) does the wave take the row max, refresh m, rescale O and l
// and redo the stage.  m must be finite on entry (the first stage of a key
// range uses softmax_stage, which sets m to that stage's row max, so every
// later row sum is >= 1).  Every accepted p is then <= its stage sum <=
// 2^16 instead of <= 1: bf16 rounding of P and the fp32 sums are relative,
// so the normalised O is unchanged, and the bound on O that this leaves is
// given with kStaleSumLimit.
template <int NSUB>
__device__ __forceinline__ void exp_pack_sum(const f32x16 (&s)[NSUB], float sl2, float m,
                                             u32x4 (&pf)[2 * NSUB], float &ps) {
  float a[16];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int r = 8 * h + 2 * w;
      float p0[NSUB], p1[NSUB];
#pragma unroll
      for (int u = 0; u < NSUB; ++u) {
        p0[u] = fast_exp2(fmaf(s[u][r], sl2, -m));
        p1[u] = fast_exp2(fmaf(s[u][r + 1], sl2, -m));
        pf[2 * u + h][w] = pack_bf16x2(p0[u], p1[u]);
      }
      a[r] = p0[0];
      a[r + 1] = p1[0];
      if constexpr (NSUB >= 2) {
        a[r] += p0[1];
        a[r + 1] += p1[1];
      }
      if constexpr (NSUB == 4) {
        a[r] += p0[2] + p0[3];
        a[r + 1] += p1[2] + p1[3];
      }
    }
  }
#pragma unroll
  for (int w = 8; w >= 1; w >>= 1)
#pragma unroll
    for (int r = 0; r < w; ++r) a[r] += a[r + w];
  ps = a[0];
}

// kMaybeEmpty: m may still be -inf on entry (every earlier stage of the row
// was fully masked, as block-sparse rows can be).  p is then formed against 0
// and the stage always refreshes.
template <int NSUB, bool kMaybeEmpty = false>
__device__ __forceinline__ void softmax_stage_stale(f32x16 (&s)[NSUB], int key0, int Skv, int g, float sl2,
                                                    float &m, float &lsum, f32x16 (&o)[4],
                                                    u32x4 (&pf)[2 * NSUB]) {
  // Both branches are rare (a stage that reaches past Skv, a refresh).  With
  // 64-key waves they are marked so (kHint), and the common path falls
  // through instead of branching around their code in every stage (measured
  // +0.4 % dense, +0.5 % 128x128 sparse); the 32-key waves of the key-split
  // kernel lost 3 % with that layout.  (The hint has to sit in the branch
  // condition itself.)
  constexpr bool kHint = NSUB >= 2;
  const bool past = key0 + 32 * NSUB > Skv;
  if (kHint ? __builtin_expect(past, 0) : past) mask_tail<NSUB>(s, key0, Skv, g);
  float ps;
  exp_pack_sum<NSUB>(s, sl2, kMaybeEmpty && m == kNegInf ? 0.f : m, pf, ps);
  // Two ballots OR'd on the scalar unit: one ballot of the lane-wise OR
  // compiles to a mask -> 0/1 -> compare round trip through VALU.
  uint64_t need = __builtin_amdgcn_ballot_w64(stage_sum_needs_refresh(ps));
  if constexpr (kMaybeEmpty) need |= __builtin_amdgcn_ballot_w64(m == kNegInf);
  const bool refresh = need != 0;
  if (kHint ? __builtin_expect(refresh, 0) : refresh) {
    const float mnew = fmaxf(m, tile_max<NSUB>(s, sl2));
    const float alpha = fast_exp2(m - (kMaybeEmpty && mnew == kNegInf ? 0.f : mnew));
    m = mnew;
    lsum *= alpha;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) o[dt] *= alpha;
    exp_pack_sum<NSUB>(s, sl2, kMaybeEmpty && m == kNegInf ? 0.f : m, pf, ps);
  }
  lsum += ps;
}

}  // namespace h3a
