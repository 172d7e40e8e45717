// Softmax attention with grouped heads over packed sequences, forward and backward (cgamd.h:
// cg_packed_attention_*).  Per sequence and key head, with the G = heads / kv_heads query heads that share it:
//
//   S = scale Q K^T,  P = softmax(S) over the keys a row may see,  O = P V
//   delta_i = sum_d dO_id O_id,  dS = P o (dO V^T - delta),  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO
//
// ROWS.  A "row" is one (query token, shared head) pair, r = token * G + head: all G heads of a key head
// run through the same tiles, so K and V are staged once for all of them, a single new token fills G columns
// of a matrix instruction instead of one, and the sum over shared heads that dK and dV need is part of the
// contraction (no atomics, one fixed order).
//
// REGISTERS.  Everything is computed transposed with v_mfma_f32_32x32x16_bf16: S^T[key][row] = K Q^T puts one
// row into a lane (16 keys of it a lane half), so the running maximum and sum of the softmax are per-lane
// values plus one exchange between the halves, and P^T leaves the accumulator in the layout that the next
// product's second operand has, up to a permutation of the 16 keys of a step:
//   element e of lane half h  <->  key 16 ks + 4 h + (e & 3) + 8 (e >> 2)
// which the first operand matches by reading V transposed (ds_read_b64_tr_b16) at those keys.  P, dS and
// all the sums never touch LDS.  Statistics and accumulators are fp32; P and dS are rounded to bf16 on their
// way into the matrix instruction (at most half a step, 2^-8 relative, each; independent errors over the sum).
//
// LDS.  Tiles are copied by buffer_load ... lds (16 bytes a lane), two buffers: tile i + 1 is in flight while
// tile i is multiplied, one barrier a tile.  Rows keep their pitch of 2 DK or 2 DV bytes; instead of padding, the
// 16-byte chunks of a row are exchanged by an XOR with bits of the row number (mha_swz) so that both the
// b128 reads of K (32 rows, one chunk) and the transposed reads of V (8 rows, 4 chunks) spread over all banks.
// Rows behind the end of a sequence and columns behind D are outside the buffer descriptor and arrive as zeros.
//
// WHAT BOUNDS IT.  Forward at 64 wide heads the vector unit: a 32 x 32 tile of scores is 8 matrix instructions of 32 cycles
// beside 16 exponentials at a quarter of the rate and some 60 other vector instructions.  Counted over 64 x 4096 tokens,
// vector instructions are issued in 70 % of a SIMD's cycles and its matrix unit is busy in 45 %, at 1.76 of 2.4 GHz (on
// inputs of zeros the same code is 25 to 35 % faster: the clock follows the power).  Backward 65 and 58 % (dQ), 55 and
// 53 % (dK, dV); 128 wide forward 44 and 51 %.  A product of two 8192 x 8192 matrices reaches 1.38 to 1.48 PFLOP/s here.
// Without effect or slower, each measured: the next tile's scores in front of the softmax, fragments read ahead,
// alternating chains of matrix instructions, wave priorities, one workgroup more or less a CU, 64 rows a wave (D = 64:
// 348 us in place of 327).
#include "cg_common.h"

#include <algorithm>
#include <new>
#include <vector>

namespace {

typedef __attribute__((ext_vector_type(4))) short mha_s16x4_t;
typedef __attribute__((address_space(3))) mha_s16x4_t* mha_tr_ptr;
typedef __attribute__((address_space(3))) unsigned char* mha_lds_ptr;
typedef __attribute__((address_space(3))) const bf16x8_t* mha_frag_ptr;

constexpr float LOG2E = 1.4426950408889634f;
constexpr int KT = 64;           // keys of a tile (rows of a tile in the dK / dV kernel)
constexpr int ROW_TILE = 128;    // rows of a forward / dQ work item: 4 waves of 32
constexpr int KEY_TILE = 128;    // keys of a dK / dV work item: 4 waves of 32
constexpr int THIN_ROWS = 32;    // rows of a thin work item: one wave's

constexpr int mha_wider(int DK, int DV) { return DK > DV ? DK : DV; }

struct MhaArgs {
  const bf16_t *q, *k, *v;
  int64_t qt, qh, kt, kh, vt, vh;
  const int4* seqs;         // {q_start, q_len, k_start, k_len}
  const int4* items;        // two int4 an item
  bf16_t* out;
  bf16_t* out_low;          // what the rounding of out left over (training): delta is formed from both
  float* lse;
  float* ws_o;              // partial results, in units of 32 rows: [unit][32][Dv]
  float* ws_ml;             //                                        [unit][32][2]
  const bf16_t *o_in, *o_low;
  const bf16_t* dout;
  const float* lse_in;
  float* delta;
  bf16_t *dq, *dk, *dv;
  int heads, G, kv_heads, D, Dv, causal;
  float c, scale;           // scale * log2(e)
  FastDiv dG;
};

struct MhaItem {
  int seq, hk, row0, k0, k1, part, units;
  int q_start, Lq, k_start, Lk, rows, shift;   // rows = Lq G; row of token t sees keys <= t + shift
};

__device__ __forceinline__ MhaItem mha_item(const MhaArgs& a, int index) {
  const int4 x = a.items[2 * index], y = a.items[2 * index + 1];
  MhaItem it;
  it.seq = __builtin_amdgcn_readfirstlane(x.x);
  it.hk = __builtin_amdgcn_readfirstlane(x.y);
  it.row0 = __builtin_amdgcn_readfirstlane(x.z);
  it.k0 = __builtin_amdgcn_readfirstlane(x.w);
  it.k1 = __builtin_amdgcn_readfirstlane(y.x);
  it.part = __builtin_amdgcn_readfirstlane(y.y);
  it.units = __builtin_amdgcn_readfirstlane(y.z);
  const int4 s = a.seqs[it.seq];
  it.q_start = __builtin_amdgcn_readfirstlane(s.x);
  it.Lq = __builtin_amdgcn_readfirstlane(s.y);
  it.k_start = __builtin_amdgcn_readfirstlane(s.z);
  it.Lk = __builtin_amdgcn_readfirstlane(s.w);
  it.rows = it.Lq * a.G;
  it.shift = a.causal ? it.Lk - it.Lq : 0x40000000;
  return it;
}

// XOR applied to the chunk number of row r (pitch 2 DP bytes).  64 banks of 4 bytes = 256 bytes: rows whose
// pitch is a multiple of that need the spread from the XOR alone (two low row bits move a 64-byte group,
// the next two a chunk inside it); shorter pitches already rotate.
template <int DP>
__device__ __forceinline__ int mha_swz(int r) {
  if constexpr (DP == 128) return ((r & 3) << 2) | ((r >> 2) & 3);
  else if constexpr (DP == 64) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
  else return (r >> 2) & 3;    // DP = 32: pitch 64; DP = 96: pitch 192 (chunk ^ 0..3 stays inside 12)
}

// Copies ROWS rows of 2 DP bytes into LDS.  Chunk i (of ROWS * DP / 8) is lane i % 64 of copy i / 64;
// copy c belongs to wave c % NW.
template <int DP, int ROWS, int NW>
struct MhaStage {
  static constexpr int CH = DP / 8;
  static constexpr int COPIES = ROWS * CH / 64;
  static constexpr int N = COPIES / NW;
  static_assert(COPIES % NW == 0, "copies per wave");
  // row and column (elements) of this lane's chunk in copy n; column >= D: outside
  static __device__ __forceinline__ void place(int n, int wave, int lane, int* row, int* col) {
    const int i = (n * NW + wave) * 64 + lane;
    const int r = i / CH, s = i - r * CH;
    *row = r;
    *col = (s ^ mha_swz<DP>(r)) * 8;
  }
};

constexpr uint32_t OUTSIDE = 0x80000000u;

// per-lane byte offsets of consecutive rows (keys): row * stride + column
template <int DP, int ROWS, int NW, int N>
__device__ __forceinline__ void mha_offsets(uint32_t (&off)[N], int wave, int lane,
                                            int64_t stride, int D) {
  static_assert(N == MhaStage<DP, ROWS, NW>::N, "one offset a copy");
#pragma unroll
  for (int n = 0; n < N; ++n) {
    int r, c;
    MhaStage<DP, ROWS, NW>::place(n, wave, lane, &r, &c);
    off[n] = c < D ? (uint32_t)(r * (uint32_t)(stride * 2) + c * 2) : OUTSIDE;
  }
}
template <int DP, int ROWS, int NW, int N>
__device__ __forceinline__ void mha_copy(const uint32_t (&off)[N], cg_i32x4_t rs,
                                         uint32_t lds, int wave) {
#pragma unroll
  for (int n = 0; n < N; ++n)
    cg_dma16_asm(rs, off[n], 0u, lds + (uint32_t)(n * NW + wave) * 1024u);
}
// descriptor of rows [row, row + ROWS) of a [.., stride] tensor that ends with row `end` (exclusive)
template <int ROWS>
__device__ __forceinline__ cg_i32x4_t mha_rows(const bf16_t* base, int64_t row, int left, int64_t stride, int D) {
  const int n = left < ROWS ? left : ROWS;
  return cg_make_rsrc(base + row * stride, n <= 0 ? 0u : (uint32_t)(n - 1) * (uint32_t)(stride * 2) + (uint32_t)D * 2u);
}

__device__ __forceinline__ bf16x8_t mha_tr2(mha_lds_ptr lo, mha_lds_ptr hi) {
  const mha_s16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((mha_tr_ptr)lo);
  const mha_s16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((mha_tr_ptr)hi);
  const s16x8_t v = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  return __builtin_bit_cast(bf16x8_t, v);
}
__device__ __forceinline__ bf16x8_t mha_pack(const f32x16_t& v, int at) {
  const f32x8_t f = {v[at], v[at + 1], v[at + 2], v[at + 3], v[at + 4], v[at + 5], v[at + 6], v[at + 7]};
  return __builtin_convertvector(f, bf16x8_t);
}
__device__ __forceinline__ f32x16_t mha_zero() {
  f32x16_t z;
#pragma unroll
  for (int v = 0; v < 16; ++v) z[v] = 0.f;
  return z;
}
// one row's (or key's) operand fragments: columns kd * 16 + half * 8 + 0..7
template <int KD>
__device__ __forceinline__ void mha_row_frags(bf16x8_t (&f)[KD], const bf16_t* p, bool ok, int D, int half) {
#pragma unroll
  for (int kd = 0; kd < KD; ++kd) {
    const int d = kd * 16 + half * 8;
    uint4 x = make_uint4(0u, 0u, 0u, 0u);
    if (ok && d < D) x = *reinterpret_cast<const uint4*>(p + d);
    f[kd] = __builtin_bit_cast(bf16x8_t, x);
  }
}

// Waits here for fragments loaded from memory.  Without it the first use is inside the tile loop, and the compiler,
// which does not see the asm copies, puts a vmcnt wait there that holds every pass for the copies of the NEXT tile
template <int KD>
__device__ __forceinline__ void mha_settle(bf16x8_t (&f)[KD]) {
#pragma unroll
  for (int kd = 0; kd < KD; ++kd) asm volatile("" : "+v"(f[kd]));
}

// LDS offsets of a lane's reads in a tile of 2 DP byte rows
template <int DP>
struct MhaReads {
  uint32_t row[DP / 16];       // b128: row lane & 31, columns kd 16 + half 8 ..
  uint32_t tr[DP / 32][2];     // b64 transposed: rows 4 half + 0..3 (+ 8), columns t 32 ..
};
template <int DP>
__device__ __forceinline__ MhaReads<DP> mha_reads(int lane) {
  MhaReads<DP> m;
  const int col = lane & 31, half = lane >> 5;
#pragma unroll
  for (int kd = 0; kd < DP / 16; ++kd)
    m.row[kd] = (uint32_t)(col * 2 * DP + (((kd * 2 + half) ^ mha_swz<DP>(col)) << 4));
  const int l16 = lane & 15, tcol = ((lane >> 4) & 1) * 16 + (l16 & 3) * 4;
#pragma unroll
  for (int t = 0; t < DP / 32; ++t)
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int r = 4 * half + 8 * p + (l16 >> 2), c = t * 32 + tcol;
      m.tr[t][p] = (uint32_t)(r * 2 * DP + (((c >> 3) ^ mha_swz<DP>(r)) << 4) + (c & 7) * 2);
    }
  return m;
}

// S^T tile of 32 keys (rows `sub` of the LDS tile) and one wave's 32 rows
template <int DP>
__device__ __forceinline__ f32x16_t mha_product(mha_lds_ptr tile, const MhaReads<DP>& m,
                                                const bf16x8_t (&f)[DP / 16], int sub, f32x16_t s = mha_zero()) {
#pragma unroll
  for (int kd = 0; kd < DP / 16; ++kd) {
    const bf16x8_t x = *(mha_frag_ptr)(tile + m.row[kd] + sub * 64 * DP);
    s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, f[kd], s, 0, 0, 0);
  }
  return s;
}
// acc[t] += (tile^T)[t 32 .. +31][32 keys of sub] * p
template <int DP>
__device__ __forceinline__ void mha_accumulate(f32x16_t (&acc)[DP / 32], mha_lds_ptr tile, const MhaReads<DP>& m,
                                               const f32x16_t& p, int sub) {
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    const bf16x8_t pf = mha_pack(p, 8 * ks);
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) {
      const uint32_t at = (uint32_t)(sub * 64 * DP + ks * 32 * DP);
      const bf16x8_t x = mha_tr2(tile + m.tr[t][0] + at, tile + m.tr[t][1] + at);
      acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, pf, acc[t], 0, 0, 0);
    }
  }
}
// Entries that are not finite, where a causal mask cuts through a tile: a masked weight is 0, but 0 times an infinity or
// NaN is NaN.  The tile's threads look its 16-byte chunks over, put zeros for such entries and keep the first (LAST: the
// last) row that held one; the caller makes NaN of every result that sees that row.  So a value that is not finite reaches
// whole rows here (elsewhere the entries that the product brings it to), and only those that see it.  Costs one read of
// the tile by its workgroup, in tiles on the diagonal only.
template <int DP, int ROWS, int NT, bool LAST>
__device__ __forceinline__ void mha_clean(unsigned char* tile, int thread, int* bad) {
  constexpr int CH = DP / 8, TOTAL = ROWS * CH;
  static_assert(TOTAL % NT == 0, "chunks per thread");
#pragma unroll 1
  for (int i = thread; i < TOTAL; i += NT) {
    uint4* at = reinterpret_cast<uint4*>(tile + i * 16);
    uint4 q = *at;
    const uint32_t odd = ((q.x & 0x7f807f80u) + 0x00800080u) | ((q.y & 0x7f807f80u) + 0x00800080u) |
                         ((q.z & 0x7f807f80u) + 0x00800080u) | ((q.w & 0x7f807f80u) + 0x00800080u);
    if (odd & 0x80008000u) {
      s16x8_t v = __builtin_bit_cast(s16x8_t, q);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if ((v[e] & 0x7f80) == 0x7f80) v[e] = 0;
      *at = __builtin_bit_cast(uint4, v);
      if (LAST) atomicMax(bad, i / CH);
      else atomicMin(bad, i / CH);
    }
  }
}
constexpr int NONE_BAD = 0x40000000;    // no row (LAST: its negative)

// what the rounding of the weights left over, for rows that see few keys (FEW): their O is the mean of a few values, the
// error of their weights does not average out, and delta = dO . O carries it into every dS of the row
template <int DP>
__device__ __forceinline__ void mha_accumulate_low(f32x16_t (&acc)[DP / 32], mha_lds_ptr tile, const MhaReads<DP>& m,
                                                   const f32x16_t& p, int sub) {
  f32x16_t low;
#pragma unroll
  for (int v = 0; v < 16; ++v) low[v] = p[v] - bf2f(f2bf(p[v]));    // (packed conversions: 34 spills, 938 -> 1092 us)
  mha_accumulate<DP>(acc, tile, m, low, sub);
}
constexpr int FEW = 64;

__device__ __forceinline__ int mha_key(int v, int half) { return (v & 3) + 8 * (v >> 2) + 4 * half; }

// Running softmax over the 64 (NS = 2) or 32 (NS = 1) keys of s: in s the scores, out the weights
// 2^(c s - m).  m, the reference exponent, is only raised when a row's maximum has passed it by more than 8:
// weights stay below 2^8 (the same relative rounding in bf16, no danger in the fp32 sums) and the rescaling
// of the accumulators is skipped in nearly every tile.
constexpr float RAISE = 8.f;
template <int NS, int NT>
__device__ __forceinline__ void mha_softmax(f32x16_t (&s)[NS], float c, float& m, float& l, f32x16_t (&o)[NT]) {
  float mx = -INFINITY;
#pragma unroll
  for (int n = 0; n < NS; ++n)
#pragma unroll
    for (int v = 0; v < 16; ++v) mx = fmaxf(mx, s[n][v]);
  mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * c;
  if (__any(mx > m + RAISE)) {      // (m = -inf: raised by the first finite maximum)
    const float up = fmaxf(m, mx);
    const float f = up == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - up);
    m = up;
    l *= f;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int v = 0; v < 16; ++v) o[t][v] *= f;
  }
  const float ref = m == -INFINITY ? 0.f : m;     // nothing seen yet: the weights are 2^-inf = 0
#pragma unroll
  for (int n = 0; n < NS; ++n)
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      s[n][v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][v], c, -ref));
      l += s[n][v];
    }
}

// factor that brings a result with reference exponent m to the common one; m = -inf: nothing was seen
// (its sums are 0, or NaN where a score was NaN, which has to stay)
__device__ __forceinline__ float mha_weight(float m, float top) {
  return m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - top);
}

// row r of the item's sequence: offset of its (token, head) in a [rows, heads] tensor, and its address
__device__ __forceinline__ void mha_token(const MhaArgs& a, const MhaItem& it, int r, int* t, int* h) {
  *t = (int)fdiv((uint32_t)r, a.dG);
  *h = it.hk * a.G + (r - *t * a.G);
}

// a lane's row of an accumulator, fp32, to a partial result
template <int DP>
__device__ __forceinline__ void mha_store_part(float* dst, const f32x16_t (&o)[DP / 32], int width, int half,
                                               float f = 1.f) {
#pragma unroll
  for (int t = 0; t < DP / 32; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = t * 32 + g * 8 + 4 * half;
      if (d < width)
        *reinterpret_cast<float4*>(dst + d) =
            make_float4(o[t][4 * g] * f, o[t][4 * g + 1] * f, o[t][4 * g + 2] * f, o[t][4 * g + 3] * f);
    }
}

// what a wave leaves behind: O^T in registers -> out, or a partial result
template <int DV, bool GRAD>
__device__ __forceinline__ void mha_store(const MhaArgs& a, const MhaItem& it, int r, float m, float l,
                                          f32x16_t (&o)[DV / 32], int half) {
  if (r >= it.rows) return;
  if (it.part >= 0) {
    const int64_t at = (int64_t)it.part * THIN_ROWS + (r - it.row0);
    mha_store_part<DV>(a.ws_o + at * a.Dv, o, a.Dv, half);
    if (half == 0) *reinterpret_cast<float2*>(a.ws_ml + at * 2) = make_float2(m, l);
    return;
  }
  int t_, h;
  mha_token(a, it, r, &t_, &h);
  const int64_t row = (int64_t)(it.q_start + t_) * a.heads + h;
  const float inv = l == 0.f ? 0.f : 1.f / l;       // a row that sees no key: 0
  bf16_t* dst = a.out + row * a.Dv;
#pragma unroll
  for (int t = 0; t < DV / 32; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = t * 32 + g * 8 + 4 * half;
      if (d < a.Dv) {
        float w[4] = {o[t][4 * g] * inv, o[t][4 * g + 1] * inv, o[t][4 * g + 2] * inv, o[t][4 * g + 3] * inv};
        const uint2 hi = pack4_bf16(w);
        *reinterpret_cast<uint2*>(dst + d) = hi;
        if (GRAD) {
          w[0] -= __uint_as_float(hi.x << 16);
          w[1] -= __uint_as_float(hi.x & 0xffff0000u);
          w[2] -= __uint_as_float(hi.y << 16);
          w[3] -= __uint_as_float(hi.y & 0xffff0000u);
          *reinterpret_cast<uint2*>(a.out_low + row * a.Dv + d) = pack4_bf16(w);
        }
      }
    }
  if (a.lse && half == 0) a.lse[row] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * (1.f / LOG2E);
}

// ---- forward, 128 rows x all keys of the item ---------------------------------------------------
// Measured: 64 x 4096 tokens, 3 heads of 64, 920 to 1020 us (810 to 900 TFLOP/s); 16 384 tokens causal, 16 heads of 128
// on 4 key heads, 1.07 to 1.18 ms (0.93 to 1.03 PFLOP/s counted without the masked half); ragged causal batch, 8 heads of
// 96 on 2, 165 to 190 us (620 to 710 TFLOP/s: diagonals and the end of the launch).
template <int DK, int DV, bool GRAD>
__global__ __launch_bounds__(256, mha_wider(DK, DV) <= 64 ? 4 : mha_wider(DK, DV) <= 96 ? 3 : 2) void mha_fwd_kernel(MhaArgs a) {
  constexpr int TK = KT * DK * 2, TILES = TK + KT * DV * 2;      // K, and K with V
  __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * TILES];
  __shared__ int sm_bad[2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, col = lane & 31;
  const MhaItem it = mha_item(a, blockIdx.x);
  const int cut = a.causal ? (int)fdiv((uint32_t)it.row0, a.dG) + it.shift : NONE_BAD;   // last key of the first row
  const int r = it.row0 + wave * 32 + col;
  int t, h;
  mha_token(a, it, r, &t, &h);
  const bool ok = r < it.rows;
  bf16x8_t qf[DK / 16];
  mha_row_frags(qf, a.q + (int64_t)(it.q_start + t) * a.qt + (int64_t)h * a.qh, ok, a.D, half);
  // last key this row sees (exclusive end of the item's keys included)
  const int last = ok ? min(it.k1 - 1, t + it.shift) : -1;
  int least = last, most = last;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    least = min(least, __shfl_xor(least, s, 64));
    most = max(most, __shfl_xor(most, s, 64));
  }
  least = __builtin_amdgcn_readfirstlane(least);
  most = __builtin_amdgcn_readfirstlane(most);
  uint32_t koff[MhaStage<DK, KT, 4>::N], voff[MhaStage<DV, KT, 4>::N];
  mha_offsets<DK, KT, 4>(koff, wave, lane, a.kt, a.D);
  mha_offsets<DV, KT, 4>(voff, wave, lane, a.vt, a.Dv);
  const MhaReads<DK> rk = mha_reads<DK>(lane);
  const MhaReads<DV> rv = mha_reads<DV>(lane);
  const bf16_t* kb = a.k + (int64_t)it.hk * a.kh;
  const bf16_t* vb = a.v + (int64_t)it.hk * a.vh;
  const uint32_t lds = cg_lds_addr(smem);
  mha_lds_ptr sm = (mha_lds_ptr)smem;
  auto stage = [&](int k0, int buf) {
    mha_copy<DK, KT, 4>(koff, mha_rows<KT>(kb, it.k_start + k0, it.Lk - k0, a.kt, a.D), lds + buf * TILES, wave);
    mha_copy<DV, KT, 4>(voff, mha_rows<KT>(vb, it.k_start + k0, it.Lk - k0, a.vt, a.Dv), lds + buf * TILES + TK, wave);
  };
  f32x16_t o[DV / 32];
#pragma unroll
  for (int i = 0; i < DV / 32; ++i) o[i] = mha_zero();
  float m = -INFINITY, l = 0.f;
  if (it.k0 < it.k1) stage(it.k0, 0);
  mha_settle(qf);
  int buf = 0;
  for (int k0 = it.k0; k0 < it.k1; k0 += KT, buf ^= 1) {
    if (threadIdx.x == 0) sm_bad[buf] = NONE_BAD;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (k0 + KT < it.k1) stage(k0 + KT, buf ^ 1);
    if (k0 + KT - 1 > cut) {                       // the diagonal
      mha_clean<DV, KT, 256, false>(smem + buf * TILES + TK, threadIdx.x, &sm_bad[buf]);
      __syncthreads();
      if (k0 + sm_bad[buf] <= last) l = __builtin_nanf("");
    }
    if (k0 > most) continue;
    mha_lds_ptr ks = sm + buf * TILES, vs = ks + TK;
    f32x16_t s[2];
    s[0] = mha_product<DK>(ks, rk, qf, 0);
    s[1] = mha_product<DK>(ks, rk, qf, 1);
    if (k0 + KT - 1 > least) {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int v = 0; v < 16; ++v)
          s[n][v] = k0 + n * 32 + mha_key(v, half) <= last ? s[n][v] : -INFINITY;
    }
    mha_softmax<2, DV / 32>(s, a.c, m, l, o);
    mha_accumulate<DV>(o, vs, rv, s[0], 0);
    mha_accumulate<DV>(o, vs, rv, s[1], 1);
    if (GRAD && most < FEW) {
      mha_accumulate_low<DV>(o, vs, rv, s[0], 0);
      mha_accumulate_low<DV>(o, vs, rv, s[1], 1);
    }
  }
  l += __shfl_xor(l, 32, 64);
  mha_store<DV, GRAD>(a, it, r, m, l, o, half);
}

// ---- forward, at most 32 rows: the keys split over the waves --------------------------------------
// One wave holds all rows; each of the NW waves takes every NW-th step of 32 keys through an LDS ring of its
// own (no barrier in the loop), and the waves' results are joined at the end.  Bound by reading K and V: 48 new tokens,
// 32 heads of 128 on 8, against up to 8192 keys each, 795 MB in 155 to 160 us (5.0 to 5.1 TB/s; a copy of 256 MiB reaches 5.4);
// of a sequence with few keys (NW = 1, one wave an item), 256 x 16 tokens, 8 heads of 64: 7 to 8 us, what launching 2048 waves
// and one trip to memory and back take.
template <int DK, int DV, int NW, bool GRAD>
__global__ __launch_bounds__(NW * 64) void mha_thin_kernel(MhaArgs a) {
  constexpr int TK = 32 * DK * 2, TILES = TK + 32 * DV * 2;      // 32 keys of K, and with V
  constexpr int RING = 2 * TILES;                // two buffers, a wave
  __shared__ __attribute__((aligned(1024))) unsigned char smem[NW * RING];
  __shared__ float sm_m[NW][32], sm_l[NW][32];
  __shared__ int sm_bad[NW];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, col = lane & 31;
  const MhaItem it = mha_item(a, blockIdx.x);
  int t, h;
  mha_token(a, it, col, &t, &h);
  const bool ok = col < it.rows;
  bf16x8_t qf[DK / 16];
  mha_row_frags(qf, a.q + (int64_t)(it.q_start + t) * a.qt + (int64_t)h * a.qh, ok, a.D, half);
  const int last = ok ? min(it.k1 - 1, t + it.shift) : -1;
  int least = last;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) least = min(least, __shfl_xor(least, s, 64));
  if (it.rows < 32) {          // columns without a row need no mask of their own: nothing of them is kept
    least = 0x7fffffff;
    for (int s = 0; s < it.rows; ++s) least = min(least, __shfl(last, s, 64));
  }
  least = __builtin_amdgcn_readfirstlane(least);
  using StageK = MhaStage<DK, 32, 1>;
  using StageV = MhaStage<DV, 32, 1>;
  uint32_t koff[StageK::N], voff[StageV::N];
  mha_offsets<DK, 32, 1>(koff, 0, lane, a.kt, a.D);
  mha_offsets<DV, 32, 1>(voff, 0, lane, a.vt, a.Dv);
  const MhaReads<DK> rk = mha_reads<DK>(lane);
  const MhaReads<DV> rv = mha_reads<DV>(lane);
  const bf16_t* kb = a.k + (int64_t)it.hk * a.kh;
  const bf16_t* vb = a.v + (int64_t)it.hk * a.vh;
  const uint32_t lds = cg_lds_addr(smem) + wave * RING;
  mha_lds_ptr sm = (mha_lds_ptr)smem + wave * RING;
  auto stage = [&](int k0, int buf) {
    mha_copy<DK, 32, 1>(koff, mha_rows<32>(kb, it.k_start + k0, it.Lk - k0, a.kt, a.D), lds + buf * TILES, 0);
    mha_copy<DV, 32, 1>(voff, mha_rows<32>(vb, it.k_start + k0, it.Lk - k0, a.vt, a.Dv), lds + buf * TILES + TK, 0);
  };
  f32x16_t o[DV / 32];
#pragma unroll
  for (int i = 0; i < DV / 32; ++i) o[i] = mha_zero();
  float m = -INFINITY, l = 0.f;
  const int first = it.k0 + wave * 32;
  constexpr int INFLIGHT = StageK::N + StageV::N;         // copies of one step
  if (first < it.k1) stage(first, 0);
  mha_settle(qf);
  int buf = 0;
  for (int k0 = first; k0 < it.k1; k0 += NW * 32, buf ^= 1) {
    // the other buffer was read in the last step: those reads have returned (their values were used)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (k0 + NW * 32 < it.k1) {
      stage(k0 + NW * 32, buf ^ 1);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(INFLIGHT) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    mha_lds_ptr ks = sm + buf * TILES, vs = ks + TK;
    if (a.causal && k0 + 31 > least) {             // the diagonal: this wave's own tile and flag
      if (lane == 0) sm_bad[wave] = NONE_BAD;
      mha_clean<DV, 32, 64, false>(smem + wave * RING + buf * TILES + TK, lane, &sm_bad[wave]);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (k0 + *(volatile int*)&sm_bad[wave] <= last) l = __builtin_nanf("");
    }
    f32x16_t s[1];
    s[0] = mha_product<DK>(ks, rk, qf, 0);
    if (k0 + 31 > least) {
#pragma unroll
      for (int v = 0; v < 16; ++v) s[0][v] = k0 + mha_key(v, half) <= last ? s[0][v] : -INFINITY;
    }
    mha_softmax<1, DV / 32>(s, a.c, m, l, o);
    mha_accumulate<DV>(o, vs, rv, s[0], 0);
    if (GRAD && it.k1 <= FEW) mha_accumulate_low<DV>(o, vs, rv, s[0], 0);
  }
  l += __shfl_xor(l, 32, 64);
  if constexpr (NW > 1) {
    if (half == 0) {
      sm_m[wave][col] = m;
      sm_l[wave][col] = l;
    }
    __syncthreads();                             // every wave is done with its ring, too
    float top = sm_m[0][col];
#pragma unroll
    for (int w = 1; w < NW; ++w) top = fmaxf(top, sm_m[w][col]);
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) total += sm_l[w][col] * mha_weight(sm_m[w][col], top);
    const float mine = mha_weight(m, top);
    // joined two waves at a time in a fixed order: wave w hands its scaled O to wave w - step
    float* box = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int i = 0; i < DV / 32; ++i)
#pragma unroll
      for (int v = 0; v < 16; ++v) o[i][v] *= mine;
#pragma unroll
    for (int step = NW / 2; step > 0; step >>= 1) {
      if (wave >= step && wave < 2 * step) {
#pragma unroll
        for (int i = 0; i < DV / 32; ++i)
#pragma unroll
          for (int v = 0; v < 16; ++v) box[((wave - step) * (DV / 32) * 16 + i * 16 + v) * 64 + lane] = o[i][v];
      }
      __syncthreads();
      if (wave < step) {
#pragma unroll
        for (int i = 0; i < DV / 32; ++i)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[i][v] += box[(wave * (DV / 32) * 16 + i * 16 + v) * 64 + lane];
      }
      __syncthreads();
    }
    if (wave != 0) return;
    m = top;
    l = total;
  }
  mha_store<DV, GRAD>(a, it, col, m, l, o, half);
}

// ---- joins the partial results of a split item ----------------------------------------------------
// item {seq, hk, row0, rows here, parts, first unit, units a part}.  A block's rows, four values a thread; where they are
// less than 256 threads the parts are dealt to groups of threads as well, and the groups' results joined through LDS in
// their order: a few rows with hundreds of parts are a few loads behind one another.  Bound by the partial results' bytes
// (ragged batch: 30 MB in 12 us); one new token against 131 072 keys, 8 heads: 125 us with the kernel in front of it.
__global__ __launch_bounds__(256) void mha_join_kernel(MhaArgs a) {
  __shared__ float box[6][256];
  const MhaItem it = mha_item(a, blockIdx.x);
  const int parts = it.k1, quads = a.Dv / 4;
  const int64_t step = (int64_t)it.units * THIN_ROWS;
  const int share = (it.k0 + gridDim.y - 1) / gridDim.y, first = blockIdx.y * share;
  const int units = min(share, it.k0 - first) * quads;
  if (units <= 0) return;
  const int groups = units < 256 ? 256 / units : 1;
  const int group = groups > 1 ? threadIdx.x / units : 0;
  for (int u = threadIdx.x - group * units; u < units; u += 256) {
    const int i = u / quads, d = (u - i * quads) * 4, n = first + i;
    const int64_t at = (int64_t)it.part * THIN_ROWS + n;
    float top = -INFINITY, total = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
    if (group < groups) {
#pragma unroll 8
      for (int p = group; p < parts; p += groups) top = fmaxf(top, a.ws_ml[(at + p * step) * 2]);
#pragma unroll 4
      for (int p = group; p < parts; p += groups) {
        const float2 ml = *reinterpret_cast<const float2*>(a.ws_ml + (at + p * step) * 2);
        const float4 o = *reinterpret_cast<const float4*>(a.ws_o + (at + p * step) * a.Dv + d);
        const float w = mha_weight(ml.x, top);
        total += ml.y * w;
        x[0] += o.x * w; x[1] += o.y * w; x[2] += o.z * w; x[3] += o.w * w;
      }
    }
    if (groups > 1) {          // (the same for all of the block, and its threads are here once)
      box[0][threadIdx.x] = top;
      box[1][threadIdx.x] = total;
#pragma unroll
      for (int j = 0; j < 4; ++j) box[2 + j][threadIdx.x] = x[j];
      __syncthreads();
      if (group > 0) return;
      float all = top;
      for (int g = 1; g < groups; ++g) all = fmaxf(all, box[0][g * units + u]);
      const float mine = mha_weight(top, all);
      total *= mine;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] *= mine;
      for (int g = 1; g < groups; ++g) {
        const float w = mha_weight(box[0][g * units + u], all);
        total += box[1][g * units + u] * w;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] += box[2 + j][g * units + u] * w;
      }
      top = all;
    }
    int t, h;
    mha_token(a, it, it.row0 + n, &t, &h);
    const int64_t row = (int64_t)(it.q_start + t) * a.heads + h;
    const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] *= inv;
    const uint2 hi = pack4_bf16(x);
    *reinterpret_cast<uint2*>(a.out + row * a.Dv + d) = hi;
    if (a.out_low) {
      x[0] -= __uint_as_float(hi.x << 16);
      x[1] -= __uint_as_float(hi.x & 0xffff0000u);
      x[2] -= __uint_as_float(hi.y << 16);
      x[3] -= __uint_as_float(hi.y & 0xffff0000u);
      *reinterpret_cast<uint2*>(a.out_low + row * a.Dv + d) = pack4_bf16(x);
    }
    if (a.lse && d == 0)
      a.lse[row] = total == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * (1.f / LOG2E);
  }
}

// ---- backward -----------------------------------------------------------------------------------
// what the weights are rebuilt from, in exponents of two; a row that saw no key: +inf (weights 0)
__device__ __forceinline__ float mha_lse2(float lse) { return lse == -INFINITY ? INFINITY : lse * LOG2E; }

// dQ: 128 rows x all keys; S^T and dP^T = V dO^T side by side, dQ^T += K^T dS^T.  delta = dO . (out + out_low) of its
// rows is formed on the way in (dO is in registers for dP) and left for the dK / dV kernel behind it.  dS = P (dP - delta)
// is a difference: with the rounded out alone its error would come on top of the rounding of dS (dQ 1.5 instead of 1.4
// roundings off).
// Measured: 64 x 4096 tokens, 3 heads of 64, 1.19 to 1.24 ms (1.0 to 1.04 PFLOP/s over its three products), delta included
// (59 us as a kernel of its own).  Three workgroups a CU at 96 wide heads (2 to 4 spills, outside the loop's products):
// 8 x 4096 tokens, 8 heads, backward 1391 -> 1373 us; ragged training batch 769 -> 758 us.
template <int DK, int DV>
__global__ __launch_bounds__(256, mha_wider(DK, DV) <= 64 ? 4 : mha_wider(DK, DV) <= 96 ? 3 : 2) void mha_bwd_q_kernel(MhaArgs a) {
  constexpr int TK = KT * DK * 2, TILES = TK + KT * DV * 2;      // K, and K with V
  __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * TILES];
  __shared__ int sm_bad[2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, col = lane & 31;
  const MhaItem it = mha_item(a, blockIdx.x);
  const int cut = a.causal ? (int)fdiv((uint32_t)it.row0, a.dG) + it.shift : NONE_BAD;   // last key of the first row
  const int r = it.row0 + wave * 32 + col;
  int t, h;
  mha_token(a, it, r, &t, &h);
  const bool ok = r < it.rows;
  const int64_t row = (int64_t)(it.q_start + t) * a.heads + h;
  bf16x8_t qf[DK / 16], df[DV / 16];
  mha_row_frags(qf, a.q + (int64_t)(it.q_start + t) * a.qt + (int64_t)h * a.qh, ok, a.D, half);
  mha_row_frags(df, a.dout + row * a.Dv, ok, a.Dv, half);
  const float lse2 = ok ? mha_lse2(a.lse_in[row]) : INFINITY;
  float delta = 0.f;
#pragma unroll
  for (int kd = 0; kd < DV / 16; ++kd) {
    const int d = kd * 16 + half * 8;
    if (ok && d < a.Dv) {
      float x[8], y[8], z[8];
      unpack8_bf16(*reinterpret_cast<const uint4*>(a.o_in + row * a.Dv + d), x);
      unpack8_bf16(*reinterpret_cast<const uint4*>(a.o_low + row * a.Dv + d), y);
      unpack8_bf16(__builtin_bit_cast(uint4, df[kd]), z);
#pragma unroll
      for (int j = 0; j < 8; ++j) delta += (x[j] + y[j]) * z[j];
    }
  }
  delta += __shfl_xor(delta, 32, 64);
  if (ok && half == 0) a.delta[row] = delta;     // (parts of a split item write the same value)
  const int last = ok ? min(it.k1 - 1, t + it.shift) : -1;
  int least = last, most = last;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    least = min(least, __shfl_xor(least, s, 64));
    most = max(most, __shfl_xor(most, s, 64));
  }
  least = __builtin_amdgcn_readfirstlane(least);
  most = __builtin_amdgcn_readfirstlane(most);
  uint32_t koff[MhaStage<DK, KT, 4>::N], voff[MhaStage<DV, KT, 4>::N];
  mha_offsets<DK, KT, 4>(koff, wave, lane, a.kt, a.D);
  mha_offsets<DV, KT, 4>(voff, wave, lane, a.vt, a.Dv);
  const MhaReads<DK> rk = mha_reads<DK>(lane);
  const MhaReads<DV> rv = mha_reads<DV>(lane);
  const bf16_t* kb = a.k + (int64_t)it.hk * a.kh;
  const bf16_t* vb = a.v + (int64_t)it.hk * a.vh;
  const uint32_t lds = cg_lds_addr(smem);
  mha_lds_ptr sm = (mha_lds_ptr)smem;
  auto stage = [&](int k0, int buf) {
    mha_copy<DK, KT, 4>(koff, mha_rows<KT>(kb, it.k_start + k0, it.Lk - k0, a.kt, a.D), lds + buf * TILES, wave);
    mha_copy<DV, KT, 4>(voff, mha_rows<KT>(vb, it.k_start + k0, it.Lk - k0, a.vt, a.Dv), lds + buf * TILES + TK, wave);
  };
  f32x16_t dq[DK / 32];
#pragma unroll
  for (int i = 0; i < DK / 32; ++i) dq[i] = mha_zero();
  if (it.k0 < it.k1) stage(it.k0, 0);
  float scale = a.scale;         // NaN: the row saw a key that is not finite
  mha_settle(qf);
  mha_settle(df);
  int buf = 0;
  for (int k0 = it.k0; k0 < it.k1; k0 += KT, buf ^= 1) {
    if (threadIdx.x == 0) sm_bad[buf] = NONE_BAD;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (k0 + KT < it.k1) stage(k0 + KT, buf ^ 1);
    if (k0 + KT - 1 > cut) {                       // the diagonal
      mha_clean<DK, KT, 256, false>(smem + buf * TILES, threadIdx.x, &sm_bad[buf]);
      __syncthreads();
      if (k0 + sm_bad[buf] <= last) scale = __builtin_nanf("");
    }
    if (k0 > most) continue;
    mha_lds_ptr ks = sm + buf * TILES, vs = ks + TK;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      __builtin_amdgcn_sched_barrier(0);      // one step's scores live at a time
      f32x16_t s = mha_product<DK>(ks, rk, qf, n);
      const f32x16_t dp = mha_product<DV>(vs, rv, df, n);
#pragma unroll
      for (int v = 0; v < 16; ++v)
        s[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], a.c, -lse2)) * (dp[v] - delta);
      if (k0 + n * 32 + 31 > least) {
#pragma unroll
        for (int v = 0; v < 16; ++v) s[v] = k0 + n * 32 + mha_key(v, half) <= last ? s[v] : 0.f;
      }
      mha_accumulate<DK>(dq, ks, rk, s, n);
    }
  }
  if (!ok) return;
  if (it.part >= 0) {
    mha_store_part<DK>(a.ws_o + ((int64_t)it.part * ROW_TILE + r - it.row0) * a.D, dq, a.D, half, scale == scale ? 1.f : scale);
    return;
  }
  bf16_t* dst = a.dq + row * a.D;
#pragma unroll
  for (int i = 0; i < DK / 32; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = i * 32 + g * 8 + 4 * half;
      if (d < a.D) {
        const float w[4] = {dq[i][4 * g] * scale, dq[i][4 * g + 1] * scale, dq[i][4 * g + 2] * scale, dq[i][4 * g + 3] * scale};
        *reinterpret_cast<uint2*>(dst + d) = pack4_bf16(w);
      }
    }
}

// dK, dV: 128 keys x the rows that see them.  S[row][key] = Q K^T and dP = dO V^T with the keys in the lanes'
// columns; dV^T += dO^T P, dK^T += Q^T dS.  Item {seq, hk, key0, first row, end row}.
// At 128 wide heads the accumulators, K and V of a wave would be 192 registers and the rest spills (each reload also
// waits for the copies in flight): V is read from LDS there, and the tiles are 32 rows so that two workgroups fit a CU.
// Measured: 64 x 4096 tokens, 3 heads of 64, 1.62 to 1.84 ms (0.90 to 1.02 PFLOP/s over its four products); ragged causal
// batch, 8 heads of 96 / 64 on 2: 285 to 330 us.
template <int DK, int DV>
__global__ __launch_bounds__(256, mha_wider(DK, DV) <= 64 ? 3 : 2) void mha_bwd_kv_kernel(MhaArgs a) {
  constexpr bool V_LDS = DK + DV > 224;
  constexpr int RT = V_LDS ? 32 : 64;             // rows of a tile
  constexpr int TQ = RT * DK * 2, TILES = TQ + RT * DV * 2;      // Q, and Q with dO
  constexpr int V_BYTES = V_LDS ? KEY_TILE * DV * 2 : 0;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * TILES + V_BYTES];
  __shared__ __attribute__((aligned(16))) float stat[2][2][RT];   // [buffer][lse, -delta][row]
  __shared__ int sm_bad[2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, col = lane & 31;
  const MhaItem it = mha_item(a, blockIdx.x);
  const int key = it.row0 + wave * 32 + col;
  const bool ok = key < it.Lk;
  bf16x8_t kf[DK / 16], vf[V_LDS ? 1 : DV / 16];
  mha_row_frags(kf, a.k + (int64_t)(it.k_start + key) * a.kt + (int64_t)it.hk * a.kh, ok, a.D, half);
  if constexpr (!V_LDS) mha_row_frags(vf, a.v + (int64_t)(it.k_start + key) * a.vt + (int64_t)it.hk * a.vh, ok, a.Dv, half);
  // first row that sees this key; rows of the wave's first and last key for skipping and masking
  auto first_row = [&](int k) { return a.causal ? max(0, k - it.shift) * a.G : 0; };
  const int mine = first_row(key);
  const int wave_first = first_row(it.row0 + wave * 32), wave_all = first_row(it.row0 + wave * 32 + 31);
  const int all_first = first_row(min(it.row0 + KEY_TILE, it.Lk) - 1);   // first row that sees all keys of the item
  const bool some = it.row0 + wave * 32 < it.Lk;
  const int rb = it.k0, re = it.k1;
  const MhaReads<DK> rk = mha_reads<DK>(lane);
  const MhaReads<DV> rv = mha_reads<DV>(lane);
  const bf16_t* qb = a.q + (int64_t)it.hk * a.G * a.qh;
  const bf16_t* db = a.dout + (int64_t)it.hk * a.G * a.Dv;
  const uint32_t lds = cg_lds_addr(smem);
  mha_lds_ptr sm = (mha_lds_ptr)smem;
  const int64_t dt = (int64_t)a.heads * a.Dv;
  auto stage = [&](int r0, int buf) {
    // rows r0 .. gathered by (token, head) relative to the first one's token
    const int t0 = __builtin_amdgcn_readfirstlane((int)fdiv((uint32_t)r0, a.dG));
    const cg_i32x4_t qr = cg_make_rsrc(qb + (int64_t)(it.q_start + t0) * a.qt, 0x7fffffffu);
    const cg_i32x4_t dr = cg_make_rsrc(db + (int64_t)(it.q_start + t0) * dt, 0x7fffffffu);
    auto gather = [&](auto stage_of, const cg_i32x4_t& rs, int width, uint32_t row_bytes, uint32_t head_bytes,
                      uint32_t to) {
      using Stage = decltype(stage_of);
#pragma unroll
      for (int n = 0; n < Stage::N; ++n) {
        int i, c;
        Stage::place(n, wave, lane, &i, &c);
        const int r = r0 + i;
        const int t = (int)fdiv((uint32_t)r, a.dG), g = r - t * a.G;
        cg_dma16_asm(rs, r < re && c < width ? (uint32_t)(t - t0) * row_bytes + (uint32_t)g * head_bytes + c * 2 : OUTSIDE,
                     0u, to + (uint32_t)(n * 4 + wave) * 1024u);
      }
    };
    gather(MhaStage<DK, RT, 4>(), qr, a.D, (uint32_t)(a.qt * 2), (uint32_t)(a.qh * 2), lds + buf * TILES);
    gather(MhaStage<DV, RT, 4>(), dr, a.Dv, (uint32_t)(dt * 2), (uint32_t)(a.Dv * 2), lds + buf * TILES + TQ);
  };
  f32x16_t dk[DK / 32], dv[DV / 32];
#pragma unroll
  for (int i = 0; i < DK / 32; ++i) dk[i] = mha_zero();
#pragma unroll
  for (int i = 0; i < DV / 32; ++i) dv[i] = mha_zero();

  // wave 0 / 1 carry the statistics of the next tile, one row a lane: loaded here, touched a tile later (a use next to
  // the load would hold the two waves, and at the barrier all, for the load's whole latency in every tile)
  auto stat_load = [&](int r0) {
    const int r = r0 + lane;
    if (wave > 1 || lane >= RT || r >= re) return wave == 0 ? -INFINITY : 0.f;
    const int t = (int)fdiv((uint32_t)r, a.dG), g = r - t * a.G;
    const int64_t row = (int64_t)(it.q_start + t) * a.heads + it.hk * a.G + g;
    return wave == 0 ? a.lse_in[row] : a.delta[row];
  };
  float next = 0.f;
  if (rb < re) {
    if constexpr (V_LDS) {                          // the item's 128 rows of V, once
      uint32_t voff[MhaStage<DV, KEY_TILE, 4>::N];
      mha_offsets<DV, KEY_TILE, 4>(voff, wave, lane, a.vt, a.Dv);
      mha_copy<DV, KEY_TILE, 4>(voff, mha_rows<KEY_TILE>(a.v + (int64_t)it.hk * a.vh, it.k_start + it.row0, it.Lk - it.row0,
                                                         a.vt, a.Dv), lds + 2 * TILES, wave);
    }
    next = stat_load(rb);
    stage(rb, 0);
  }
  float scale = a.scale;         // NaN: the key was seen by a row that is not finite
  mha_settle(kf);
  if constexpr (!V_LDS) mha_settle(vf);
  int buf = 0;
  for (int r0 = rb; r0 < re; r0 += RT, buf ^= 1) {
    if (threadIdx.x == 0) sm_bad[buf] = -NONE_BAD;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (wave < 2 && lane < RT) stat[buf][wave][lane] = wave == 0 ? mha_lse2(next) : -next;
    __syncthreads();
    if (r0 + RT < re) {
      next = stat_load(r0 + RT);
      stage(r0 + RT, buf ^ 1);
    }
    if (r0 < all_first) {                          // the diagonal
      mha_clean<DK, RT, 256, true>(smem + buf * TILES, threadIdx.x, &sm_bad[buf]);
      mha_clean<DV, RT, 256, true>(smem + buf * TILES + TQ, threadIdx.x, &sm_bad[buf]);
      __syncthreads();
      if (r0 + sm_bad[buf] >= mine) scale = __builtin_nanf("");
    }
    if (!some) continue;
    mha_lds_ptr qs = sm + buf * TILES, ds = qs + TQ;
#pragma unroll
    for (int n = 0; n < RT / 32; ++n) {
      __builtin_amdgcn_sched_barrier(0);      // one step's scores live at a time
      const int rs = r0 + n * 32;
      if (rs + 31 < wave_first || rs >= re) continue;
      // dP starts from -delta: the rows of an accumulator are 4 v / 4 + .. , four statistics a read
      f32x16_t dp;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4_t de = *reinterpret_cast<const f32x4_t*>(&stat[buf][1][n * 32 + 8 * g + 4 * half]);
#pragma unroll
        for (int j = 0; j < 4; ++j) dp[4 * g + j] = de[j];
      }
      f32x16_t s = mha_product<DK>(qs, rk, kf, n);
      if (mha_wider(DK, DV) > 64) __builtin_amdgcn_sched_barrier(0);
      if constexpr (V_LDS) {
        mha_lds_ptr vs = sm + 2 * TILES + wave * 64 * DV;
#pragma unroll
        for (int kd = 0; kd < DV / 16; ++kd) {
          const bf16x8_t x = *(mha_frag_ptr)(ds + rv.row[kd] + n * 64 * DV), y = *(mha_frag_ptr)(vs + rv.row[kd]);
          dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, dp, 0, 0, 0);
        }
      } else {
        dp = mha_product<DV>(ds, rv, vf, n, dp);
      }
      if (mha_wider(DK, DV) > 64) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4_t ls = *reinterpret_cast<const f32x4_t*>(&stat[buf][0][n * 32 + 8 * g + 4 * half]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int v = 4 * g + j;
          s[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], a.c, -ls[j]));
          dp[v] *= s[v];
        }
      }
      if (rs < wave_all) {
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const bool see = rs + mha_key(v, half) >= mine;
          s[v] = see ? s[v] : 0.f;
          dp[v] = see ? dp[v] : 0.f;
        }
      }
      if (mha_wider(DK, DV) > 64) __builtin_amdgcn_sched_barrier(0);
      mha_accumulate<DV>(dv, ds, rv, s, n);
      if (mha_wider(DK, DV) > 64) __builtin_amdgcn_sched_barrier(0);
      mha_accumulate<DK>(dk, qs, rk, dp, n);
    }
  }
  if (!ok) return;
  const float one = scale == scale ? 1.f : scale;
  if (it.part >= 0) {
    float* dst = a.ws_o + ((int64_t)it.part * KEY_TILE + key - it.row0) * (a.D + a.Dv);
    mha_store_part<DK>(dst, dk, a.D, half, one);
    mha_store_part<DV>(dst + a.D, dv, a.Dv, half, one);
    return;
  }
  bf16_t* dkp = a.dk + ((int64_t)(it.k_start + key) * a.kv_heads + it.hk) * a.D;
  bf16_t* dvp = a.dv + ((int64_t)(it.k_start + key) * a.kv_heads + it.hk) * a.Dv;
  auto store = [&](const f32x16_t& acc, int i, float f, bf16_t* dst, int width) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = i * 32 + g * 8 + 4 * half;
      const float w[4] = {acc[4 * g] * f, acc[4 * g + 1] * f, acc[4 * g + 2] * f, acc[4 * g + 3] * f};
      if (d < width) *reinterpret_cast<uint2*>(dst + d) = pack4_bf16(w);
    }
  };
#pragma unroll
  for (int i = 0; i < DK / 32; ++i) store(dk[i], i, scale, dkp, a.D);
#pragma unroll
  for (int i = 0; i < DV / 32; ++i) store(dv[i], i, one, dvp, a.Dv);
}

// sums the partial gradients of a split item in their order: item {seq, hk, row0, rows here, parts, first part},
// partial results [part][128][width]; dq: width D; dk and dv: D + Dv, the first D scaled.  Bound by reading them: 121 MB
// in 22 us (5.5 TB/s)
template <bool KEYS>
__global__ __launch_bounds__(256) void mha_join_grad_kernel(MhaArgs a) {
  const MhaItem it = mha_item(a, blockIdx.x);
  const int width = KEYS ? a.D + a.Dv : a.D, quads = width / 4;
  const int64_t step = (int64_t)ROW_TILE * width;
  for (int i = blockIdx.y * 256 + threadIdx.x; i < it.k0 * quads; i += gridDim.y * 256) {
    const int n = i / quads, d = (i - n * quads) * 4;
    const float* src = a.ws_o + ((int64_t)it.part * ROW_TILE + n) * width + d;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int p = 0; p < it.k1; ++p) {
      const float4 x = *reinterpret_cast<const float4*>(src + p * step);
      sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
    }
    const float f = d < a.D ? a.scale : 1.f;
    const float w[4] = {sum.x * f, sum.y * f, sum.z * f, sum.w * f};
    bf16_t* dst;
    if (KEYS) {
      const int64_t row = (int64_t)(it.k_start + it.row0 + n) * a.kv_heads + it.hk;
      dst = d < a.D ? a.dk + row * a.D + d : a.dv + row * a.Dv + (d - a.D);
    } else {
      int t, h;
      mha_token(a, it, it.row0 + n, &t, &h);
      dst = a.dq + ((int64_t)(it.q_start + t) * a.heads + h) * a.D + d;
    }
    *reinterpret_cast<uint2*>(dst) = pack4_bf16(w);
  }
}

// All gradients of a sequence with at most 32 rows and 32 keys: one wave a key head, nothing but its own Q, K, V
// and dO read.  The scores are formed both ways round (S^T for dQ, S for dK and dV); the softmax statistics and
// delta = sum_k P dP come from the scores themselves, exact in fp32, and reach the other orientation by lane
// exchanges.  Bound by latency: a launch of one wave workgroups, many a CU; 256 x 16 tokens, 8 heads of 64: 11 us (of
// which the bytes are 6).
template <int DK, int DV>
__global__ __launch_bounds__(64) void mha_bwd_small_kernel(MhaArgs a) {
  constexpr int TK = 32 * DK * 2;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * TK + 32 * DV * 2];   // K, Q, dO
  __shared__ int sm_bad[2];
  const int lane = threadIdx.x, half = lane >> 5, col = lane & 31;
  const MhaItem it = mha_item(a, blockIdx.x);
  const MhaReads<DK> rk = mha_reads<DK>(lane);
  const MhaReads<DV> rv = mha_reads<DV>(lane);
  const uint32_t lds = cg_lds_addr(smem);
  mha_lds_ptr ks = (mha_lds_ptr)smem, qs = ks + TK, ds = ks + 2 * TK;
  const int64_t dt = (int64_t)a.heads * a.Dv;
  {
    uint32_t koff[MhaStage<DK, 32, 1>::N];
    mha_offsets<DK, 32, 1>(koff, 0, lane, a.kt, a.D);
    mha_copy<DK, 32, 1>(koff, mha_rows<32>(a.k + (int64_t)it.hk * a.kh, it.k_start, it.Lk, a.kt, a.D), lds, 0);
    const cg_i32x4_t qr = cg_make_rsrc(a.q + (int64_t)it.hk * a.G * a.qh + (int64_t)it.q_start * a.qt, 0x7fffffffu);
    const cg_i32x4_t dr = cg_make_rsrc(a.dout + (int64_t)it.hk * a.G * a.Dv + (int64_t)it.q_start * dt, 0x7fffffffu);
    auto gather = [&](auto stage_of, const cg_i32x4_t& rs, int width, uint32_t row_bytes, uint32_t head_bytes,
                      uint32_t to) {
      using Stage = decltype(stage_of);
#pragma unroll
      for (int n = 0; n < Stage::N; ++n) {
        int r, c;
        Stage::place(n, 0, lane, &r, &c);
        const int t = (int)fdiv((uint32_t)r, a.dG), g = r - t * a.G;
        // rows that see no key are left out: their dO may hold anything
        const bool in = r < it.rows && t + it.shift >= 0 && c < width;
        cg_dma16_asm(rs, in ? (uint32_t)t * row_bytes + (uint32_t)g * head_bytes + c * 2 : OUTSIDE, 0u, to + n * 1024u);
      }
    };
    gather(MhaStage<DK, 32, 1>(), qr, a.D, (uint32_t)(a.qt * 2), (uint32_t)(a.qh * 2), lds + TK);
    gather(MhaStage<DV, 32, 1>(), dr, a.Dv, (uint32_t)(dt * 2), (uint32_t)(a.Dv * 2), lds + 2 * TK);
  }
  int t, h;
  mha_token(a, it, col, &t, &h);
  const bool row_ok = col < it.rows, key_ok = col < it.Lk;
  bf16x8_t vf[DV / 16];
  mha_row_frags(vf, a.v + (int64_t)(it.k_start + col) * a.vt + (int64_t)it.hk * a.vh, key_ok, a.Dv, half);
  if (lane < 2) sm_bad[lane] = lane ? -NONE_BAD : NONE_BAD;
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  bf16x8_t kf[DK / 16], qf[DK / 16], df[DV / 16];
#pragma unroll
  for (int kd = 0; kd < DK / 16; ++kd) {
    kf[kd] = *(mha_frag_ptr)(ks + rk.row[kd]);
    qf[kd] = *(mha_frag_ptr)(qs + rk.row[kd]);
  }
#pragma unroll
  for (int kd = 0; kd < DV / 16; ++kd) df[kd] = *(mha_frag_ptr)(ds + rv.row[kd]);
  int bad_key = NONE_BAD, bad_row = -NONE_BAD;
  if (a.causal) {       // (the scores above keep what is not finite: they are masked one by one)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    mha_clean<DK, 32, 64, false>(smem, lane, &sm_bad[0]);
    mha_clean<DK, 32, 64, true>(smem + TK, lane, &sm_bad[1]);
    mha_clean<DV, 32, 64, true>(smem + 2 * TK, lane, &sm_bad[1]);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    bad_key = *(volatile int*)&sm_bad[0];
    bad_row = *(volatile int*)&sm_bad[1];
  }
  auto product = [&](const auto& x, const auto& y) {
    f32x16_t s = mha_zero();
#pragma unroll
    for (size_t kd = 0; kd < sizeof(x) / sizeof(x[0]); ++kd)
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[kd], y[kd], s, 0, 0, 0);
    return s;
  };
  // rows in the lanes' columns: statistics, delta, dQ
  f32x16_t s = product(kf, qf);
  const f32x16_t dp = product(vf, df);
  const int last = row_ok ? min(it.Lk - 1, t + it.shift) : -1;
  float m = -INFINITY, l = 0.f, delta = 0.f;
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    s[v] = mha_key(v, half) <= last ? s[v] * a.c : -INFINITY;
    m = fmaxf(m, s[v]);
  }
  m = fmaxf(m, __shfl_xor(m, 32, 64));
  if (m == -INFINITY) m = 0.f;
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    s[v] = __builtin_amdgcn_exp2f(s[v] - m);
    l += s[v];
  }
  l += __shfl_xor(l, 32, 64);
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    s[v] *= inv;
    delta += mha_key(v, half) <= last ? s[v] * dp[v] : 0.f;
  }
  delta += __shfl_xor(delta, 32, 64);
#pragma unroll
  for (int v = 0; v < 16; ++v) s[v] = mha_key(v, half) <= last ? s[v] * (dp[v] - delta) : 0.f;
  auto finish = [&](auto& acc, mha_lds_ptr tile, const auto& reads, const f32x16_t& w, bf16_t* dst, bool ok, float f,
                    int width) {
    constexpr int N = sizeof(acc) / sizeof(acc[0]);
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = mha_zero();
    mha_accumulate<N * 32>(acc, tile, reads, w, 0);
    if (!ok) return;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = i * 32 + g * 8 + 4 * half;
        const float x[4] = {acc[i][4 * g] * f, acc[i][4 * g + 1] * f, acc[i][4 * g + 2] * f, acc[i][4 * g + 3] * f};
        if (d < width) *reinterpret_cast<uint2*>(dst + d) = pack4_bf16(x);
      }
  };
  f32x16_t acc_k[DK / 32], acc_v[DV / 32];
  finish(acc_k, ks, rk, s, a.dq + ((int64_t)(it.q_start + t) * a.heads + h) * a.D, row_ok,
         bad_key <= last ? __builtin_nanf("") : a.scale, a.D);
  // keys in the lanes' columns: dK, dV
  f32x16_t sk = product(qf, kf);
  f32x16_t dk = product(df, vf);
  const int mine = a.causal ? max(0, col - it.shift) * a.G : 0;    // first row that sees this key
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    const int r = mha_key(v, half);
    const float rm = __shfl(m, r, 64), ri = __shfl(inv, r, 64), rdelta = __shfl(delta, r, 64);
    const bool see = key_ok && r >= mine && r < it.rows;
    sk[v] = see ? __builtin_amdgcn_exp2f(__builtin_fmaf(sk[v], a.c, -rm)) * ri : 0.f;
    dk[v] = see ? sk[v] * (dk[v] - rdelta) : 0.f;
  }
  const int64_t key = (int64_t)(it.k_start + col) * a.kv_heads + it.hk;
  const float one = bad_row >= mine ? __builtin_nanf("") : 1.f;
  finish(acc_v, ds, rv, sk, a.dv + key * a.Dv, key_ok, one, a.Dv);
  finish(acc_k, qs, rk, dk, a.dk + key * a.D, key_ok, a.scale * one, a.D);
}

// ---- the plan ------------------------------------------------------------------------------------
struct Work {
  int32_t v[8];
  int64_t cost;
  int32_t unit;      // (sequence, key head): what shares K and V
};

// Longest first, and the tiles of one unit on one XCD (blocks go to the XCDs in turn) so that its keys stay in
// that XCD's L2: units are given to the least loaded XCD, with fewer units than XCDs each has several of them.
void mha_deal(std::vector<Work>* items, int units) {
  constexpr int X = 8;
  std::vector<Work>& w = *items;
  if (w.empty()) return;
  std::vector<int64_t> unit_cost(units, 0);
  for (const Work& i : w) unit_cost[i.unit] += i.cost;
  std::vector<int32_t> order(units);
  for (int u = 0; u < units; ++u) order[u] = u;
  std::stable_sort(order.begin(), order.end(), [&](int a, int b) { return unit_cost[a] > unit_cost[b]; });
  int live = 0;
  while (live < units && unit_cost[order[live]] > 0) ++live;
  if (live == 0) live = units;
  std::vector<int32_t> first(units, 0), count(units, 1), next(units, 0);
  if (live >= X) {
    int64_t load[X] = {0};
    for (int i = 0; i < units; ++i) {
      int best = 0;
      for (int x = 1; x < X; ++x)
        if (load[x] < load[best]) best = x;
      first[order[i]] = best;
      load[best] += unit_cost[order[i]] + 1;
    }
  } else {
    for (int i = 0; i < units; ++i) {
      first[order[i]] = i % live;
      count[order[i]] = (X - 1 - i % live) / live + 1;     // XCDs first, first + live, ...
    }
  }
  std::stable_sort(w.begin(), w.end(), [](const Work& a, const Work& b) { return a.cost > b.cost; });
  std::vector<Work> queue[X];
  for (const Work& i : w) {
    const int u = i.unit;
    queue[live >= X ? first[u] : first[u] + live * (next[u]++ % count[u])].push_back(i);
  }
  size_t at[X] = {0};
  for (size_t n = 0; n < w.size(); ++n) {
    int x = (int)(n % X);
    if (at[x] >= queue[x].size()) {            // an empty one helps where most is left
      for (int y = 0; y < X; ++y)
        if (queue[y].size() - at[y] > queue[x].size() - at[x]) x = y;
    }
    w[n] = queue[x][at[x]++];
  }
}

// A launch's items are split along the axis that they sum over (keys; rows for dK and dV) where one item is longer
// than its share of the launch.  A tile item's share is the total over 1536 (a third of what one of the chip's 512 places,
// 2 workgroups a CU, has to do: the longest items no longer delay the end; ragged training batch of 25 k rows, all its
// kernels: 790 us, over 1024 823 us, over 768 849 us, over 2048 794 us), but not below 1024 keys or rows where the total
// over 512 is more (a part's fp32 result, written once and read once, has to be small against its work: 8 causal sequences
// of 4096, 2 key heads of 128 with 4 query heads each, forward 294 us and over 2048 335 us; one sequence of 8192, 2 heads
// of 128, causal: backward 206 us, in parts of 512 rows 231 us), and not below 512 at all.  Thin items have no tile of 128
// rows and no part of 1024 keys to lose.
constexpr int THIN1_KEYS = 128;     // up to so many keys one wave does a thin item alone

int64_t mha_share(int64_t all, bool thin) {
  const int64_t most = (all + 511) / 512, third = (all + 1535) / 1536;
  return std::max<int64_t>(512, thin ? third : std::min(most, std::max<int64_t>(1024, third)));
}

void mha_split(std::vector<Work>* items, int step, int tile, int units_a_part, const std::vector<int64_t>& length,
               std::vector<Work>* joins, int64_t* parts) {
  int64_t all = 0;
  for (const Work& w : *items) all += w.v[4] - w.v[3];
  const int64_t chunk = mha_share(all, tile == THIN_ROWS);
  std::vector<Work> out;
  for (const Work& w : *items) {
    const int64_t len = w.v[4] - w.v[3], steps = (len + step - 1) / step;
    const int64_t n = (len + chunk / 2) / chunk;
    if (n <= 1) {
      out.push_back(w);
      continue;
    }
    Work j = w;
    j.v[3] = (int32_t)std::min<int64_t>(tile, length[w.v[0]] - w.v[2]);
    j.v[4] = (int32_t)n;
    j.v[5] = (int32_t)*parts;
    j.v[6] = units_a_part;
    joins->push_back(j);
    for (int64_t i = 0; i < n; ++i) {
      Work p = w;
      p.v[3] = w.v[3] + (int32_t)(steps * i / n) * step;
      p.v[4] = (int32_t)std::min<int64_t>(w.v[4], w.v[3] + steps * (i + 1) / n * step);
      p.v[5] = (int32_t)*parts;
      p.cost = p.v[4] - p.v[3] + 64;
      *parts += units_a_part;
      out.push_back(p);
    }
  }
  items->swap(out);
}

// Up to so many items of a one wave form (one a CU) go into the launch of a wider form if there is one anyway: they fill
// its end, and a launch of their own is 7 to 10 us (48 new tokens, a few of them with up to 128 keys: 177 -> 168 us;
// ragged training batch: 793 -> 776 us; two causal sequences of 2048 with 32, 128 or 256 one wave units beside them:
// forward 41, 39, 39 -> 34, 32, 32 us, backward 88, 83, 83 -> 80, 76, 74 us).
constexpr int FOLD = 256;

int mha_plan(const int32_t* q_start, const int32_t* q_len, const int32_t* k_start, const int32_t* k_len,
             int B, int heads, int kv_heads, int causal, int32_t* data, int64_t capacity, cgAttentionPlan* info) {
  const int G = heads / kv_heads;
  int64_t few = 0;           // units for the small form of the backward pass, and whether there are others
  bool others = false;
  for (int b = 0; b < B; ++b) {
    const bool fits = (int64_t)q_len[b] * G <= 32 && k_len[b] <= 32;
    if (!fits) others = true;
    else if (q_len[b] > 0 || k_len[b] > 0) few += kv_heads;
  }
  const bool small_form = !others || few > FOLD;
  std::vector<Work> tiles, thin4, thin1, joins, dq, dq_joins, dkv, dkv_joins, small;
  std::vector<int64_t> all_rows(B), all_keys(B);
  cgAttentionPlan p = {};
  for (int b = 0; b < B; ++b) {
    const int64_t Lq = q_len[b], Lk = k_len[b], rows = Lq * G, shift = Lk - Lq;
    if (Lq > 0) p.max_q_row = std::max<int32_t>(p.max_q_row, (int32_t)(q_start[b] + Lq));
    if (Lk > 0) p.max_k_row = std::max<int32_t>(p.max_k_row, (int32_t)(k_start[b] + Lk));
    all_rows[b] = rows;
    all_keys[b] = Lk;
    auto keys_of = [&](int64_t end_row) {     // keys that the rows below end_row see
      if (!causal) return Lk;
      return std::min(Lk, std::max<int64_t>(0, (end_row - 1) / G + shift + 1));
    };
    for (int h = 0; h < kv_heads; ++h) {
      const int32_t unit = b * kv_heads + h;
      for (int64_t r = 0; r < rows; r += ROW_TILE) {
        const int64_t keys = keys_of(std::min(rows, r + ROW_TILE));
        Work w = {{b, h, (int32_t)r, 0, (int32_t)keys, -1, 0, 0}, keys + 64, unit};
        if (rows > 32 || Lk > 32 || !small_form) dq.push_back(w);
        if (rows > THIN_ROWS) tiles.push_back(w);
        else (keys <= THIN1_KEYS ? thin1 : thin4).push_back(w);
      }
      if (rows <= 32 && Lk <= 32 && small_form) {
        if (rows > 0 || Lk > 0) small.push_back(Work{{b, h, 0, 0, (int32_t)Lk, -1, 0, 0}, 1, unit});
        continue;
      }
      for (int64_t k = 0; k < Lk; k += KEY_TILE) {
        const int64_t from = causal ? std::min(rows, std::max<int64_t>(0, k - shift) * G) : 0;
        dkv.push_back(Work{{b, h, (int32_t)k, (int32_t)from, (int32_t)rows, -1, 0, 0}, rows - from + 64, unit});
      }
    }
  }
  if ((int64_t)thin1.size() <= FOLD && (!thin4.empty() || !tiles.empty())) {
    std::vector<Work>& wider = thin4.empty() ? tiles : thin4;
    wider.insert(wider.end(), thin1.begin(), thin1.end());
    thin1.clear();
  }
  int64_t parts = 0, dq_parts = 0, dkv_parts = 0;
  mha_split(&tiles, KT, ROW_TILE, ROW_TILE / 32, all_rows, &joins, &parts);
  mha_split(&thin4, 32, THIN_ROWS, 1, all_rows, &joins, &parts);
  mha_split(&dq, KT, ROW_TILE, 1, all_rows, &dq_joins, &dq_parts);
  mha_split(&dkv, KT, KEY_TILE, 1, all_keys, &dkv_joins, &dkv_parts);
  if (parts > 0x7fffffff || dq_parts > 0x7fffffff || dkv_parts > 0x7fffffff) CG_FAIL(CG_ERR_UNSUPPORTED, "cg_host_attention_plan: too many partial results");
  const int units = B * kv_heads;
  std::vector<Work>* lists[9] = {&tiles, &thin4, &thin1, &joins, &dq, &dq_joins, &dkv, &dkv_joins, &small};
  int64_t ints = 4 * (int64_t)B;
  for (auto* l : lists) ints += 8 * (int64_t)l->size();
  if (ints > 0x7fffffff) CG_FAIL(CG_ERR_UNSUPPORTED, "cg_host_attention_plan: too many work items");
  p.ints = ints;
  p.parts = parts;
  p.sequences = B;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.causal = causal ? 1 : 0;
  p.tiles = (int32_t)tiles.size();
  p.thin4 = (int32_t)thin4.size();
  p.thin1 = (int32_t)thin1.size();
  p.joins = (int32_t)joins.size();
  p.dq_tiles = (int32_t)dq.size();
  p.dkv_tiles = (int32_t)dkv.size();
  p.dq_joins = (int32_t)dq_joins.size();
  p.dkv_joins = (int32_t)dkv_joins.size();
  p.small = (int32_t)small.size();
  p.dq_parts = dq_parts;
  p.dkv_parts = dkv_parts;
  *info = p;
  if (!data) return CG_OK;
  if (capacity < ints) CG_FAIL(CG_ERR_WORKSPACE, "cg_host_attention_plan: %lld ints of %lld", (long long)capacity, (long long)ints);
  for (int b = 0; b < B; ++b) {
    const int32_t s[4] = {q_start[b], q_len[b], k_start[b], k_len[b]};
    memcpy(data + 4 * (int64_t)b, s, sizeof(s));
  }
  int32_t* at = data + 4 * (int64_t)B;
  for (auto* l : lists) {
    if (l != &joins && l != &dq_joins && l != &dkv_joins) mha_deal(l, units);
    for (const Work& w : *l) {
      memcpy(at, w.v, sizeof(w.v));
      at += 8;
    }
  }
  return CG_OK;
}

int mha_check(const char* name, const cgAttentionInput* in, const cgAttentionPlan* p, const int32_t* data, MhaArgs* a) {
  if (!in || !p || !data) CG_FAIL(CG_ERR_BAD_ARG, "%s: null input or plan", name);
  if (p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads || p->ints < 1)
    CG_FAIL(CG_ERR_BAD_ARG, "%s: not a plan of cg_host_attention_plan", name);
  if (in->D < 8 || in->D > 128 || in->D % 8 || in->Dv < 8 || in->Dv > 128 || in->Dv % 8)
    CG_FAIL(CG_ERR_UNSUPPORTED, "%s: head widths %d and %d (multiples of 8, at most 128)", name, in->D, in->Dv);
  if (!(in->scale >= 0.99e-30f && in->scale <= 1.01e30f)) CG_FAIL(CG_ERR_BAD_ARG, "%s: scale has to be in [1e-30, 1e30]", name);
  if (in->q_rows < p->max_q_row || in->k_rows < p->max_k_row)
    CG_FAIL(CG_ERR_BAD_ARG, "%s: %d query and %d key rows, the plan's sequences need %d and %d", name, in->q_rows,
            in->k_rows, p->max_q_row, p->max_k_row);
  const int64_t G = p->heads / p->kv_heads;
  const int64_t st[6] = {in->q_stride_t, in->q_stride_h, in->k_stride_t, in->k_stride_h, in->v_stride_t, in->v_stride_h};
  for (int i = 0; i < 6; ++i)
    if (st[i] < 0 || st[i] % 8) CG_FAIL(CG_ERR_UNSUPPORTED, "%s: strides have to be multiples of 8 elements", name);
  for (int i = 0; i < 6; ++i)     // (no tensor is that long; the products below and the kernels' offsets stay in 64 bits)
    if (st[i] > (1ll << 40)) CG_FAIL(CG_ERR_UNSUPPORTED, "%s: strides too large", name);
  if ((uintptr_t)data % 16) CG_FAIL(CG_ERR_UNSUPPORTED, "%s: the plan has to be 16-byte aligned", name);
  const void* ptr[3] = {in->q, in->k, in->v};
  for (int i = 0; i < 3; ++i) {
    // (no keys at all: K and V may be null, no work item reads them)
    if (!ptr[i] && (i == 0 ? p->max_q_row : p->max_k_row) > 0) CG_FAIL(CG_ERR_BAD_ARG, "%s: null tensor", name);
    if ((uintptr_t)ptr[i] % 16) CG_FAIL(CG_ERR_UNSUPPORTED, "%s: tensors have to be 16-byte aligned", name);
  }
  // a tile's byte offsets are 32-bit (its base is 64-bit): up to 128 rows, and the shared heads of one
  if ((int64_t)KEY_TILE * 2 * std::max(std::max(st[0], st[2]), st[4]) + 2 * G * st[1] >= 0x7fffff00ll ||
      (int64_t)KT * 2 * p->heads * 128 >= 0x3fffff00ll)
    CG_FAIL(CG_ERR_UNSUPPORTED, "%s: strides too large", name);
  a->q = (const bf16_t*)in->q;
  a->k = (const bf16_t*)in->k;
  a->v = (const bf16_t*)in->v;
  a->qt = st[0]; a->qh = st[1]; a->kt = st[2]; a->kh = st[3]; a->vt = st[4]; a->vh = st[5];
  a->seqs = (const int4*)data;
  a->heads = p->heads;
  a->kv_heads = p->kv_heads;
  a->G = (int)G;
  a->dG = make_fastdiv((uint32_t)G);
  a->D = in->D;
  a->Dv = in->Dv;
  a->causal = p->causal;
  a->scale = in->scale;
  a->c = in->scale * LOG2E;
  return CG_OK;
}

// item lists behind the sequences
const int4* mha_list(const cgAttentionPlan* p, const int32_t* data, int which) {
  const int64_t n[9] = {p->tiles, p->thin4, p->thin1, p->joins, p->dq_tiles, p->dq_joins, p->dkv_tiles, p->dkv_joins,
                        p->small};
  int64_t at = 4 * (int64_t)p->sequences;
  for (int i = 0; i < which; ++i) at += 8 * n[i];
  return (const int4*)(data + at);
}

// padded head width
int mha_width(int D) { return (D + 31) / 32 * 32; }

}  // namespace

// the kernel of the two padded head widths
#define MHA_LAUNCH_DV(dk, dv, kernel, grid, block, st, args)                   \
  switch (dv) {                                                                \
    case 32: kernel(dk, 32)<<<grid, block, 0, st>>>(args); break;              \
    case 64: kernel(dk, 64)<<<grid, block, 0, st>>>(args); break;              \
    case 96: kernel(dk, 96)<<<grid, block, 0, st>>>(args); break;              \
    default: kernel(dk, 128)<<<grid, block, 0, st>>>(args); break;             \
  }
#define MHA_LAUNCH(dk, dv, kernel, grid, block, st, args)                      \
  switch (dk) {                                                                \
    case 32: MHA_LAUNCH_DV(32, dv, kernel, grid, block, st, args) break;       \
    case 64: MHA_LAUNCH_DV(64, dv, kernel, grid, block, st, args) break;       \
    case 96: MHA_LAUNCH_DV(96, dv, kernel, grid, block, st, args) break;       \
    default: MHA_LAUNCH_DV(128, dv, kernel, grid, block, st, args) break;      \
  }
#define MHA_FWD(dk, dv) mha_fwd_kernel<dk, dv, false>
#define MHA_THIN4(dk, dv) mha_thin_kernel<dk, dv, 4, false>
#define MHA_THIN1(dk, dv) mha_thin_kernel<dk, dv, 1, false>
#define MHA_FWD_GRAD(dk, dv) mha_fwd_kernel<dk, dv, true>
#define MHA_THIN4_GRAD(dk, dv) mha_thin_kernel<dk, dv, 4, true>
#define MHA_THIN1_GRAD(dk, dv) mha_thin_kernel<dk, dv, 1, true>
#define MHA_BWD_Q(dk, dv) mha_bwd_q_kernel<dk, dv>
// (96 with 128 would spill like 128 with 128 does without V in LDS: padded to it)
#define MHA_BWD_KV(dk, dv) mha_bwd_kv_kernel<(dk + dv == 224 ? 128 : dk), (dk + dv == 224 ? 128 : dv)>
#define MHA_BWD_SMALL(dk, dv) mha_bwd_small_kernel<dk, dv>

extern "C" int cg_host_attention_plan(const int32_t* q_start, const int32_t* q_len, const int32_t* k_start,
                                      const int32_t* k_len, int sequences, int heads, int kv_heads, int causal,
                                      int32_t* data_host, int64_t capacity, cgAttentionPlan* info) {
  const char* name = "cg_host_attention_plan";
  if (!q_start || !q_len || !k_start || !k_len || !info) CG_FAIL(CG_ERR_BAD_ARG, "%s: null argument", name);
  if (sequences < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || heads > 4096)
    CG_FAIL(CG_ERR_BAD_ARG, "%s: %d sequences, %d heads over %d", name, sequences, heads, kv_heads);
  const int64_t G = heads / kv_heads;
  if ((int64_t)sequences * kv_heads > 0x3fffffff) CG_FAIL(CG_ERR_UNSUPPORTED, "%s: too many sequences", name);
  for (int b = 0; b < sequences; ++b) {
    if (q_start[b] < 0 || q_len[b] < 0 || k_start[b] < 0 || k_len[b] < 0)
      CG_FAIL(CG_ERR_BAD_ARG, "%s: sequence %d has a negative start or length", name, b);
    if ((int64_t)q_len[b] * G > 0x3fffffff || (int64_t)q_start[b] + q_len[b] > 0x3fffffff ||
        (int64_t)k_start[b] + k_len[b] > 0x3fffffff)
      CG_FAIL(CG_ERR_UNSUPPORTED, "%s: sequence %d is too long", name, b);
  }
  try {
    return mha_plan(q_start, q_len, k_start, k_len, sequences, heads, kv_heads, causal, data_host, capacity, info);
  } catch (const std::bad_alloc&) {
    CG_FAIL(CG_ERR_WORKSPACE, "%s: out of host memory", name);
  } catch (...) {
    CG_FAIL(CG_ERR_BAD_ARG, "%s: failed", name);
  }
}

extern "C" size_t cg_packed_attention_fwd_workspace_bytes(const cgAttentionPlan* plan, int Dv) {
  if (!plan || Dv < 1) return 0;
  return (size_t)plan->parts * THIN_ROWS * ((size_t)Dv + 2) * sizeof(float);
}

extern "C" int cg_packed_attention_fwd(const cgAttentionInput* in, const cgAttentionPlan* plan, const int32_t* data,
                                       void* out, void* out_low, float* lse, void* ws, size_t ws_bytes,
                                       cgStream stream) {
  const char* name = "cg_packed_attention_fwd";
  MhaArgs a = {};
  const int rc = mha_check(name, in, plan, data, &a);
  if (rc) return rc;
  if (plan->max_q_row == 0) return CG_OK;
  if (!out) CG_FAIL(CG_ERR_BAD_ARG, "%s: null output", name);
  if ((uintptr_t)out % 16 || (uintptr_t)out_low % 16 || (uintptr_t)ws % 16) CG_FAIL(CG_ERR_UNSUPPORTED, "%s: tensors and workspace have to be 16-byte aligned", name);
  if (plan->parts > 0 && (!ws || ws_bytes < cg_packed_attention_fwd_workspace_bytes(plan, in->Dv)))
    CG_FAIL(CG_ERR_WORKSPACE, "%s: workspace of %zu bytes", name, ws_bytes);
  a.out = (bf16_t*)out;
  a.out_low = (bf16_t*)out_low;
  a.lse = lse;
  a.ws_o = (float*)ws;
  a.ws_ml = a.ws_o + plan->parts * THIN_ROWS * (int64_t)in->Dv;
  const hipStream_t st = (hipStream_t)stream;
  const int dkp = mha_width(in->D), dvp = mha_width(in->Dv);
  if (plan->tiles) {
    a.items = mha_list(plan, data, 0);
    if (out_low) {
      MHA_LAUNCH(dkp, dvp, MHA_FWD_GRAD, plan->tiles, 256, st, a);
    } else {
      MHA_LAUNCH(dkp, dvp, MHA_FWD, plan->tiles, 256, st, a);
    }
    CG_CHECK_LAUNCH(name);
  }
  if (plan->thin4) {
    a.items = mha_list(plan, data, 1);
    if (out_low) {
      MHA_LAUNCH(dkp, dvp, MHA_THIN4_GRAD, plan->thin4, 256, st, a);
    } else {
      MHA_LAUNCH(dkp, dvp, MHA_THIN4, plan->thin4, 256, st, a);
    }
    CG_CHECK_LAUNCH(name);
  }
  if (plan->thin1) {
    a.items = mha_list(plan, data, 2);
    if (out_low) {
      MHA_LAUNCH(dkp, dvp, MHA_THIN1_GRAD, plan->thin1, 64, st, a);
    } else {
      MHA_LAUNCH(dkp, dvp, MHA_THIN1, plan->thin1, 64, st, a);
    }
    CG_CHECK_LAUNCH(name);
  }
  if (plan->joins) {
    a.items = mha_list(plan, data, 3);
    // a thousand blocks and more (few items: fewer rows a block), at most one for each row of an item
    const int each = std::min(plan->tiles ? ROW_TILE : THIN_ROWS, std::max(plan->tiles ? 8 : 1, 1024 / plan->joins));
    mha_join_kernel<<<dim3(plan->joins, each), 256, 0, st>>>(a);
    CG_CHECK_LAUNCH(name);
  }
  return CG_OK;
}

// workspace: delta [q_rows, heads], then the partial results of dq, then (the same memory) of dk and dv
static int64_t mha_delta_bytes(const cgAttentionPlan* p, int q_rows) {
  return ((int64_t)q_rows * p->heads * (int64_t)sizeof(float) + 255) / 256 * 256;
}

extern "C" size_t cg_packed_attention_bwd_workspace_bytes(const cgAttentionPlan* plan, int q_rows, int D, int Dv) {
  if (!plan || q_rows < 1 || D < 1 || Dv < 1 || plan->dq_tiles + plan->dkv_tiles == 0) return 0;
  const int64_t a = plan->dq_parts * D, b = plan->dkv_parts * (D + Dv);
  return (size_t)(mha_delta_bytes(plan, q_rows) + (a > b ? a : b) * ROW_TILE * (int64_t)sizeof(float));
}

extern "C" int cg_packed_attention_bwd(const cgAttentionInput* in, const cgAttentionPlan* plan, const int32_t* data,
                                       const void* out, const void* out_low, const float* lse, const void* dout,
                                       void* dq, void* dk, void* dv, void* ws, size_t ws_bytes, cgStream stream) {
  const char* name = "cg_packed_attention_bwd";
  MhaArgs a = {};
  const int rc = mha_check(name, in, plan, data, &a);
  if (rc) return rc;
  if (plan->max_q_row > 0) {
    if (!out || !lse || !dout || !dq || (plan->dq_tiles && !out_low)) CG_FAIL(CG_ERR_BAD_ARG, "%s: null tensor", name);
    const size_t need = cg_packed_attention_bwd_workspace_bytes(plan, in->q_rows, in->D, in->Dv);
    if (need > 0 && (!ws || ws_bytes < need))
      CG_FAIL(CG_ERR_WORKSPACE, "%s: workspace of %zu bytes", name, ws_bytes);
  }
  if (plan->max_k_row > 0 && (!dk || !dv)) CG_FAIL(CG_ERR_BAD_ARG, "%s: null gradient", name);
  const void* ptr[7] = {out, out_low, dout, dq, dk, dv, ws};
  for (const void* p : ptr)
    if ((uintptr_t)p % 16) CG_FAIL(CG_ERR_UNSUPPORTED, "%s: tensors have to be 16-byte aligned", name);
  a.lse_in = lse;
  a.dout = (const bf16_t*)dout;
  a.dq = (bf16_t*)dq;
  a.dk = (bf16_t*)dk;
  a.dv = (bf16_t*)dv;
  a.o_in = (const bf16_t*)out;
  a.o_low = (const bf16_t*)out_low;
  a.delta = (float*)ws;
  if (ws) a.ws_o = (float*)((char*)ws + mha_delta_bytes(plan, in->q_rows));
  const hipStream_t st = (hipStream_t)stream;
  const int dkp = mha_width(in->D), dvp = mha_width(in->Dv);
  if (plan->dq_tiles) {
    a.items = mha_list(plan, data, 4);
    MHA_LAUNCH(dkp, dvp, MHA_BWD_Q, plan->dq_tiles, 256, st, a);
    CG_CHECK_LAUNCH(name);
  }
  if (plan->dq_joins) {
    a.items = mha_list(plan, data, 5);
    mha_join_grad_kernel<false><<<dim3(plan->dq_joins, 16), 256, 0, st>>>(a);
    CG_CHECK_LAUNCH(name);
  }
  if (plan->dkv_tiles) {
    a.items = mha_list(plan, data, 6);
    MHA_LAUNCH(dkp, dvp, MHA_BWD_KV, plan->dkv_tiles, 256, st, a);
    CG_CHECK_LAUNCH(name);
  }
  if (plan->dkv_joins) {
    a.items = mha_list(plan, data, 7);
    mha_join_grad_kernel<true><<<dim3(plan->dkv_joins, 16), 256, 0, st>>>(a);
    CG_CHECK_LAUNCH(name);
  }
  if (plan->small) {
    a.items = mha_list(plan, data, 8);
    MHA_LAUNCH(dkp, dvp, MHA_BWD_SMALL, plan->small, 64, st, a);
    CG_CHECK_LAUNCH(name);
  }
  return CG_OK;
}
