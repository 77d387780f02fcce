// Attention with a learned bias per (bucket of the key-query distance, head): forward, and the backward that recomputes
// the probabilities.  The formulas are in include/csship.h (csship_relbias).
//
// Matrix products are v_mfma_f32_32x32x16 (lane l of an operand: row l & 31, eight k values 8 (l >> 5) ..; accumulator register
// r of lane l: row 8 (r >> 2) + 4 (l >> 5) + (r & 3), column l & 31).  Scores are computed TRANSPOSED where the queries are
// what a wave owns, S^T[key, query] = K Q^T: a lane then holds one query and four consecutive keys per register group, so
//   * row maxima and sums are register sums plus ONE exchange between the two half waves;
//   * the rounded probabilities are already the B operand of the next product: its reduction index may run over the keys in
//     any order as long as both operands agree, and register group order (keys 4 hi .. + 3, 8 + 4 hi .. + 3) is the order in
//     which two ds_read_b64_tr_b16 deliver V^T;
//   * the bias of the four keys is four consecutive floats of the head's table, spread over distances once per workgroup in
//     LDS, and goes into the product as its initial accumulator: no addition per score.  Tiles wholly beyond the largest
//     distance start from a constant.
#include "common.hpp"

namespace {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) f32x4 lds_f32x4;

constexpr float RB_LOG2E = 1.4426950408889634f, RB_LN2 = 0.6931471805599453f;
constexpr int RB_PAD = 96;          // entries of the spread table beyond the largest distance on each side: a 64 x 32 tile that
                                    // is not wholly beyond it reaches at most 64 + 32 - 2 further
constexpr float RB_BIG = 1048576.f; // table entries at or below -2^20 ban their distances; entries above 2^20 count as 2^20
constexpr int SPAN_MAX = 2 * (CSSHIP_RELBIAS_MAX_DISTANCE + RB_PAD) + 1;
constexpr int RB_MAX_POS = 1 << 28;  // lengths and offsets stay below it: distances in 32 bits
constexpr float RB_INF = __builtin_inff();

template <int N>
struct Const { static constexpr int value = N; };
using True = Const<1>;
using False = Const<0>;

struct ElemBf {
  static constexpr bool narrow = false;  // exponents as wide as f32's
  static constexpr float up = 0.f, grow = 8.f;  // forward, log2: P of the reference, and how far a score may outgrow it
  DEV f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  DEV unsigned pack(float lo, float hi) { return pack_bf2(lo, hi); }
  DEV float lo(unsigned u) { return __uint_as_float(u << 16); }
  DEV float hi(unsigned u) { return __uint_as_float(u & 0xffff0000u); }
};
// fp16 reaches from 2^-24 to 2^16 only.  In the forward P is 2^7 at a row's reference and up to 2^14 (2^16 if the exponents of scores of
// 2^24 are off by a step): what rounds to zero is below 2^-32 of the reference, rows of one large and thousands of small P keep
// the latter.  In the backward dS has the size of dout v / Tk, which may be anything, and a key may have little of every row's P: both are
// multiplied by a power of two before they are rounded, and the sums are divided by it (fit).
struct ElemHf {
  static constexpr bool narrow = true;
  static constexpr float up = 7.f, grow = 7.f;
  DEV f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  DEV unsigned pack(float lo, float hi) {
    const f32x2_cvt f = {lo, hi};
    return __builtin_bit_cast(unsigned, __builtin_convertvector(f, f16x2));
  }
  DEV float lo(unsigned u) { return (float)__builtin_bit_cast(f16x2, u)[0]; }
  DEV float hi(unsigned u) { return (float)__builtin_bit_cast(f16x2, u)[1]; }
};

struct Strides { int64_t b, t, h; };  // elements

// division of 0 <= n < 2^31 by a number known on the host: n mul >> shift, exact (mul = ceil(2^shift / d), shift = 31 + ceil(log2 d))
struct Divisor {
  unsigned mul, shift;
  int d;
  void set(int by) {
    d = by;
    shift = 31;
    while ((1ll << (shift - 31)) < by) ++shift;
    mul = (unsigned)(((1ull << shift) + (unsigned)by - 1) / (unsigned)by);
  }
  __device__ __forceinline__ int over(int n) const { return (int)(((uint64_t)(unsigned)n * mul) >> shift); }
};
struct Quot { int q, r; };
DEV Quot split(int n, const Divisor& d) {
  const int q = d.over(n);
  return Quot{q, n - q * d.d};
}

struct RbArgs {
  Divisor per_tile, per_head, per_group, per_split;  // ntile; H or Hk, as the kernel counts; H / Hk; nsplit
  const uint16_t *q, *k, *v, *o, *dout;
  Strides sq, sk, sv, so, sdo, sdq, sdk, sdv;
  const float* table;
  const int16_t* bucket_of;
  const int32_t* bucket_range;
  const int32_t *k_lens, *q_lens, *offsets;
  uint16_t *out, *dq, *dk, *dv;
  float *lse, *dtable;
  const float* lse_in;
  float *delta, *lse2, *part, *part2;  // workspace; delta (negated), lse2 [B, H, tq128]
  int B, Tq, Tk, H, Hk, D, nb, md, mde, causal, offset;  // mde: md, or the furthest distance that occurs
  float scale, inv_scale, c2;  // c2 = scale * log2(e)
  int ntile, nblk, nsplit, nqtile, tq128;     // row tiles per (sequence, head); workgroups; key ranges (rb_few_kernel)
};

// rows of 2 DP bytes in 16-byte pieces; piece c of row r lies at piece c ^ swz(r).  The key makes both kinds of reads spread over
// the banks: 16 rows at one piece (ds_read_b128 operands) and 8 rows at four neighbouring pieces (the transposing reads).
template <int DP>
DEV int swz(int r) {
  if constexpr (DP == 128) return ((r & 3) << 2) | ((r >> 2) & 3);
  else if constexpr (DP == 64) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
  else return (r >> 2) & 3;
}
template <int DP>
DEV int tile_at(int r, int c) { return r * (2 * DP) + ((c ^ swz<DP>(r)) << 4); }

// the sequence's lengths and query offset; values outside the tensors' extents are cut to them.  Keys behind the last query's
// position are seen by none under `causal` and count as behind the sequence's end: a cache may hold anything there.
struct Seq { int qlen, klen, off; };
DEV Seq seq_of(const RbArgs& a, int b) {
  Seq s;
  s.klen = a.k_lens ? min(max(a.k_lens[b], 0), a.Tk) : a.Tk;
  s.qlen = a.q_lens ? min(max(a.q_lens[b], 0), a.Tq) : a.Tq;
  s.off = min(max(a.offsets ? a.offsets[b] : a.offset, -RB_MAX_POS), RB_MAX_POS);
  if (a.causal) s.klen = min(s.klen, max(s.off + s.qlen, 0));
  return s;
}

// workgroup -> (sequence, head, row tile): workgroups go to the 8 XCDs in turn; neighbours in (sequence, key head) share K and V
// and are put on one XCD, so that they meet in its L2
DEV int xcd_order(int id, int n) {
  const int x = id & 7, i = id >> 3, full = n >> 3, rest = n & 7;
  return x * full + min(x, rest) + i;
}

// The tile and key or query range of a workgroup.  Under `causal` tiles differ in length and the longest come first.  A CU that
// takes one of an XCD's first 32 workgroups gets one of its next 32 as well, and both sit on it at once: every second 32 are
// taken in reverse, within each head, so that a long one meets a short one (2 x 2047, 16 heads: forward 66 -> 55 us).
struct Place { int head, rank, part; };  // (sequence, head); tile counted from the longest
DEV Place place_of(const RbArgs& a) {
  const int n = a.nblk, x = blockIdx.x & 7, i = blockIdx.x >> 3, id = xcd_order(blockIdx.x, n), base = id - i;
  const int head = a.per_tile.over(a.per_split.over(id)), first = head * a.ntile * a.nsplit, last = first + a.ntile * a.nsplit;
  int r = id;
  if (a.causal && (i & 32)) r = max(first, base + (i & ~31)) + min(last, base + min((i | 31) + 1, (n >> 3) + (x < (n & 7)))) - 1 - id;
  const Quot q = split(r - first, a.per_split);
  return Place{head, q.q, q.r};
}

// table entry -> score units (the products' accumulators hold q . k, scaled later by c2)
DEV float bias_units(const RbArgs& a, float w) { return w <= -RB_BIG ? -RB_INF : (w > RB_BIG ? RB_BIG : w) * a.inv_scale; }
DEV float bias_entry(const RbArgs& a, int r, int h) { return bias_units(a, a.table[a.bucket_of[r + a.md] * a.H + h]); }
// A head's table by distance, -mde - RB_PAD .. mde + RB_PAD, in LDS; 256 threads, barriers inside.  The table's column goes
// through `scratch` (`cap` floats), so that it and the bucket numbers are loaded side by side and not one behind the other.
DEV void spread_table(const RbArgs& a, int h, float* sB, float* scratch, int cap, int tid) {
  const int n = 2 * (a.mde + RB_PAD) + 1;
  const bool staged = a.nb <= cap;
  if (staged)
    for (int i = tid; i < a.nb; i += 256) scratch[i] = bias_units(a, a.table[i * a.H + h]);
  constexpr int AHEAD = 4;
  int id[AHEAD];
#pragma unroll
  for (int e = 0; e < AHEAD; ++e) {
    const int i = tid + e * 256;
    id[e] = i < n ? a.bucket_of[min(max(i - a.mde - RB_PAD, -a.mde), a.mde) + a.md] : 0;
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < AHEAD; ++e) {
    const int i = tid + e * 256;
    if (i < n) sB[i] = staged ? scratch[id[e]] : bias_units(a, a.table[id[e] * a.H + h]);
  }
  for (int i = tid + AHEAD * 256; i < n; i += 256) {
    const int x = a.bucket_of[min(max(i - a.mde - RB_PAD, -a.mde), a.mde) + a.md];
    sB[i] = staged ? scratch[x] : bias_units(a, a.table[x * a.H + h]);
  }
}

// over the two half waves (lanes l and l ^ 32), in both
DEV float half_max(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const unsigned a0 = r[0], a1 = r[1];
  return fmaxf(__uint_as_float(a0), __uint_as_float(a1));
}
DEV float half_sum(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const unsigned a0 = r[0], a1 = r[1];
  return __uint_as_float(a0) + __uint_as_float(a1);
}

// fp16: the values that a lane rounds for its column of a sum are multiplied by a power of two, `fac`, which starts as large as the
// products allow (|dS| < 2^40: 2^120 in f32) and goes down, the sum with it, whenever a value x (multiplied already) reaches
// 2^15: the largest is then in 2^9 .. 2^10.  So nothing overflows, and from 2^-23 of the column's largest value on, all keep
// 11 bits; what is smaller is off by at most 2^-34 of that largest one.  Both half waves hold the same columns.
constexpr float RB_FAC0 = 0x1p80f;
template <int ND>
DEV void fit(f32x16& x, f32x16 (&sum)[ND], float& fac) {
  float top = fabsf(x[0]);
#pragma unroll
  for (int r = 1; r < 16; ++r) top = fmaxf(top, fabsf(x[r]));
  top = half_max(top);
  if (__any(top >= 32768.f)) {
    const float down = top >= 32768.f ? __builtin_ldexpf(1.f, 9 + 127 - (int)(__float_as_uint(top) >> 23)) : 1.f;
    fac *= down;
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] *= down;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) sum[d][r] *= down;
  }
}
DEV double wave_total(double x) {
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) x += __shfl_xor(x, w);
  return x;
}

// ---- tiles of ROWS rows of a [T, heads, D] tensor, memory -> LDS without passing registers (buffer_load_dwordx4 ... lds): one
// instruction of a wave fills 1 KB in lane order, so the swizzle is applied to the address each lane fetches.  Rows at or behind
// `rows` and pieces at or behind D / 8 lie outside the descriptor: zeros.  Written as inline assembly because the compiler, which
// cannot tell the double buffer's halves apart, otherwise waits for the transfer before every LDS read behind it; the
// statement has no result registers, and dma_wait() stands before the barrier that hands the tile over.
template <int DP, int ROWS = 64>
struct TileDma {
  static constexpr int CPR = DP / 8, RPI = 64 / CPR, N = ROWS / 4 / RPI;  // pieces a row, rows an instruction, instructions a wave
  unsigned off[N];
  uint64_t at;    // address of the next tile
  int64_t left;   // bytes from there to the end of the last row, 0 and less: none
  unsigned step;  // bytes of ROWS rows
  __device__ __forceinline__ void init(const uint16_t* base, int64_t stride, int tile, int rows, int D, int wave, int lane) {
    step = (unsigned)stride * (2u * ROWS);
    at = (uint64_t)(base + (int64_t)tile * ROWS * stride);
    left = rows > 0 ? ((int64_t)(rows - 1) * stride + D) * 2 - (int64_t)tile * step : 0;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int r = (wave * N + n) * RPI + lane / CPR, c = (lane % CPR) ^ swz<DP>(r);
      off[n] = c * 8 < D ? (unsigned)r * (unsigned)stride * 2u + c * 16u : 0xfffffff0u;
    }
  }
  // the next ROWS rows to LDS byte address `lds`; all four waves take part
  __device__ __forceinline__ void next(unsigned lds, int wave) {
    const u32x4 rs = {(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)at), (unsigned)__builtin_amdgcn_readfirstlane((int)(at >> 32)) & 0xffffu,
                      (unsigned)__builtin_amdgcn_readfirstlane((int)(left <= 0 ? 0u : left < (int64_t)step ? (unsigned)left : step)), 0x00020000u};
#pragma unroll
    for (int n = 0; n < N; ++n)
      asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                   ::"{m0}"(lds + (unsigned)(wave * N + n) * 1024u), "v"(off[n]), "s"(rs)
                   : "memory");
    at += step;
    left -= step;
  }
};
DEV void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
DEV unsigned lds_addr(const void* p) { return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const void*)p; }

// a lane's operand fragments (pieces 2 ks + hi) of row first + (lane & 31), zeros where the row does not count (first + .. >= rows).
// Descriptor loads: no branch around a load, all of them in flight together.
template <int DP>
DEV void row_frags(const uint16_t* base, int64_t st, int first, int rows, int D, int lane, u32x4 (&f)[DP / 16]) {
  const __amdgpu_buffer_rsrc_t rs =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(base + (int64_t)first * st), 0, 0x7ffffff0, 0x00020000);
  const int n = lane & 31, hi = lane >> 5;
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) {
    const int c = 2 * ks + hi;
    f[ks] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                          rs, first + n < rows && c * 8 < D ? (int)((unsigned)n * (unsigned)st * 2u + c * 16u) : -16, 0, 0));
  }
}

// Where a lane reads its operand fragments in a tile: two addresses, the others differ from them in piece bits (an exclusive or)
// and by constants.
template <int DP>
struct LaneAt {
  static constexpr unsigned P = 2 * DP;
  unsigned row, tr;
  __device__ __forceinline__ LaneAt(const void* smem, int lane) {  // tiles are then named by their offset in smem (at LDS address 0)
    const int l16 = lane & 15, hi = lane >> 5;
    row = lds_addr(smem) + tile_at<DP>(lane & 31, hi);
    tr = lds_addr(smem) + tile_at<DP>(4 * hi + (l16 >> 2), ((lane >> 4) & 1) * 2 + ((l16 & 3) >> 1)) + (l16 & 1) * 8;
  }
  // Makes the compiler derive the other addresses here: held over the loop they do not fit the registers beside 128 columns, and
  // a reload from scratch waits for the tiles under way as well.
  __device__ __forceinline__ void renew() { asm volatile("" : "+v"(row), "+v"(tr)); }
  // row first + (lane & 31), piece 2 ks + hi; first: a multiple of 32
  __device__ __forceinline__ u32x4 frag(unsigned tile, int first, int ks) const {
    return *(const lds_u32x4*)(uintptr_t)((row ^ (ks << 5)) + (tile + first * P));
  }
  // transposed: rows (= reduction index) kb + 4 hi + 0..3 and kb + 8 + 4 hi + 0..3, column 32 dt + (lane & 31); kb: a multiple of 16
  __device__ __forceinline__ u32x4 frag_t(unsigned tile, int kb, int dt) const {
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)((tr ^ (dt << 6)) + (tile + kb * P)));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)((tr ^ (dt << 6 | 32)) + (tile + (kb + 8) * P)));
    return __builtin_bit_cast(u32x4, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

template <class E>
DEV u32x4 pack8(const f32x16& s, int first) {
  return u32x4{E::pack(s[first], s[first + 1]), E::pack(s[first + 2], s[first + 3]), E::pack(s[first + 4], s[first + 5]),
               E::pack(s[first + 6], s[first + 7])};
}
DEV f32x16 splat16(float x) { return f32x16{x, x, x, x, x, x, x, x, x, x, x, x, x, x, x, x}; }

// four rows' worth of one lane's column: 4 consecutive elements of a row as one 8-byte store
template <class E>
DEV void store4(uint16_t* p, float a, float b, float c, float d) {
  *reinterpret_cast<uint2*>(p) = make_uint2(E::pack(a, b), E::pack(c, d));
}

// a wave's 32 finished rows: out = O / sum, log-sum-exp; rows behind the sequence and rows without keys: zeros, and -inf
template <class E, int DP>
DEV void store_rows(const RbArgs& a, const f32x16 (&o)[DP / 32], float m, float l, int b, int h, int i, int hi, bool valid) {
  const float all = half_sum(l);
  if (i >= a.Tq) return;
  const float sum = valid ? all : 0.f, inv = 1.f / sum;
  uint16_t* const op = a.out + b * a.so.b + (int64_t)i * a.so.t + h * a.so.h;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = 32 * d + 8 * g + 4 * hi;
      if (c >= a.D) continue;
      if (sum == 0.f) store4<E>(op + c, 0.f, 0.f, 0.f, 0.f);
      else store4<E>(op + c, o[d][4 * g] * inv, o[d][4 * g + 1] * inv, o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv);
    }
  if (a.lse != nullptr && hi == 0)
    a.lse[((int64_t)b * a.H + h) * a.Tq + i] = sum == 0.f ? -RB_INF : (m * a.c2 - E::up + __builtin_amdgcn_logf(sum)) * RB_LN2;
}

// =============================================================================================== forward
// One workgroup = 4 waves x 32 queries of one (sequence, head); 64-key tiles of K and V, double buffered in LDS, softmax in one pass
// with a running maximum and sum in f32.  P is rounded to the tensors' type as the second product's operand (half a step of each
// term, while the sum that divides it is not rounded): f32 operands would take eight times the matrix unit's time.
// At 64 columns the vector unit works for 62% of the busy cycles (an exponential and some four instructions a score) and the matrix
// unit for 39%: 101% together, so on a SIMD they take turns - two or three waves do not bring them side by side.
// 11250 x 11250, 8 heads of 64: 317 to 325 us from card to card, 800 to 818 TFLOP/s (a large matrix product reaches 1178 here).  At
// 128 columns, 2 x 2047 causal, 16 heads: 55.6 us, 618 TFLOP/s, each unit at work for 28%: on average 1.3 waves a SIMD (two fit the
// registers, and the row tiles end one by one), which wait for 37% of their time.  32 x 400, 4 heads: 15.2 us, of which some 3.4 pass
// before the first product.  Scores of the next tile issued ahead of this one's exponentials took 496 us for the long
// case: the registers of both tiles do not fit beside two waves.
template <class E, int DP>
__global__ __launch_bounds__(256, DP == 128 ? 2 : 3) void rb_fwd_kernel(RbArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  constexpr int P = 2 * DP, TILE = 64 * P, NK = DP / 16, ND = DP / 32;
  unsigned char* const sK = smem;
  unsigned char* const sV = smem + 2 * TILE;
  float* const sB = reinterpret_cast<float*>(smem + 4 * TILE);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hi = lane >> 5, n32 = lane & 31;
  const Place at = place_of(a);
  const Quot bh = split(at.head, a.per_head);
  const int b = bh.q, h = bh.r, hk = a.per_group.over(h), tile = a.ntile - 1 - at.rank;
  const Seq sq = seq_of(a, b);
  const int q0 = tile * 128, i = q0 + wave * 32 + n32, p0 = sq.off + q0 + wave * 32;
  int kend = q0 < sq.qlen ? sq.klen : 0, wend = q0 + wave * 32 < sq.qlen ? sq.klen : 0;
  if (a.causal) {
    kend = min(kend, sq.off + min(q0 + 128, sq.qlen));
    wend = min(wend, p0 + 32);
  }
  const int nt = kend > 0 ? (kend + 63) >> 6 : 0;

  TileDma<DP> dk, dv;
  dk.init(a.k + b * a.sk.b + hk * a.sk.h, a.sk.t, 0, sq.klen, a.D, wave, lane);
  dv.init(a.v + b * a.sv.b + hk * a.sv.h, a.sv.t, 0, sq.klen, a.D, wave, lane);
  const unsigned lK = lds_addr(sK), lV = lds_addr(sV);
  const LaneAt<DP> in(smem, lane);
  if (nt > 0) {
    dk.next(lK, wave);
    dv.next(lV, wave);
  }
  u32x4 qf[NK];
  f32x16 o[ND];
  float m = -RB_INF, l = 0.f;
  row_frags<DP>(a.q + b * a.sq.b + h * a.sq.h, a.sq.t, q0 + wave * 32, sq.qlen, a.D, lane, qf);
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = splat16(0.f);
  spread_table(a, h, sB, reinterpret_cast<float*>(sK + TILE), TILE / 4, tid);
  dma_wait();
  __syncthreads();
  const float left = sB[0], right = sB[2 * (a.mde + RB_PAD)];

  // one tile; the buffer's parity is a constant (LDS addresses are then lane addresses and immediates)
  auto step = [&](int t, auto parity) {
    constexpr int buf = decltype(parity)::value;
    const int j0 = t * 64;
    // the next tile's transfer: requested behind the first products, whose results the wave waits for anyway
    auto transfer = [&] {
      if (t + 1 >= nt) return;
      dk.next(lK + (buf ^ 1) * TILE, wave);
      dv.next(lV + (buf ^ 1) * TILE, wave);
    };
    if (j0 < wend) {
      constexpr unsigned kt = buf * TILE, vt = (2 + buf) * TILE;
      f32x16 s[2];
      // S^T = K Q^T + bias.  Operands are requested in groups ahead of the products that use them: left alone, the compiler
      // reads, waits and multiplies one fragment at a time.
      auto scores = [&](auto zero) {
        constexpr int GK = 4;
        u32x4 kf[GK][2];
#pragma unroll
        for (int k0 = 0; k0 < NK; k0 += GK) {
#pragma unroll
          for (int ks = 0; ks < GK && k0 + ks < NK; ++ks)
#pragma unroll
            for (int u = 0; u < 2; ++u) kf[ks][u] = in.frag(kt, 32 * u, k0 + ks);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int ks = 0; ks < GK && k0 + ks < NK; ++ks)
#pragma unroll
            for (int u = 0; u < 2; ++u) s[u] = E::mma(kf[ks][u], qf[k0 + ks], decltype(zero)::value && k0 + ks == 0 ? splat16(0.f) : s[u]);
        }
      };
      // far tiles: the bias is a constant, added with the running reference
      const bool far = j0 - (p0 + 31) >= a.mde || j0 + 63 - p0 <= -a.mde;
      const float cb = far ? (j0 > p0 ? right : left) : 0.f;
      if (far) {
        scores(True{});
      } else {
        const float* const bp = sB + (j0 - p0 - n32 + 4 * hi + a.mde + RB_PAD);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[u][r] = bp[32 * u + 8 * (r >> 2) + (r & 3)];
        scores(False{});
      }
      transfer();
      u32x4 vf[2][ND];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int d = 0; d < ND; ++d) vf[kk][d] = in.frag_t(vt, 16 * kk, d);
      __builtin_amdgcn_sched_barrier(0);
      if (j0 + 64 > sq.klen || (a.causal && j0 + 63 > p0)) {
        const int lim = (a.causal ? min(sq.klen, p0 + n32 + 1) : sq.klen) - j0 - 4 * hi;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (32 * u + 8 * (r >> 2) + (r & 3) >= lim) s[u][r] = -RB_INF;
      }
      float mx[2] = {fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1])};
#pragma unroll
      for (int r = 2; r < 16; r += 2)
#pragma unroll
        for (int u = 0; u < 2; ++u) mx[u] = fmaxf(fmaxf(mx[u], s[u][r]), s[u][r + 1]);
      const float top = half_max(fmaxf(mx[0], mx[1])) + cb;
      // the running reference moves only when some row's scores outgrow it by 2^8 (2^7): probabilities stay below 256 (2^14), the
      // sums in f32
      if (__any((top - m) * a.c2 > E::grow)) {
        const float up = fmaxf(m, top);
        const float al = up == -RB_INF ? 1.f : __builtin_amdgcn_exp2f((m - up) * a.c2);
        m = up;
        l *= al;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] *= al;
      }
      const float mc = ((m == -RB_INF ? 0.f : m) - cb) * a.c2 - E::up;
      u32x4 pb[4];
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[u][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][r], a.c2, -mc));
          sum[u] += s[u][r];
        }
        pb[2 * u] = pack8<E>(s[u], 0);
        pb[2 * u + 1] = pack8<E>(s[u], 8);
      }
      l += sum[0] + sum[1];
      u32x4 vg[2][ND];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int d = 0; d < ND; ++d) vg[kk][d] = in.frag_t(vt, 32 + 16 * kk, d);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] = E::mma(vf[kk][d], pb[kk], o[d]);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] = E::mma(vg[kk][d], pb[2 + kk], o[d]);
    } else {
      transfer();
    }
    dma_wait();
    __syncthreads();
  };
  for (int t = 0; t < nt; t += 2) {
    step(t, Const<0>{});
    if (t + 1 < nt) step(t + 1, Const<1>{});
  }
  store_rows<E, DP>(a, o, m, l, b, h, i, hi, i < sq.qlen);
}

// ------------------------------------------------------------------------------------ forward, few query rows
// Rows = (query, head of the group) of one (sequence, key head), 32 to a workgroup: a head's group shares the K and V it reads.
// Nothing is reused across waves, so each of the NW waves streams its own 32-key tiles (every NW-th of the workgroup's), K straight
// into operand registers, V through a wave's own LDS tile for the transposing reads, the next tile's loads in flight; the waves'
// running softmax states are joined in LDS.  Bound by the bytes of K and V: 32 x 1 against up to 8192 keys, 16 heads in groups of 4,
// 128 columns: 95.5 us, 4.17 TB/s (a large copy reaches 5.16); 4 x 8 x 30001, 8 heads of 64: 53.7 us, 4.6 TB/s; 1 x 500, 4 heads:
// 12.1 us, one workgroup's chain of loads (8.6 us).  Where few workgroups would run, the keys are split over `nsplit` of them: states go
// to the workspace and rb_join_kernel joins them in order (4.8 us for the first of these).
constexpr int RB_FEW_TABLE = 4096;  // floats of LDS for the group's tables by distance; wider ones are gathered from memory
template <int DP, int NW>
constexpr int few_area() {  // bytes: the waves' V tiles, later their O rows [NW][32][DP + 4] and (reference, sum) [NW][2][32]
  return NW * 32 * (DP + 4) * 4 + NW * 256;
}
template <class E, int DP, int NW>
__global__ __launch_bounds__(64 * NW, 2) void rb_few_kernel(RbArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  constexpr int P = 2 * DP, NK = DP / 16, ND = DP / 32, CPR = DP / 8, RPI = 64 / CPR, NV = 32 / RPI, NT = 64 * NW;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hi = lane >> 5, n32 = lane & 31;
  unsigned char* const sV = smem + wave * 32 * P;
  const LaneAt<DP> at(smem, lane);
  float* const sT = reinterpret_cast<float*>(smem + few_area<DP, NW>());
  const int G = a.per_group.d, R = a.Tq * G;
  const int id = xcd_order(blockIdx.x, a.nblk);
  const Quot is = split(id, a.per_split), it = split(is.q, a.per_tile), bh = split(it.q, a.per_head);
  const int part = is.r, rb = it.r, bk = it.q, b = bh.q, hk = bh.r;
  const Seq sq = seq_of(a, b);
  const Quot ig = split(rb * 32 + n32, a.per_group);
  const int row = rb * 32 + n32, i = ig.q, g = ig.r, h = hk * G + g;
  const bool valid = row < R && i < sq.qlen;
  const int p = sq.off + i, i_first = a.per_group.over(rb * 32), i_end = a.per_group.over(rb * 32 + 31), i_last = min(i_end, sq.qlen - 1);
  int kend = i_first < sq.qlen ? sq.klen : 0;
  if (a.causal) kend = min(kend, sq.off + i_last + 1);
  const int ntile = kend > 0 ? (kend + 31) >> 5 : 0, per = a.per_split.over(ntile + a.nsplit - 1);
  const int t0 = part * per, t1 = min(ntile, t0 + per);
  const uint16_t* const kp = a.k + b * a.sk.b + hk * a.sk.h;
  const uint16_t* const vp = a.v + b * a.sv.b + hk * a.sv.h;

  u32x4 qf[NK], kf[NK], vr[NV];
  auto load = [&](int t) {
    const int j0 = t * 32, left_rows = sq.klen - j0;
    const __amdgpu_buffer_rsrc_t rk =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(kp + (int64_t)j0 * a.sk.t), 0, 0x7ffffff0, 0x00020000);
    const __amdgpu_buffer_rsrc_t rv =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(vp + (int64_t)j0 * a.sv.t), 0, 0x7ffffff0, 0x00020000);
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) {
      const int c = 2 * ks + hi;
      kf[ks] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                             rk, n32 < left_rows && c * 8 < a.D ? (int)((unsigned)n32 * (unsigned)a.sk.t * 2u + c * 16) : -16, 0, 0));
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int r = n * RPI + lane / CPR, c = lane % CPR;
      vr[n] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                            rv, r < left_rows && c * 8 < a.D ? (int)((unsigned)r * (unsigned)a.sv.t * 2u + c * 16) : -16, 0, 0));
    }
  };
  int t = t0 + wave;
  if (t < t1) load(t);
  const uint16_t* const qp = a.q + b * a.sq.b + (int64_t)(valid ? i : 0) * a.sq.t + (valid ? h : hk * G) * a.sq.h;
#pragma unroll
  for (int ks = 0; ks < NK; ++ks) {  // (a row that does not count reads row 0 and drops it)
    const int c = 2 * ks + hi;
    qf[ks] = u32x4{0, 0, 0, 0};
    if (a.Tq > 0 && c * 8 < a.D) qf[ks] = *reinterpret_cast<const u32x4*>(qp + c * 8);
    if (!valid) qf[ks] = u32x4{0, 0, 0, 0};
  }
  const int hc = hk * G + min(g, G - 1);
  const float left = bias_entry(a, -a.mde, hc), right = bias_entry(a, a.mde, hc);
  const int p_lo = sq.off + i_first, p_hi = sq.off + i_end;  // positions of the workgroup's rows
  // the group's tables by distance, if any tile of the workgroup's needs them
  const int wide = 2 * a.mde + 1;
  const bool staged = G * wide <= RB_FEW_TABLE;
  if (staged && t0 < t1 && t0 * 32 - p_hi < a.mde && t1 * 32 - 1 - p_lo > -a.mde) {
    for (int x = tid; x < G * wide; x += NT) sT[x] = bias_entry(a, x % wide - a.mde, hk * G + x / wide);
    __syncthreads();
  }
  const float* const tp = sT + min(g, G - 1) * wide + a.mde;
  f32x16 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = splat16(0.f);
  float m = -RB_INF, l = 0.f;
  for (; t < t1; t += NW) {
    const int j0 = t * 32;
    f32x16 s;
    if (j0 - p_hi >= a.mde || j0 + 31 - p_lo <= -a.mde) {
      s = splat16(j0 > p_lo ? right : left);
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int dist = min(max(j0 + 8 * (r >> 2) + 4 * hi + (r & 3) - p, -a.mde), a.mde);
        s[r] = staged ? tp[dist] : bias_entry(a, dist, hc);
      }
    }
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) s = E::mma(kf[ks], qf[ks], s);
#pragma unroll
    for (int n = 0; n < NV; ++n) *reinterpret_cast<u32x4*>(sV + tile_at<DP>(n * RPI + lane / CPR, lane % CPR)) = vr[n];
    if (t + NW < t1) load(t + NW);
    if (j0 + 32 > sq.klen || (a.causal && j0 + 31 > p_lo)) {
      const int lim = (a.causal ? min(sq.klen, p + 1) : sq.klen) - j0 - 4 * hi;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (8 * (r >> 2) + (r & 3) >= lim) s[r] = -RB_INF;
    }
    float mx = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
    mx = half_max(mx);
    if (__any((mx - m) * a.c2 > E::grow)) {  // as in rb_fwd_kernel
      const float up = fmaxf(m, mx);
      const float al = up == -RB_INF ? 1.f : __builtin_amdgcn_exp2f((m - up) * a.c2);
      m = up;
      l *= al;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= al;
    }
    const float mc = (m == -RB_INF ? 0.f : m * a.c2) - E::up;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.c2, -mc));
      l += s[r];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave's V tile is written before other lanes read it
    __builtin_amdgcn_wave_barrier();
    // P as a rounded value and the rounded rest: the products are free here, and a row of few keys has no other rounding to hide it
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      const u32x4 pb = pack8<E>(s, 8 * kk);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[8 * kk + 2 * e] -= E::lo(pb[e]);
        s[8 * kk + 2 * e + 1] -= E::hi(pb[e]);
      }
      const u32x4 rest = pack8<E>(s, 8 * kk);
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const u32x4 vf = at.frag_t(wave * 32 * P, 16 * kk, d);
        o[d] = E::mma(vf, pb, o[d]);
        o[d] = E::mma(vf, rest, o[d]);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }

  // join the waves: rows of O [NW][32][DP + 4] f32 (the padding spreads a column's 32 rows over the banks), references, sums
  l = half_sum(l);
  float* const sO = reinterpret_cast<float*>(smem);
  float* const sM = sO + NW * 32 * (DP + 4);  // [NW][2][32]
  __syncthreads();                            // the V tiles are read
  if (hi == 0) sM[wave * 64 + n32] = m, sM[wave * 64 + 32 + n32] = valid ? l : 0.f;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      *reinterpret_cast<f32x4*>(sO + (wave * 32 + n32) * (DP + 4) + 32 * d + 8 * e + 4 * hi) =
          f32x4{o[d][4 * e], o[d][4 * e + 1], o[d][4 * e + 2], o[d][4 * e + 3]};
  __syncthreads();
  const int rows = min(32, R - rb * 32);
  const int64_t first = (int64_t)bk * R + rb * 32;
  float2* const ml = reinterpret_cast<float2*>(a.part + (int64_t)a.B * a.Hk * R * a.nsplit * DP);
  for (int x = tid; x < rows * (DP / 4); x += NT) {
    const int r = x / (DP / 4), c = x % (DP / 4) * 4, rr = rb * 32 + r;
    float top = -RB_INF, sum = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) top = fmaxf(top, sM[w * 64 + r]);
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {  // in order
      const float lw = sM[w * 64 + 32 + r];
      if (lw == 0.f) continue;
      const float f = __builtin_amdgcn_exp2f((sM[w * 64 + r] - top) * a.c2);
      sum += lw * f;
      y += *reinterpret_cast<const f32x4*>(sO + (w * 32 + r) * (DP + 4) + c) * f;
    }
    if (a.nsplit > 1) {  // O rows [row][split][DP], then (reference, sum) [row][split]
      *reinterpret_cast<f32x4*>(a.part + ((first + r) * a.nsplit + part) * DP + c) = y;
      if (c == 0) ml[(first + r) * a.nsplit + part] = make_float2(top * a.c2 - E::up, sum);
      continue;
    }
    const int64_t hq = hk * G + rr % G, iq = rr / G;
    if (c < a.D) {
      uint16_t* const op = a.out + b * a.so.b + iq * a.so.t + hq * a.so.h + c;
      const float inv = 1.f / sum;
      if (sum == 0.f) store4<E>(op, 0.f, 0.f, 0.f, 0.f);
      else store4<E>(op, y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
    }
    if (c == 0 && a.lse != nullptr)
      a.lse[((int64_t)b * a.H + hq) * a.Tq + iq] = sum == 0.f ? -RB_INF : (top * a.c2 - E::up + __builtin_amdgcn_logf(sum)) * RB_LN2;
  }
}

// one wave per row: the splits' states in order, 64 at a time (their weights in the lanes, so that the loads of O do not wait)
template <class E, int DP>
__global__ __launch_bounds__(256) void rb_join_kernel(RbArgs a) {
  const int G = a.H / a.Hk, R = a.Tq * G, lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), nrow = (int64_t)a.B * a.Hk * R;
  if (row >= nrow) return;
  const float2* const ml = reinterpret_cast<const float2*>(a.part + nrow * a.nsplit * DP) + row * a.nsplit;
  constexpr int N = DP == 128 ? 2 : 1;
  float m = -RB_INF, sum = 0.f, o[N] = {};
  for (int s0 = 0; s0 < a.nsplit; s0 += 64) {
    const int n = min(64, a.nsplit - s0);
    float2 x = make_float2(-RB_INF, 0.f);
    if (lane < n) x = ml[s0 + lane];
    if (x.y == 0.f) x.x = -RB_INF;
    const float up = fmaxf(m, wave_max(x.x));
    if (up == -RB_INF) continue;
    const float al = __builtin_amdgcn_exp2f(m - up), w = x.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(x.x - up);
    m = up;
    sum = sum * al + wave_sum(x.y * w);
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] *= al;
    const float* const op = a.part + (row * a.nsplit + s0) * DP + (DP == 128 ? 2 : 1) * (lane & (DP - 1));
    for (int s = 0; s < n; s += 8)
#pragma unroll
      for (int e = 0; e < 8; ++e) {  // (behind the last split: its row again, with weight 0)
        const float ws = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), s + e));
        const float* const at = op + min(s + e, n - 1) * DP;
        if constexpr (DP == 128) {
          const float2 y = *reinterpret_cast<const float2*>(at);
          o[0] += y.x * ws;
          o[1] += y.y * ws;
        } else {
          o[0] += *at * ws;
        }
      }
  }
  const int64_t bk = row / R;
  const int rr = (int)(row % R), b = (int)(bk / a.Hk), h = (int)(bk % a.Hk) * G + rr % G, i = rr / G;
  uint16_t* const at = a.out + b * a.so.b + (int64_t)i * a.so.t + h * a.so.h;
  const float inv = 1.f / sum;
  if constexpr (DP == 128) {
    if (2 * lane < a.D) *reinterpret_cast<unsigned*>(at + 2 * lane) = sum == 0.f ? 0u : E::pack(o[0] * inv, o[1] * inv);
  } else {
    if (lane < a.D) at[lane] = sum == 0.f ? (uint16_t)0 : (uint16_t)E::pack(o[0] * inv, 0.f);
  }
  if (a.lse != nullptr && lane == 0) a.lse[((int64_t)b * a.H + h) * a.Tq + i] = sum == 0.f ? -RB_INF : (m + __builtin_amdgcn_logf(sum)) * RB_LN2;
}

// =============================================================================================== backward
// The table's gradient is the sum of dS along diagonals (equal distance r).  A lane holds one query and groups of four
// consecutive keys, and a diagonal runs through neighbouring lanes, so a group is summed along its diagonals by three DPP
// additions that pass the partial sums one lane up:  N = x3 + up(x2 + up(x1 + up(x0))): lane i then holds the sum of distance
// r = k0 + 3 - i.  What passes from lane 31 to lane 32 (from 63 to 0) belongs to the same distance as lanes 0..2 of the SAME half
// 32 keys before: lanes 0..2 of a half separate their own part (`own`, a chain that starts at their half) from what came
// over, which is added to the part kept from 32 keys before, `kept`.  So each (group, half) writes 32 neighbouring cells of its own
// array per sub-tile, cells that the other waves do not touch in the same step (their queries are 32 further): plain
// read-add-write with a barrier per step, no atomics, and a fixed order.  The arrays are rings of 256 distances: a step's tile
// touches 191, and the 64 that it leaves behind are added up and put away during the next one (arrays over all distances leave
// one workgroup a CU for wide tables: 2 x 8 heads of 64, 1500 x 1500, 800 distances: backward 98 us against 119).  11 vector instructions per group of four; ds_add_f32
// took 187 cycles per instruction here (124 us for the 32 x 400 backward's dq kernel).
constexpr int DPP_WAVE_ROR1 = 0x13c, DPP_ROW_SHR1 = 0x111;
DEV float from_below(float x) { return dpp_mov<DPP_WAVE_ROR1>(x); }      // lane l: the value of lane l - 1, lane 0: of lane 63
DEV float from_below_row(float x) { return dpp_mov<DPP_ROW_SHR1>(x); }   // within 16 lanes, 0 enters
DEV float swap_halves(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const unsigned a0 = r[0], a1 = r[1];
  return __uint_as_float((threadIdx.x & 32) ? a0 : a1);
}

// dq and the table's gradient: 4 waves x 32 queries of one (sequence, head) against 64-key tiles.
//   S^T = K Q^T (+ bias), dP^T = V dO^T (from -delta), dS = P dP, dQ^T += K^T dS^T
// dS is rounded to the tensors' type for the last product only; the table's gradient takes it in f32.  dk and dv have a kernel of
// their own, which computes S and dP again (7 products for 5): sums over queries and over keys in one kernel would need atomics,
// and results that change from run to run, or a T x T operand in memory.
// Bound by both units in turn: 6001 x 6001, 8 heads of 64: 141 us, 782 TFLOP/s of its three products, the vector unit busy for 58%
// of the time, the matrix unit for 40%.  2 x 2047 causal, 16 heads of 128: 89 us, each unit 28% (with the operands' addresses held
// in registers, which did not fit, half as long again); 32 x 400, 4 heads: 28 to 30 us.  fp16: the factor of dS (fit) and what it
// pushes out of the registers take 159 us instead of 151 for the first of these, 97 instead of 93 for the second.
// Where few workgroups would run, the keys are split over `nsplit` of them, whose sums rb_dq_join_kernel adds in order.
// It also leaves delta_i = do_i . o_i and the rows' log-sum-exp in log2 units for the next kernel, +inf where a row has no
// keys or lies behind its sequence (exp2(s - inf) = 0: such rows drop out of every product).
// WAVES a SIMD: 64 columns fit three (fewer operands ahead, addresses derived per sub-tile), for more than two workgroups a CU
// (6001 x 6001, whole backward: 326 us against 340); up to there the wider form is faster (24 ragged windows: 36.4 us
// against 37.6; 32 x 400: 54.1 against 54.9, eager calls).
template <class E, int DP, int WAVES>
__global__ __launch_bounds__(256, WAVES) void rb_dq_kernel(RbArgs a) {
  constexpr bool TIGHT = DP == 128 || WAVES == 3;
  constexpr bool LATE = DP == 128 || (WAVES == 3 && E::narrow);  // no registers to hold K's columns across the exponentials
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  constexpr int P = 2 * DP, TILE = 64 * P, NK = DP / 16, ND = DP / 32;
  unsigned char* const sK = smem;
  unsigned char* const sV = smem + 2 * TILE;
  float* const sB = reinterpret_cast<float*>(smem + 4 * TILE);
  const int span = 2 * (a.mde + RB_PAD) + 1;
  float* const sSum = sB + span;                                    // [span] sums by distance
  float* const sG = sSum + span;                                    // [4 groups][2 halves][256] the sums still open
  double* const sFar = reinterpret_cast<double*>(smem + 4 * TILE + (span + 1) / 2 * 16 + 8192);  // [4][2], [4]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hi = lane >> 5, n32 = lane & 31;
  const Place at = place_of(a);
  const Quot bh = split(at.head, a.per_head);
  const int part = at.part, b = bh.q, h = bh.r, hk = a.per_group.over(h), tile = a.ntile - 1 - at.rank;
  const Seq sq = seq_of(a, b);
  const int q0 = tile * 128, i = q0 + wave * 32 + n32, p0 = sq.off + q0 + wave * 32;
  int kend = q0 < sq.qlen ? sq.klen : 0, wend = q0 + wave * 32 < sq.qlen ? sq.klen : 0;
  if (a.causal) {
    kend = min(kend, sq.off + min(q0 + 128, sq.qlen));
    wend = min(wend, p0 + 32);
  }
  const int tiles = kend > 0 ? (kend + 63) >> 6 : 0;
  const int ta = a.per_split.over(tiles * part), nt = a.per_split.over(tiles * (part + 1));  // this workgroup's key tiles

  TileDma<DP> dK, dV;
  dK.init(a.k + b * a.sk.b + hk * a.sk.h, a.sk.t, ta, sq.klen, a.D, wave, lane);
  dV.init(a.v + b * a.sv.b + hk * a.sv.h, a.sv.t, ta, sq.klen, a.D, wave, lane);
  const unsigned lK = lds_addr(sK), lV = lds_addr(sV);
  LaneAt<DP> in(smem, lane);
  if (ta < nt) {
    dK.next(lK, wave);
    dV.next(lV, wave);
  }
  u32x4 qf[NK], df[NK];
  row_frags<DP>(a.q + b * a.sq.b + h * a.sq.h, a.sq.t, q0 + wave * 32, sq.qlen, a.D, lane, qf);
  row_frags<DP>(a.dout + b * a.sdo.b + h * a.sdo.h, a.sdo.t, q0 + wave * 32, sq.qlen, a.D, lane, df);
  const float sign = wave & 1 ? -1.f : 1.f;
  float delta = 0.f, lse2 = RB_INF, fac = RB_FAC0;  // fac: of the rounded dS (fp16)
  {
    u32x4 of[NK];
    row_frags<DP>(a.o + b * a.so.b + h * a.so.h, a.so.t, q0 + wave * 32, sq.qlen, a.D, lane, of);
    const float given = a.lse_in[((int64_t)b * a.H + h) * a.Tq + min(i, a.Tq - 1)];
    for (int x = tid; x < span + 2048; x += 256) sSum[x] = 0.f;
    const float x = i < sq.qlen ? given : -RB_INF;
#pragma unroll
    for (int ks = 0; ks < NK; ++ks)
#pragma unroll
      for (int e = 0; e < 4; ++e) delta += E::lo(df[ks][e]) * E::lo(of[ks][e]) + E::hi(df[ks][e]) * E::hi(of[ks][e]);
    delta = half_sum(delta);
    if (x != -RB_INF) lse2 = x * RB_LOG2E;
    // The matrix unit's sums lean to the negative side by about 2^-25 each; over the 36 million pairs of a 6001 x 6001 head that
    // showed as 10^-5 of the table's gradient.  Odd waves therefore compute -dP (and all behind it), so that it cancels (5 10^-7 left
    // against these formulas in 64 bits; that delta takes the rounded out costs far more, see include/csship.h).
    if (wave & 1) {
#pragma unroll
      for (int ks = 0; ks < NK; ++ks) df[ks] ^= 0x80008000u;
    }
    const int64_t to = ((int64_t)b * a.H + h) * a.tq128 + i;  // rows up to the tile's end: the next kernel reads whole tiles
    if (hi == 0 && part == 0) a.delta[to] = -delta, a.lse2[to] = lse2;
    delta *= sign;
  }
  f32x16 dq[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) dq[d] = splat16(0.f);
  double farl = 0., farr = 0.;   // 64 bits: thousands of terms of both signs
  float kept[4] = {0.f, 0.f, 0.f, 0.f};
  bool pending = false;
  spread_table(a, h, sB, reinterpret_cast<float*>(sK + TILE), TILE / 4, tid);
  dma_wait();
  __syncthreads();
  const float left = sB[0], right = sB[span - 1];
  // lane's distance for key base 0 and its class (half); lanes 0..2: of the other half, 32 keys before.  Open sums stand at
  // (distance - base) mod 256 of their class and group: a step touches the 191 from `low` on.
  const int cls = n32 < 3 ? hi ^ 1 : hi, dist0 = 4 * cls + 3 - n32 - (n32 < 3 ? 32 : 0) - p0;
  float* const cells = sG + cls * 256;
  const int pw = sq.off + q0;
  auto cell = [&](int k, int g) { return cells + (2 * g * 256 + ((dist0 + k + 8 * g) & 255)); };
  // the 64 distances that no later step touches, from all classes to sSum, by one wave
  auto close = [&](int from) {
    const int r = from + lane, x = r + a.mde + RB_PAD;
    if (x < 0 || x >= span) return;
    float y = 0.f;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      float* const at = sG + c * 256 + (r & 255);
      y += *at;
      *at = 0.f;
    }
    sSum[x] = y;
  };

  auto step = [&](int t, auto parity) {
    constexpr int buf = decltype(parity)::value;
    const int j0 = t * 64;
    auto transfer = [&] {  // the next tile's, behind the first products as in rb_fwd_kernel
      if (t + 1 >= nt) return;
      dK.next(lK + (buf ^ 1) * TILE, wave);
      dV.next(lV + (buf ^ 1) * TILE, wave);
    };
    if (!(j0 < wend)) transfer();
    constexpr unsigned kt = buf * TILE, vt = (2 + buf) * TILE;
    const bool active = j0 < wend;
    const bool near = active && j0 - (p0 + 31) < a.mde && j0 + 63 - p0 > -a.mde;
    const int low = j0 - pw - 127;  // the step's smallest distance
    if (t > ta && wave == (t & 3) && low - 64 <= a.mde + RB_PAD && low > -a.mde - RB_PAD) close(low - 64);
    const bool any_near = j0 - (pw + 127) < a.mde && j0 + 63 - pw > -a.mde;  // of any wave: they share the barrier
    if (!near && pending) {  // the last parts kept have nothing to wait for
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if (n32 < 3) *cell(j0, g) += sign * kept[g];
#pragma unroll
      for (int g = 0; g < 4; ++g) kept[g] = 0.f;
      pending = false;
    }
    const bool edge = j0 + 64 > sq.klen || (a.causal && j0 + 63 > p0);
    const int lim = (a.causal ? min(sq.klen, p0 + n32 + 1) : sq.klen) - j0 - 4 * hi;
    const float l2 = near ? lse2 : lse2 - (j0 > p0 ? right : left) * a.c2;  // far: the bias is a constant
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (u == 1 && any_near) __syncthreads();
      if (!active) continue;
      if (TIGHT) in.renew();
      f32x16 s, dp = splat16(-delta);
      // operands in groups ahead of the products that use them, as in rb_fwd_kernel
      auto scores = [&](auto zero) {
        constexpr int GK = TIGHT ? 2 : 4;
        u32x4 kf[GK], vf[GK];
#pragma unroll
        for (int c = 0; c < NK; c += GK) {
#pragma unroll
          for (int ks = 0; ks < GK && c + ks < NK; ++ks) {
            kf[ks] = in.frag(kt, 32 * u, c + ks);
            vf[ks] = in.frag(vt, 32 * u, c + ks);
          }
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int ks = 0; ks < GK && c + ks < NK; ++ks) {
            s = E::mma(kf[ks], qf[c + ks], decltype(zero)::value && c + ks == 0 ? splat16(0.f) : s);
            dp = E::mma(vf[ks], df[c + ks], dp);
          }
        }
      };
      if (near) {
        const float* const bp = sB + (j0 - p0 - n32 + 4 * hi + 32 * u + a.mde + RB_PAD);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = bp[8 * (r >> 2) + (r & 3)];
        scores(False{});
      } else {
        scores(True{});
      }
      if (u == 0) transfer();
      u32x4 kf[2][ND];
#pragma unroll
      for (int kk = 0; kk < (LATE ? 0 : 2); ++kk)
#pragma unroll
        for (int d = 0; d < ND; ++d) kf[kk][d] = in.frag_t(kt, 32 * u + 16 * kk, d);
      __builtin_amdgcn_sched_barrier(0);
      if (edge) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (32 * u + 8 * (r >> 2) + (r & 3) >= lim) s[r] = -RB_INF;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.c2, -l2)) * dp[r];
      if (near) {
        float old[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) old[g] = *cell(j0 + 32 * u, g);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float all = s[4 * g + 3] + from_below(s[4 * g + 2] + from_below(s[4 * g + 1] + from_below(s[4 * g])));
          const float own = s[4 * g + 3] + from_below_row(s[4 * g + 2] + from_below_row(s[4 * g + 1]));
          const float x = n32 < 3 ? (all - own) + kept[g] : all;
          kept[g] = swap_halves(own);
          *cell(j0 + 32 * u, g) = __builtin_fmaf(sign, x, old[g]);
        }
        pending = true;
      } else {
        float x[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int r = 4; r < 16; ++r) x[r & 3] += s[r];
        const double y = (double)((x[0] + x[1]) + (x[2] + x[3]));
        if (j0 > p0) farr += y;
        else farl += y;
      }
      if constexpr (E::narrow) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= fac;
        fit(s, dq, fac);
      }
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const u32x4 ds = pack8<E>(s, 8 * kk);
        if (LATE) {
#pragma unroll
          for (int d = 0; d < ND; ++d) kf[kk][d] = in.frag_t(kt, 32 * u + 16 * kk, d);
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) dq[d] = E::mma(kf[kk][d], ds, dq[d]);
      }
    }
    dma_wait();
    __syncthreads();
  };
  for (int t = ta; t < nt; t += 2) {
    step(t, Const<0>{});
    if (t + 1 < nt) step(t + 1, Const<1>{});
  }
  if (pending) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
      if (n32 < 3) *cell(nt * 64, g) += sign * kept[g];
  }

  if (i < a.Tq && a.nsplit > 1) {  // sums in f32: [split][sequence, head, query][DP]
    float* const pq = a.part2 + ((((int64_t)part * a.B + b) * a.H + h) * a.Tq + i) * DP;
    const float f = E::narrow ? sign / fac : sign;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(pq + 32 * d + 8 * g + 4 * hi) =
            f32x4{dq[d][4 * g] * f, dq[d][4 * g + 1] * f, dq[d][4 * g + 2] * f, dq[d][4 * g + 3] * f};
  } else if (i < a.Tq) {
    uint16_t* const op = a.dq + b * a.sdq.b + (int64_t)i * a.sdq.t + h * a.sdq.h;
    const float f = E::narrow ? sign * a.scale / fac : sign * a.scale;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = 32 * d + 8 * g + 4 * hi;
        if (c < a.D) store4<E>(op + c, dq[d][4 * g] * f, dq[d][4 * g + 1] * f, dq[d][4 * g + 2] * f, dq[d][4 * g + 3] * f);
      }
  }
  // The workgroup's share of the table's gradient.  A bucket's distances are contiguous: running sums over the distances in 64
  // bits, and a bucket is the difference of two (one thread per bucket adding up its distances took 4 us).
  const int nwg = a.B * a.ntile * a.nsplit, wg = (b * a.ntile + tile) * a.nsplit + part;
  int lo = 0, end = 0;
  if (tid < a.nb) lo = a.bucket_range[2 * tid], end = a.bucket_range[2 * tid + 1];
  farl = sign * wave_total(farl);
  farr = sign * wave_total(farr);
  if (lane == 0) sFar[2 * wave] = farl, sFar[2 * wave + 1] = farr;
  __syncthreads();
  if (ta < nt && wave < 3) close((nt - 1) * 64 - pw - 127 + 64 * wave);  // the last step's
  __syncthreads();
  const int each = (span + 255) >> 8, first = tid * each;
  double mine = 0.;
  for (int x = first; x < min(first + each, span); ++x) mine += (double)sSum[x];
  double upto = mine;  // inclusive over the wave, then over the workgroup
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) {
    const double y = __shfl_up(upto, w);
    if (lane >= w) upto += y;
  }
  if (lane == 63) sFar[8 + wave] = upto;
  __syncthreads();
  double* const run = reinterpret_cast<double*>(smem);  // [span + 1], where the tiles and, for narrow ones, sB were
  static_assert(4 * TILE + 4 * SPAN_MAX >= 8 * (SPAN_MAX + 1), "run ends before sSum");
  upto -= mine;
  for (int w = 0; w < wave; ++w) upto += sFar[8 + w];
  for (int x = first; x < min(first + each, span); ++x) {
    run[x] = upto;
    upto += (double)sSum[x];
    if (x == span - 1) run[span] = upto;
  }
  __syncthreads();
  const double lefts = (sFar[0] + sFar[2]) + (sFar[4] + sFar[6]), rights = (sFar[1] + sFar[3]) + (sFar[5] + sFar[7]);
  for (int n = tid; n < a.nb; n += 256) {
    if (n != tid) lo = a.bucket_range[2 * n], end = a.bucket_range[2 * n + 1];
    double y = 0.;
    if (lo < end && end > -a.mde && lo <= a.mde) {  // the ends hold everything beyond them
      y = run[end > a.mde ? span : end + a.mde + RB_PAD] - run[lo <= -a.mde ? 0 : lo + a.mde + RB_PAD];
      if (lo <= -a.mde) y += lefts;
      if (end > a.mde) y += rights;
    }
    a.part[((int64_t)h * a.nb + n) * nwg + wg] = (float)y;
  }
}

// dtable[n, h] = sum over the workgroups of head h, in 64 bits and a fixed order; one wave per entry
DEV void table_sum(const RbArgs& a, int entry, int nwg) {
  if (entry >= a.nb * a.H) return;
  const int lane = threadIdx.x & 63, h = entry / a.nb, n = entry % a.nb;
  double s = 0.;
  for (int x = lane; x < nwg; x += 64) s += (double)a.part[(int64_t)entry * nwg + x];
  s = wave_total(s);
  if (lane == 0) a.dtable[n * a.H + h] = (float)s;
}

// dk and dv: 4 waves x 32 keys of one (sequence, key head) against 64-query tiles of every head of its group.
//   S = Q K^T (+ bias), dV^T += dO^T P, dP = dO V^T (from -delta), dK^T += Q^T dS
// P and dS are rounded to the tensors' type as operands, the sums are f32.  Operands are requested ahead of their products through
// a whole sub-tile, which else waited for LDS twelve times (6001 x 6001, 8 heads of 64: 214 -> 202 us, 730 TFLOP/s of its four products).
// WIDE: K and the sums are 160 of 256 registers, V stays in LDS and tiles have 32 rows (2 x 2047 causal, 4 key heads of 128: 91 us,
// 750 TFLOP/s; with V in registers one wave a SIMD remains: 107).  32 x 400, 4 heads: 26 us.  Both units are busy for 35% of the
// 6001 x 6001 case: its 376 workgroups leave every second SIMD with one wave, and 220 registers allow no third.  fp16: the factors of
// P and dS (fit) take 242 us instead of 228 there, 110 instead of 108 at 128 columns.  Where few workgroups would run, the (head, query tile) steps are split over `nsplit`
// workgroups, whose sums rb_dkv_join_kernel adds in order.
template <class E, int DP>
__global__ __launch_bounds__(256, 2) void rb_dkv_kernel(RbArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  if ((int)blockIdx.x >= a.nblk) {  // more table entries than waves (few keys)
    table_sum(a, blockIdx.x * 4 + (threadIdx.x >> 6), a.B * a.nqtile);
    return;
  }
  constexpr bool WIDE = DP == 128;
  constexpr int ROWS = WIDE ? 32 : 64, P = 2 * DP, TILE = ROWS * P, NK = DP / 16, ND = DP / 32;
  unsigned char* const sQ = smem;
  unsigned char* const sO = smem + 2 * TILE;
  unsigned char* const sV = smem + 4 * TILE;  // [128 keys] of V (WIDE)
  float* const sL = reinterpret_cast<float*>(sV + (WIDE ? 128 * P : 0));  // [2][2][64] lse2 | -delta of a tile's rows
  float* const sB = sL + 256;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hi = lane >> 5, n32 = lane & 31;
  const Place at = place_of(a);
  const Quot bh = split(at.head, a.per_head);
  const int part = at.part, tile = at.rank, b = bh.q, hk = bh.r, G = a.per_group.d;
  const Seq sq = seq_of(a, b);
  const int k0 = tile * 128, j0 = k0 + wave * 32, j = j0 + n32;
  u32x4 kf[NK], vf[WIDE ? 1 : NK];
  row_frags<DP>(a.k + b * a.sk.b + hk * a.sk.h, a.sk.t, j0, sq.klen, a.D, lane, kf);
  if constexpr (!WIDE) row_frags<DP>(a.v + b * a.sv.b + hk * a.sv.h, a.sv.t, j0, sq.klen, a.D, lane, vf);
  f32x16 dk[ND], dv[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) dk[d] = dv[d] = splat16(0.f);
  // causal: the first query that sees key k0 sits at position k0.  Steps are numbered head by head.
  const int t0 = a.causal ? max(k0 - sq.off, 0) / ROWS : 0;
  const int per = k0 < sq.klen ? max((sq.qlen + ROWS - 1) / ROWS - t0, 0) : 0, steps = per * G;
  const int it0 = (int)((int64_t)steps * part / a.nsplit), it1 = (int)((int64_t)steps * (part + 1) / a.nsplit);
  const unsigned lQ = lds_addr(sQ), lO = lds_addr(sO);
  LaneAt<DP> in(smem, lane);
  const unsigned stats = lds_addr(sL) + hi * 16;   // row statistics: a lane reads four rows at a time
  const unsigned mine = 4 * TILE + wave * 32 * P;  // the wave's keys of V
  if constexpr (WIDE) {
    if (it0 < it1) {  // arrives with the first tile
      TileDma<DP> dV;
      dV.init(a.v + b * a.sv.b + hk * a.sv.h, a.sv.t, 2 * tile, sq.klen, a.D, wave, lane);
      dV.next(lds_addr(sV), wave);
      dV.next(lds_addr(sV) + 64 * P, wave);
    }
  }
  float lrow = 0.f, fac = RB_FAC0, facP = RB_FAC0;  // of the rounded dS and P (fp16)

  for (int it = it0; it < it1;) {
    const int g = it / per, ta = t0 + it % per, tb = min(t0 + per, ta + it1 - it);  // one head's run of tiles
    it += tb - ta;
    const int h = hk * G + g;
    TileDma<DP, ROWS> dQ, dO;
    dQ.init(a.q + b * a.sq.b + h * a.sq.h, a.sq.t, ta, sq.qlen, a.D, wave, lane);
    dO.init(a.dout + b * a.sdo.b + h * a.sdo.h, a.sdo.t, ta, sq.qlen, a.D, wave, lane);
    const float* const rl = (wave == 0 ? a.lse2 : a.delta) + ((int64_t)b * a.H + h) * a.tq128;  // two waves bring a tile's row statistics
    auto load = [&](int t, int buf) {
      dQ.next(lQ + buf * TILE, wave);
      dO.next(lO + buf * TILE, wave);
      if (wave < 2) lrow = rl[t * ROWS + (lane & (ROWS - 1))];
    };
    auto store = [&](int buf) {
      if (wave < 2) sL[buf * 128 + wave * 64 + lane] = lrow;
    };
    __syncthreads();  // the head before has been read
    load(ta, 0);
    spread_table(a, h, sB, reinterpret_cast<float*>(sQ + TILE), TILE / 4, tid);
    store(0);
    dma_wait();
    __syncthreads();
    const float left = sB[0], right = sB[2 * (a.mde + RB_PAD)];
    auto step = [&](int t, auto parity) {
      constexpr int buf = decltype(parity)::value;
      const bool more = t + 1 < tb;
      if (more) load(t + 1, buf ^ 1);
      constexpr unsigned qt = buf * TILE, ot = (2 + buf) * TILE;
#pragma unroll
      for (int u = 0; u < ROWS / 32; ++u) {
        const int p0 = sq.off + t * ROWS + 32 * u;  // position of the sub-tile's first query
        if (j0 >= sq.klen || (a.causal && j0 > p0 + 31)) continue;
        if (WIDE) in.renew();
        // The operands in the order of their products, requested RING ahead: rows of q, rows of dout (WIDE: each with its piece of
        // V), dout transposed, q transposed.  The exponentials stand between the products of dP, P (dP - delta) between those of dV.
        constexpr int ROW2 = WIDE ? 2 * NK : NK, N2 = NK + ROW2, N3 = N2 + 2 * ND, N4 = N3 + 2 * ND, RING = WIDE ? 4 : 6;
        auto fetch = [&](int n) {
          if (n < NK) return in.frag(qt, 32 * u, n);
          if (n < N2) return WIDE && (n & 1) ? in.frag(mine, 0, (n - NK) >> 1) : in.frag(ot, 32 * u, WIDE ? (n - NK) >> 1 : n - NK);
          const int x = n < N3 ? n - N2 : n - N3;
          return in.frag_t(n < N3 ? ot : qt, 32 * u + 16 * (x / ND), x % ND);
        };
        auto row4 = [&](int first) { return *(const lds_f32x4*)(uintptr_t)(stats + (buf * 128 + 32 * u + first) * 4); };
        u32x4 ring[RING];
        f32x16 s, dp;
        f32x4 ls[4];
        if (j0 - (p0 + 31) >= a.mde || j0 + 31 - p0 <= -a.mde) {
          s = splat16(j0 > p0 ? right : left);
        } else {
          const float* const bp = sB + (j - p0 - 4 * hi + a.mde + RB_PAD);
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = bp[-(8 * (r >> 2) + (r & 3))];
        }
#pragma unroll
        for (int n = 0; n < RING; ++n) ring[n] = fetch(n);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < NK; ++n) {
          s = E::mma(ring[n % RING], kf[n], s);
          ring[n % RING] = fetch(n + RING);
          if (n % (NK / 2) == 0) {
#pragma unroll
            for (int g = 4 * n / NK; g < 4 * n / NK + 2; ++g) {
              const f32x4 y = row4(64 + 8 * g);
#pragma unroll
              for (int r = 0; r < 4; ++r) dp[4 * g + r] = y[r];
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if (a.causal && j0 + 31 > p0) {
          const int lim = j - p0 - 4 * hi;  // queries before it do not see the key
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (8 * (r >> 2) + (r & 3) < lim) s[r] = -RB_INF;
        }
        constexpr int EACH = 16 / NK;  // exponentials behind a product; their rows' sums are requested two products ahead
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (4 * g < 2 * EACH) ls[g] = row4(8 * g);
#pragma unroll
        for (int n = 0; n < NK; ++n) {
          if constexpr (WIDE) {
            const int x = NK + 2 * n;
            dp = E::mma(ring[x % RING], ring[(x + 1) % RING], dp);
            ring[x % RING] = fetch(x + RING);
            ring[(x + 1) % RING] = fetch(x + 1 + RING);
          } else {
            dp = E::mma(ring[(NK + n) % RING], vf[n], dp);
            ring[(NK + n) % RING] = fetch(NK + n + RING);
          }
#pragma unroll
          for (int g = 0; g < 4; ++g)
            if (4 * g >= (n + 2) * EACH && 4 * g < (n + 3) * EACH) ls[g] = row4(8 * g);
#pragma unroll
          for (int r = n * EACH; r < (n + 1) * EACH; ++r) s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.c2, -ls[r >> 2][r & 3]));
          __builtin_amdgcn_sched_barrier(0);
        }
        float each = 1.f;  // from P as it is multiplied to dS's factor
        if constexpr (E::narrow) {
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] *= facP;
          fit(s, dv, facP);
          each = fac * __uint_as_float(0x7f000000u - __float_as_uint(facP));  // (fac / facP: the reciprocal of a power of two)
        }
        u32x4 xb[2] = {pack8<E>(s, 0), pack8<E>(s, 8)};
#pragma unroll
        for (int n = 0; n < 2 * ND; ++n) {
          dv[n % ND] = E::mma(ring[(N2 + n) % RING], xb[n / ND], dv[n % ND]);
          if (N2 + n + RING < N4) ring[(N2 + n) % RING] = fetch(N2 + n + RING);
          constexpr int M = 8 / ND;
#pragma unroll
          for (int r = n * M; r < (n + 1) * M; ++r) dp[r] *= E::narrow ? s[r] * each : s[r];
          __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (E::narrow) fit(dp, dk, fac);
        xb[0] = pack8<E>(dp, 0), xb[1] = pack8<E>(dp, 8);
#pragma unroll
        for (int n = 0; n < 2 * ND; ++n) {
          dk[n % ND] = E::mma(ring[(N3 + n) % RING], xb[n / ND], dk[n % ND]);
          if (N3 + n + RING < N4) ring[(N3 + n) % RING] = fetch(N3 + n + RING);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (more) store(buf ^ 1);
      dma_wait();
      __syncthreads();
    };
    for (int t = ta; t < tb; t += 2) {
      step(t, Const<0>{});
      if (t + 1 < tb) step(t + 1, Const<1>{});
    }
  }
  if constexpr (E::narrow) {
    const float f = 1.f / fac, fP = 1.f / facP;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) dk[d][r] *= f, dv[d][r] *= fP;
  }
  table_sum(a, blockIdx.x * 4 + wave, a.B * a.nqtile);  // each wave one entry of the table's gradient, from the dq kernel's shares
  if (j >= a.Tk) return;
  if (a.nsplit > 1) {  // sums in f32: [split][dk | dv][sequence, key head, key][DP]
    const int64_t rows = (int64_t)a.B * a.Hk * a.Tk, row = ((int64_t)b * a.Hk + hk) * a.Tk + j;
    float* const pk = a.part2 + ((int64_t)part * 2 * rows + row) * DP;
    float* const pv = pk + rows * DP;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = 32 * d + 8 * g + 4 * hi;
        *reinterpret_cast<f32x4*>(pk + c) = f32x4{dk[d][4 * g], dk[d][4 * g + 1], dk[d][4 * g + 2], dk[d][4 * g + 3]};
        *reinterpret_cast<f32x4*>(pv + c) = f32x4{dv[d][4 * g], dv[d][4 * g + 1], dv[d][4 * g + 2], dv[d][4 * g + 3]};
      }
    return;
  }
  const bool key = j < sq.klen;  // rows behind the sequence get zeros
  uint16_t* const kp = a.dk + b * a.sdk.b + (int64_t)j * a.sdk.t + hk * a.sdk.h;
  uint16_t* const vp = a.dv + b * a.sdv.b + (int64_t)j * a.sdv.t + hk * a.sdv.h;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = 32 * d + 8 * g + 4 * hi;
      if (c >= a.D) continue;
      float x[8];
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = key ? dk[d][4 * g + r] * a.scale : 0.f, x[4 + r] = key ? dv[d][4 * g + r] : 0.f;
      store4<E>(kp + c, x[0], x[1], x[2], x[3]);
      store4<E>(vp + c, x[4], x[5], x[6], x[7]);
    }
}

// dk and dv from the splits' sums, in order; a thread has 4 elements of one row of one of the two
template <class E, int DP>
__global__ __launch_bounds__(256) void rb_dkv_join_kernel(RbArgs a) {
  const int64_t rows = (int64_t)a.B * a.Hk * a.Tk, x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t r2 = x / (DP / 4);
  const int c = (int)(x % (DP / 4)) * 4;
  if (r2 >= 2 * rows || c >= a.D) return;
  const int64_t row = r2 % rows, bh = row / a.Tk;
  const int j = (int)(row % a.Tk), b = (int)(bh / a.Hk), hk = (int)(bh % a.Hk);
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.nsplit; ++s) y += *reinterpret_cast<const f32x4*>(a.part2 + ((int64_t)s * 2 * rows + r2) * DP + c);
  const bool key = r2 < rows;
  const Strides st = key ? a.sdk : a.sdv;
  if (key) y *= a.scale;
  if (j >= seq_of(a, b).klen) y = f32x4{0.f, 0.f, 0.f, 0.f};
  store4<E>((key ? a.dk : a.dv) + b * st.b + (int64_t)j * st.t + hk * st.h + c, y[0], y[1], y[2], y[3]);
}

// dq from the splits' sums, in order; a thread has 4 elements of one row
template <class E, int DP>
__global__ __launch_bounds__(256) void rb_dq_join_kernel(RbArgs a) {
  const int64_t rows = (int64_t)a.B * a.H * a.Tq, x = (int64_t)blockIdx.x * 256 + threadIdx.x, row = x / (DP / 4);
  const int c = (int)(x % (DP / 4)) * 4;
  if (row >= rows || c >= a.D) return;
  const int64_t bh = row / a.Tq;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.nsplit; ++s) y += *reinterpret_cast<const f32x4*>(a.part2 + ((int64_t)s * rows + row) * DP + c);
  y *= a.scale;
  store4<E>(a.dq + bh / a.H * a.sdq.b + row % a.Tq * a.sdq.t + bh % a.H * a.sdq.h + c, y[0], y[1], y[2], y[3]);
}

// =============================================================================================== host side
bool strides_ok(const int64_t* s, int D) {
  // 16-byte rows that do not overlap; a tile of 64 rows must stay within a 31-bit byte offset
  return s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0 && s[1] >= D && s[1] < (1 << 23) && s[0] >= 0 && s[2] >= 0;
}
Strides to_strides(const int64_t* s) { return Strides{s[0], s[1], s[2]}; }

int check_args(const csship_relbias* p) {
  if (p == nullptr) return CSSHIP_ENULL;
  if (p->B < 0 || p->Tq < 0 || p->Tk < 0 || p->H < 1 || p->Hk < 1 || p->H % p->Hk != 0) return CSSHIP_EBADSHAPE;
  if (p->Tq > RB_MAX_POS || p->Tk > RB_MAX_POS) return CSSHIP_EBADSHAPE;
  if ((int64_t)p->B * p->H * ((int64_t)(p->Tq > p->Tk ? p->Tq : p->Tk) + 128) > 0x7fffffff) return CSSHIP_EBADSHAPE;
  if (p->D < 8 || p->D > 128 || p->D % 8 != 0) return CSSHIP_EUNSUPPORTED;
  if (p->dtype != CSSHIP_RELBIAS_BF16 && p->dtype != CSSHIP_RELBIAS_FP16) return CSSHIP_EUNSUPPORTED;
  if (p->n_buckets < 2 || p->n_buckets > 32767 || p->max_distance < 1 || p->max_distance > CSSHIP_RELBIAS_MAX_DISTANCE)
    return CSSHIP_EUNSUPPORTED;
  if ((int64_t)p->n_buckets * p->H > 0x7fffffff) return CSSHIP_EBADSHAPE;  // the table's indexes are 32-bit
  if (!(p->scale > 1e-6f && p->scale < 1e6f)) return CSSHIP_EUNSUPPORTED;
  if (p->table == nullptr || p->bucket_of == nullptr) return CSSHIP_ENULL;
  const bool rows = p->B > 0 && p->Tq > 0, keys = p->B > 0 && p->Tk > 0;
  if ((rows && p->q == nullptr) || (keys && (p->k == nullptr || p->v == nullptr))) return CSSHIP_ENULL;
  if (!aligned16(p->q) || !aligned16(p->k) || !aligned16(p->v)) return CSSHIP_EALIGN;
  if (!strides_ok(p->q_stride, p->D) || !strides_ok(p->k_stride, p->D) || !strides_ok(p->v_stride, p->D)) return CSSHIP_EALIGN;
  return CSSHIP_OK;
}

// the largest distance whose table entry a call can need: with one offset for all sequences, no pair is further apart than this
int reach(const csship_relbias* p) {
  if (p->offsets != nullptr) return p->max_distance;
  const int off = p->offset < -RB_MAX_POS ? -RB_MAX_POS : p->offset > RB_MAX_POS ? RB_MAX_POS : p->offset;
  const int back = p->Tq - 1 + off, front = p->Tk - 1 - off, far = (back > front ? back : front) + 1;
  return far < 1 ? 1 : far < p->max_distance ? far : p->max_distance;
}

RbArgs to_args(const csship_relbias* p) {
  RbArgs a{};
  a.q = p->q; a.k = p->k; a.v = p->v;
  a.sq = to_strides(p->q_stride); a.sk = to_strides(p->k_stride); a.sv = to_strides(p->v_stride);
  a.table = p->table; a.bucket_of = p->bucket_of; a.bucket_range = p->bucket_range;
  a.k_lens = p->k_lens; a.q_lens = p->q_lens; a.offsets = p->offsets;
  a.B = p->B; a.Tq = p->Tq; a.Tk = p->Tk; a.H = p->H; a.Hk = p->Hk; a.D = p->D;
  a.nb = p->n_buckets; a.md = p->max_distance; a.mde = reach(p); a.causal = p->causal != 0; a.offset = p->offset;
  a.scale = p->scale; a.inv_scale = 1.f / p->scale; a.c2 = p->scale * RB_LOG2E;
  return a;
}

size_t fwd_lds(int DP, int md) { return (size_t)4 * 64 * 2 * DP + (2 * (md + RB_PAD) + 1) * 4; }
size_t dq_lds(int DP, int md) { return (size_t)4 * 64 * 2 * DP + (size_t)(md + RB_PAD + 1) * 16 + 8192 + 96; }
size_t dkv_lds(int DP, int md) { return fwd_lds(DP, md) + 1024; }

// launches with more than 64 KB of LDS have to be allowed, per device: asked for at each such launch
template <class K>
int launch(K kernel, int64_t blocks, size_t lds, RbArgs a, int heads, hipStream_t s, int threads = 256) {
  if (a.nsplit < 1) a.nsplit = 1;
  a.per_tile.set(a.ntile < 1 ? 1 : a.ntile);
  a.per_head.set(heads);
  a.per_group.set(a.H / a.Hk);
  a.per_split.set(a.nsplit);
  if (lds > 64 * 1024 &&
      hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess)
    return CSSHIP_ELAUNCH;
  kernel<<<(unsigned)blocks, threads, lds, s>>>(a);
  CSSHIP_CHECK_LAUNCH();
  return CSSHIP_OK;
}

// Which forward: rb_fwd_kernel reuses a K / V tile for 128 queries, rb_few_kernel for 32 rows but takes all heads of a group at
// once and may split the keys.  The latter from 256 keys on, where the former would leave most of the chip idle (4 heads of 64,
// 256 x 1000: 12.2 us against 20.5; 2000 x 2000, 64 workgroups: 26.9 against 35.9) or most of its 128 rows empty (16 x 16 heads
// in groups of 4, 20 x 2000: 22.4 against 33.3).  At 256 keys both take 8 us, at 64 the former 5 and the latter 6.7.
struct FwdPlan { bool few; int ntile, nsplit; };
FwdPlan fwd_plan(const csship_relbias* p) {
  const int64_t rows = (int64_t)p->Tq * (p->H / p->Hk), tiles = (rows + 31) / 32, wide = (int64_t)p->B * p->H * ((p->Tq + 127) / 128);
  FwdPlan f{p->Tk >= 256 && (p->Tq <= 32 || wide < 128), (int)tiles, 1};
  if (f.few && p->Tk > 1024) {  // up to there no second launch pays: 4 x 8 heads, 256 x 1000: 14.2 us against 22.1 split at 256
    const int64_t want = 768 / ((int64_t)p->B * p->Hk * tiles), most = (p->Tk + 511) / 512;
    f.nsplit = (int)(want < 1 ? 1 : want < most ? want : most);
  }
  return f;
}
int width_of(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }

template <class E, int DP>
int launch_fwd(RbArgs a, const csship_relbias* p, hipStream_t s) {
  const FwdPlan f = fwd_plan(p);
  if (f.few) {
    a.ntile = f.ntile;
    a.nsplit = f.nsplit;
    a.nblk = a.B * a.Hk * a.ntile * a.nsplit;
    const int table = (a.H / a.Hk) * (2 * a.mde + 1), staged = table <= RB_FEW_TABLE ? table * 4 : 0;
    // few workgroups: twice the waves, half the tiles for each (1 x 500 keys, 4 heads: 8.5 us for 9.9)
    const int rc = a.nblk < 256 ? launch(rb_few_kernel<E, DP, 8>, a.nblk, few_area<DP, 8>() + staged, a, a.Hk, s, 512)
                                : launch(rb_few_kernel<E, DP, 4>, a.nblk, few_area<DP, 4>() + staged, a, a.Hk, s);
    if (rc) return rc;
    if (a.nsplit == 1) return CSSHIP_OK;
    return launch(rb_join_kernel<E, DP>, ((int64_t)a.B * a.H * a.Tq + 3) / 4, 0, a, a.H, s);
  }
  a.ntile = (a.Tq + 127) / 128;
  a.nblk = a.B * a.H * a.ntile;
  if (a.nblk == 0) return CSSHIP_OK;
  return launch(rb_fwd_kernel<E, DP>, a.nblk, fwd_lds(DP, a.mde), a, a.H, s);
}

// Workgroups of the dk / dv kernel take 128 keys of a sequence and key head; where those leave most of the chip idle, each one's
// steps (64 queries of one head) are split, up to 512 workgroups and not below 4 steps (2 x 2047 causal, 4 key heads of 128,
// backward: 189 us; up to 256: 227, up to 768: 190; 1 x 3000, 8 heads sharing one key head: 122, 128, 129).
int dkv_splits(const csship_relbias* p) {
  const int64_t wgs = (int64_t)p->B * p->Hk * ((p->Tk + 127) / 128), steps = (int64_t)(p->H / p->Hk) * ((p->Tq + 63) / 64);
  if (wgs == 0) return 1;
  const int64_t want = 512 / wgs, most = steps / 4 < 32 ? steps / 4 : 32;
  return (int)(want < 1 || most < 1 ? 1 : want < most ? want : most);
}

// The same for the dq kernel's 128 queries and their keys (64 at a time), up to 768 workgroups and not below 2 steps
// (6001 x 6001, 8 heads, backward: 333 us; up to 512, no split there: 341; both with two waves a SIMD).
int dq_splits(const csship_relbias* p) {
  const int64_t wgs = (int64_t)p->B * p->H * ((p->Tq + 127) / 128), steps = (p->Tk + 63) / 64;
  if (wgs == 0) return 1;
  const int64_t want = 768 / wgs, most = steps / 2 < 8 ? steps / 2 : 8;
  return (int)(want < 1 || most < 1 ? 1 : want < most ? want : most);
}

template <class E, int DP>
int launch_bwd(RbArgs a, const csship_relbias* p, hipStream_t s) {
  a.ntile = (a.Tq + 127) / 128;
  a.tq128 = a.ntile * 128;
  a.nsplit = dq_splits(p);
  a.nqtile = a.ntile * a.nsplit;
  a.nblk = a.B * a.H * a.nqtile;
  if (a.nblk > 0) {
    const int rc = DP == 64 && a.nblk > 512 ? launch(rb_dq_kernel<E, DP, DP == 64 ? 3 : 2>, a.nblk, dq_lds(DP, a.mde), a, a.H, s)
                                            : launch(rb_dq_kernel<E, DP, 2>, a.nblk, dq_lds(DP, a.mde), a, a.H, s);
    if (rc) return rc;
    if (a.nsplit > 1)
      if (const int rc = launch(rb_dq_join_kernel<E, DP>, ((int64_t)a.B * a.H * a.Tq * (DP / 4) + 255) / 256, 0, a, a.H, s)) return rc;
  }
  // (part2 again: the dq kernel's sums have been joined)
  a.ntile = (a.Tk + 127) / 128;
  a.nsplit = dkv_splits(p);
  a.nblk = a.B * a.Hk * a.ntile * a.nsplit;
  const int64_t entries = ((int64_t)a.nb * a.H + 3) / 4;
  if (const int rc = launch(rb_dkv_kernel<E, DP>, a.nblk > entries ? a.nblk : entries, dkv_lds(DP, a.mde), a, a.Hk, s)) return rc;
  if (a.nsplit == 1) return CSSHIP_OK;
  return launch(rb_dkv_join_kernel<E, DP>, ((int64_t)2 * a.B * a.Hk * a.Tk * (DP / 4) + 255) / 256, 0, a, a.Hk, s);
}

template <class E>
int fwd_by_width(const RbArgs& a, const csship_relbias* p, hipStream_t s) {
  return a.D <= 32 ? launch_fwd<E, 32>(a, p, s) : a.D <= 64 ? launch_fwd<E, 64>(a, p, s) : launch_fwd<E, 128>(a, p, s);
}
template <class E>
int bwd_by_width(const RbArgs& a, const csship_relbias* p, hipStream_t s) {
  return a.D <= 32 ? launch_bwd<E, 32>(a, p, s) : a.D <= 64 ? launch_bwd<E, 64>(a, p, s) : launch_bwd<E, 128>(a, p, s);
}

int64_t row_words(const csship_relbias* p) { return (int64_t)p->B * p->H * ((p->Tq + 127) / 128 * 128); }

// the table gradient's shares: one number per workgroup of the dq kernel and bucket, in whole 16 bytes
int64_t part_words(const csship_relbias* p) {
  return ((int64_t)p->B * p->H * ((p->Tq + 127) / 128) * dq_splits(p) * p->n_buckets + 3) / 4 * 4;
}

}  // namespace

extern "C" {

size_t csship_relbias_fwd_workspace(const csship_relbias* p) {
  if (check_args(p) != CSSHIP_OK || p->B == 0 || p->Tq == 0) return 0;
  const FwdPlan f = fwd_plan(p);
  return f.nsplit == 1 ? 0 : (size_t)p->B * p->H * p->Tq * f.nsplit * (width_of(p->D) + 2) * 4;
}

int csship_relbias_fwd(const csship_relbias* p, uint16_t* out, const int64_t* out_stride, float* lse, void* workspace,
                       size_t workspace_bytes, csship_stream_t stream) {
  if (const int rc = check_args(p)) return rc;
  const size_t need = csship_relbias_fwd_workspace(p);
  if (need > 0 && workspace == nullptr) return CSSHIP_ENULL;
  if (workspace_bytes < need) return CSSHIP_EWORKSPACE;
  if (!aligned16(workspace)) return CSSHIP_EALIGN;
  if (p->B == 0 || p->Tq == 0) return CSSHIP_OK;
  if (out == nullptr || out_stride == nullptr) return CSSHIP_ENULL;
  if (!aligned8(out) || !strides_ok(out_stride, p->D)) return CSSHIP_EALIGN;
  RbArgs a = to_args(p);
  a.out = out;
  a.so = to_strides(out_stride);
  a.lse = lse;
  a.part = static_cast<float*>(workspace);
  return p->dtype == CSSHIP_RELBIAS_BF16 ? fwd_by_width<ElemBf>(a, p, as_stream(stream)) : fwd_by_width<ElemHf>(a, p, as_stream(stream));
}

size_t csship_relbias_bwd_workspace(const csship_relbias* p) {
  if (check_args(p) != CSSHIP_OK) return 0;
  const int splits = dkv_splits(p);
  const int qsplits = dq_splits(p);
  const int64_t sums_k = splits == 1 ? 0 : (int64_t)splits * 2 * p->B * p->Hk * p->Tk * width_of(p->D);
  const int64_t sums_q = qsplits == 1 ? 0 : (int64_t)qsplits * p->B * p->H * p->Tq * width_of(p->D);
  const int64_t sums = sums_k > sums_q ? sums_k : sums_q;  // one after the other in the same memory
  return (size_t)(2 * row_words(p) + part_words(p) + sums) * 4 + 16;
}

int csship_relbias_bwd(const csship_relbias* p, const uint16_t* out, const int64_t* out_stride, const float* lse, const uint16_t* dout,
                       const int64_t* dout_stride, uint16_t* dq, const int64_t* dq_stride, uint16_t* dk, const int64_t* dk_stride,
                       uint16_t* dv, const int64_t* dv_stride, float* dtable, void* workspace, size_t workspace_bytes,
                       csship_stream_t stream) {
  if (const int rc = check_args(p)) return rc;
  if ((int64_t)p->n_buckets * p->H > (1 << 26) - 4) return CSSHIP_EBADSHAPE;  // a wave for each entry: fewer than 2^32 threads
  const bool rows = p->B > 0 && p->Tq > 0, keys = p->B > 0 && p->Tk > 0;
  if (p->bucket_range == nullptr || dtable == nullptr || out_stride == nullptr || dout_stride == nullptr || dq_stride == nullptr ||
      dk_stride == nullptr || dv_stride == nullptr || workspace == nullptr)
    return CSSHIP_ENULL;
  if ((rows && (out == nullptr || lse == nullptr || dout == nullptr || dq == nullptr)) || (keys && (dk == nullptr || dv == nullptr)))
    return CSSHIP_ENULL;
  if (!aligned16(out) || !aligned16(dout) || !aligned8(dq) || !aligned8(dk) || !aligned8(dv) || !aligned16(workspace)) return CSSHIP_EALIGN;
  if (!strides_ok(out_stride, p->D) || !strides_ok(dout_stride, p->D) || !strides_ok(dq_stride, p->D) || !strides_ok(dk_stride, p->D) || !strides_ok(dv_stride, p->D))
    return CSSHIP_EALIGN;
  if (workspace_bytes < csship_relbias_bwd_workspace(p)) return CSSHIP_EWORKSPACE;
  RbArgs a = to_args(p);
  a.o = out; a.so = to_strides(out_stride);
  a.dout = dout; a.sdo = to_strides(dout_stride);
  a.lse_in = lse;
  a.dq = dq; a.sdq = to_strides(dq_stride);
  a.dk = dk; a.sdk = to_strides(dk_stride);
  a.dv = dv; a.sdv = to_strides(dv_stride);
  a.dtable = dtable;
  a.delta = static_cast<float*>(workspace);
  a.lse2 = a.delta + row_words(p);
  a.part = a.lse2 + row_words(p);
  a.part2 = a.part + part_words(p);
  return p->dtype == CSSHIP_RELBIAS_BF16 ? bwd_by_width<ElemBf>(a, p, as_stream(stream)) : bwd_by_width<ElemHf>(a, p, as_stream(stream));
}

}  // extern "C"
