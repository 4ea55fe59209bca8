// Attention over a KV cache held in MXFP4 (format: mxfp4.h): decode steps and
// prefill chunks. Keys and values are (B, Hkv, cap, D) with a row's codes (D / 2
// bytes) and scales (D / 32 bytes) packed, blocks along the head dim.
//
// Decode (q3_decode_attention_mxfp4): per query head
//   s_j = scale q . k_j,  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  m = max_j s_j
// over the sequence's rows, in one pass with a running m, sum and o in fp32.
//
//  * Work units are 32-row tiles of a (sequence, KV head) pair. Where pairs are many or
//    rows few (pair_waves), a block takes one pair, its waves equal ranges of the units,
//    and their sums meet in LDS. Otherwise all units, listed pair-major, are split
//    between all waves in ranges of equal length, so ragged lengths cost nothing: a pair
//    that one wave finishes is stored at once, one split between waves leaves a record
//    (m, sum, o) per wave (record wave + pair, unique and increasing in both), merged by
//    mx_decode_combine. Every wave finds its range by itself: no barrier, and no block
//    waits for another.
//  * The up to 16 columns of a 16x16x32 MFMA are the query heads of the group
//    (times the tokens of a short chunk); larger groups take several columns
//    sets, each a pair of its own.
//  * A unit's codes and scales go global -> LDS past the registers into one of the
//    wave's two ring slots while it works on the other; 12 waves per CU keep 52 KB
//    in flight. Lane (r = l % 16, g = l / 16) then reads bytes [g D/8, (g + 1) D/8) of
//    row r, which lie in one block of 32, and converts them into A operands of S^T = K
//    Q^T (the k index of a product is any permutation of the head dim, the same for K
//    and Q).
//  * V is needed transposed (A operand rows = head dim): a tile's values are
//    converted by the same lanes, written over the slot's codes as bf16 rows, 16 at a
//    time, and read with ds_read_b64_tr_b16. P^T comes straight from the S^T
//    accumulators (lane (c, g) holds rows 4 g + i and 16 + 4 g + i of column c; V's
//    fragment reads follow that order).
//  * P is rounded to bf16 for the second product (at most 2^-8 of each weight), as in the
//    kernels of the bf16 cache; q, K and V enter exactly; m, the sum and o are fp32. The
//    roundings of a row's weights are independent, so numerator and error shrink alike and
//    the share stays: the outputs are 0.0023 of their norm from float64, 0.0017 of which
//    their own rounding to bf16 makes. P in two bf16 terms would leave those 0.0017 alone
//    and takes a second product per tile of V: the 32 sequences below 43.9 -> 46.1 us
//    with the merge, 37 tokens on 4 x 2000 rows 23.3 -> 25.0.
//
// Measured (us; the floor is the cache's bytes at 6.5 TB/s, what such a read reaches
// here): 32 sequences of 8 KV heads x 4, lengths to 8192, 138 MB of rows in use 31 and 6
// for the merge (floor 21), 178 MB 36.5 and 5.7 (27); one of 1500 rows, 1.6 MB: 5.6 and
// 4.5, all of it latency; a block per pair, 32 sequences to 2000: 19 (split 23.5); 64
// tokens on 4 x 2000 rows (512 pairs of 16 columns, which read the same rows from the
// L2): 27 (split 37).
#include <algorithm>
#include <type_traits>

#include "gemm_tile.h"
#include "mxfp4.h"

namespace {

using namespace q3;

constexpr int kUnit = 32;        // rows of a unit
constexpr int kMaxBatch = 1024;  // sequences
constexpr int kCols = 16;        // MFMA columns
constexpr int kWavesPerBlock = 12;  // three per SIMD, one block per CU
constexpr int kBlocks = 256;
constexpr int kSlots = 2;  // ring slots of a wave: the unit at hand and the next
constexpr int kWaves = kBlocks * kWavesPerBlock;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescale = 8.0f;  // log2 units the running max may lag behind

typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

struct MxAttn {
  const bf16* q;
  const uint8_t *kc, *ks, *vc, *vs;
  bf16* o;
  int B, Hkv, groups, Sq;
  int nset;             // column sets per KV head
  int cap;              // rows a sequence may have
  int64_t qb, qh, qs, ob, oh, os;
  int64_t kcb, kch, ksb, ksh, vcb, vch, vsb, vsh;  // bytes
  const int* lens;
  int len_add;          // token i sees lens[b] + len_add + i rows
  int* lens_inc;        // if set, lens_inc[b] += inc once the call has read the lengths
  int inc;
  float scale_log2;
  int* hdr;             // workspace: unit prefix over sequences (B + 1)
  float* rec;           // workspace: records
};

// A record: m[kCols], sum[kCols], o[kCols][D], fp32.
__host__ __device__ constexpr int rec_floats(int D) { return kCols * (D + 2); }

__device__ __forceinline__ int rows_of(const MxAttn& p, int b) {
  return (int)min(max((int64_t)p.lens[b] + p.len_add + p.Sq - 1, (int64_t)0), (int64_t)p.cap);
}

__device__ __forceinline__ int units_of(const MxAttn& p, int b) { return (rows_of(p, b) + kUnit - 1) / kUnit; }

// U units over n waves: the first U % n take one more than the others. Up to 512 units
// have a wave each; more units take more waves only while each has at least 8 units, as
// every wave that shares a pair costs the merge a record (8 units against 1, in us with the
// merge, 8 KV heads of 4: one sequence of 8192 rows 12.2 / 14.0, of 16 tokens 22.5 / 26.5,
// of 64 46.4 / 46.0; 8 of 8192 24.2 / 25.4; 16 of 3000 x 4 heads of 8 19.4 / 23.7; 32 of
// 8192, where all waves are full, 57.9 / 58.1).
constexpr int kMinWaves = 512, kMinUnits = 8;
struct Split {
  int n, q, r;
  __device__ __forceinline__ explicit Split(int U) {
    n = min(kWaves, max(U / kMinUnits, min(U, kMinWaves)));
    q = n ? U / n : 0;
    r = U - n * q;
  }
  __device__ __forceinline__ int first(int w) const { return w * q + min(w, r); }
  __device__ __forceinline__ int wave_of(int u) const {
    const int big = r * (q + 1);
    return u < big ? u / (q + 1) : r + (u - big) / q;
  }
};

struct Cursor {
  int b, hs, tile, nb;  // sequence, KV head and column set, tile, tiles of the sequence
};

// Inclusive sum over the wave's lanes.
__device__ __forceinline__ int wave_scan(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_up(v, o, 64);
    if (lane >= o) v += x;
  }
  return v;
}

// Over the lanes l % 16 = c, whose l / 16 hold the same column.
__device__ __forceinline__ float max4(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  x = fmaxf(__builtin_bit_cast(float, a[0]), __builtin_bit_cast(float, a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  return fmaxf(__builtin_bit_cast(float, b[0]), __builtin_bit_cast(float, b[1]));
}

// LDS element of value d of row r (0..15) of the V rows being transposed. A row's
// 16-byte chunk c sits at slot c ^ swizzle(r), so that the 16 rows of a write (one
// chunk each) and of a transposed read (two neighbouring chunks each) use all banks.
template <int D>
__device__ __forceinline__ int v_at(int r, int d) {
  const int sw = D == 128 ? (((r & 7) << 1) | (r >> 3)) : (r & 7);
  return r * D + ((((d >> 3) ^ sw) << 3) | (d & 7));
}

__device__ __forceinline__ short4v read_tr16(const bf16* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (short4v __attribute__((address_space(3)))*)(reinterpret_cast<uintptr_t>(p)));
}

// LDS of a wave: kSlots slots, each the unit's codes as the lanes read them (K then
// V, 32 rows) and a word with the scales of each K and each V row. Once those are in
// registers, the slot holds 16 rows of V in bf16 at a time.
template <int D>
struct WaveLds {
  static constexpr int kCodes = kUnit * D / 2;  // bytes of K's codes
  static constexpr int kSlot = 2 * kCodes + 256;
  static constexpr int kBytes = kSlots * kSlot;
  static_assert(16 * D * 2 <= 2 * kCodes, "the rows of V being transposed");
};

// PW = 0: the units of all pairs split between all waves. PW > 0: a block of PW waves takes one pair, each wave an
// equal range of its units; their sums meet in LDS and the block stores the pair's outputs. ONCE: the rows are read
// once (non-temporal loads).
template <int D, bool ONCE, int PW>
__global__ __launch_bounds__(64 * (PW ? PW : kWavesPerBlock)) void mx_decode_kernel(const MxAttn p) {
  constexpr int LB = D / 8;         // bytes of codes a lane takes of a row
  constexpr int LW = LB / 4;        // the same in words: A fragments of 8 values
  constexpr int DT = D / 16;        // output tiles along the head dim
  constexpr int NB = D / kMxBlock;  // blocks of a row
  constexpr int PIECES = D / 64;    // 16-byte loads per lane of a unit's K (or V) codes
  constexpr int LOADS = 2 * PIECES + 1;
  typedef WaveLds<D> Lds;
  typedef uint32_t words __attribute__((ext_vector_type(LW)));
  __shared__ __attribute__((aligned(1024))) char s_mem[(PW ? PW : kWavesPerBlock) * Lds::kBytes];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int HS = p.Hkv * p.nset;

  int w = 0, count;  // the wave among all, and its units
  Cursor cc{};
  if constexpr (PW > 0) {
    cc.b = (int)blockIdx.x / HS;
    cc.hs = (int)blockIdx.x - cc.b * HS;
    cc.nb = units_of(p, cc.b);
    cc.tile = cc.nb * wave / PW;
    count = cc.nb * (wave + 1) / PW - cc.tile;
  } else {
    // The wave's units: every wave sums the sequences' unit counts by itself (64 a
    // round), so nothing waits at a barrier.
    const bool first_wave = blockIdx.x == 0 && wave == 0;
    int total = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
      const int incl = wave_scan(b0 + lane < p.B ? units_of(p, b0 + lane) : 0, lane);
      if (first_wave && b0 + lane < p.B) p.hdr[b0 + lane + 1] = total + incl;  // for the merge, which must not read the lengths
      total += __builtin_amdgcn_readlane(incl, 63);
    }
    if (first_wave && lane == 0) p.hdr[0] = 0;
    const Split split(total * HS);
    // Blocks run round-robin on the 8 XCDs. Each XCD takes an eighth of the active waves,
    // consecutive ones (which read the same rows where there are several column sets) on
    // different CUs.
    const int xcd = blockIdx.x & 7, j = wave * (kBlocks / 8) + ((int)blockIdx.x >> 3);
    const int here = split.n / 8 + (xcd < split.n % 8);
    if (j >= here) return;
    w = xcd * (split.n / 8) + min(xcd, split.n % 8) + j;
    const int u0 = split.first(w);
    count = split.first(w + 1) - u0;
    for (int b0 = 0, before = 0; b0 < p.B; b0 += 64) {
      const int n = b0 + lane < p.B ? units_of(p, b0 + lane) : 0;
      const int incl = before + wave_scan(n, lane);
      const int at = __popcll(__builtin_amdgcn_ballot_w64(incl * HS <= u0));  // sequences that end at or before u0
      if (at < 64) {
        cc.b = b0 + at;
        cc.nb = __builtin_amdgcn_readlane(n, at);
        const int r = u0 - (__builtin_amdgcn_readlane(incl, at) - cc.nb) * HS;
        cc.hs = r / cc.nb;
        cc.tile = r - cc.hs * cc.nb;
        break;
      }
      before = __builtin_amdgcn_readlane(incl, 63);
    }
  }
  char* mem = s_mem + wave * Lds::kBytes;
  const uint32_t lmem = lds_addr(mem);

  auto advance = [&](Cursor& x) {  // to the next pair
    x.tile = 0;
    if (++x.hs < HS) return;
    x.hs = 0;
    do {
      ++x.b;
      x.nb = x.b < p.B ? units_of(p, x.b) : 1;
    } while (x.nb == 0);
  };

  // The pair whose units are being loaded. The codes' buffers end after the sequence's
  // rows: what lies behind (and, past the wave's range, everything) reads as zeros
  // without memory traffic; scales behind repeat the last row's.
  Cursor ic = cc;
  __amdgpu_buffer_rsrc_t rk, rv;
  const uint8_t* sp;  // lanes 0-31 the K, 32-63 the V scales of the pair
  int last = 0;       // last row
  auto open = [&](const Cursor& x) {
    const int kvh = __builtin_amdgcn_readfirstlane(x.hs / p.nset), b = __builtin_amdgcn_readfirstlane(x.b);
    const int64_t n = __builtin_amdgcn_readfirstlane(rows_of(p, b));
    rk = make_rsrc(p.kc + b * p.kcb + kvh * p.kch, n * (D / 2));
    rv = make_rsrc(p.vc + b * p.vcb + kvh * p.vch, n * (D / 2));
    sp = lane < 32 ? p.ks + b * p.ksb + kvh * p.ksh : p.vs + b * p.vsb + kvh * p.vsh;
    last = (int)n - 1;
  };
  // Piece of the codes a lane fetches: with D = 128 the one it will use itself (16
  // bytes of row c), with D = 64 chunk g / 2 of row l % 32.
  const uint32_t c_off = D == 128 ? c * 64 + g * 16 : (lane & 31) * 32 + (lane >> 5) * 16;
  auto issue = [&](bool live, int slot) {
    const uint32_t at = lmem + slot;
    const uint32_t row = ic.tile * kUnit;
    auto codes = [&](__amdgpu_buffer_rsrc_t r, uint32_t to) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const uint32_t off = live ? (row + 16 * i) * (D / 2) + c_off : kOOB;
        if constexpr (ONCE) dma16_nt(r, off, to + 1024 * i);
        else dma16(r, off, to + 1024 * i);
      }
    };
    codes(rk, at);
    codes(rv, at + Lds::kCodes);
    const uint8_t* from = sp + (int64_t)min((int)row + (lane & 31), last) * NB;
    if constexpr (D == 128) dma4_at(from, at + 2 * Lds::kCodes);
    else dma2_at(from, at + 2 * Lds::kCodes);
  };
  // Lane's codes of row 16 i + c, and its block's scale, from a slot.
  auto codes_at = [&](const char* slot, int i) {
    const int off = D == 128 ? 1024 * i + 16 * lane : ((g >> 1) * 32 + 16 * i + c) * 16 + (g & 1) * 8;
    return *reinterpret_cast<const words*>(slot + off);
  };

  bf16x8 qf[LW];
  floatx4 o[DT];
  float m = -INFINITY, lsum = 0.f;
  int vis = 0;  // rows this lane's column sees
  bool valid = false;
  int64_t o_off = 0;
  auto start = [&](const Cursor& x) {  // the query columns of a pair, and empty statistics
    const int kvh = x.hs / p.nset, col = (x.hs - kvh * p.nset) * kCols + c;
    const int tok = col / p.groups, hd = col - tok * p.groups;
    valid = tok < p.Sq;
    const int64_t head = (int64_t)kvh * p.groups + hd;
    const bf16* q = p.q + x.b * p.qb + head * p.qh + tok * p.qs;
    o_off = x.b * p.ob + head * p.oh + tok * p.os;
    vis = (int)min((int64_t)p.lens[x.b] + p.len_add + tok, (int64_t)p.cap);
#pragma unroll
    for (int t = 0; t < LW; ++t) {
      qf[t] = bf16x8{};
      if (valid) qf[t] = *reinterpret_cast<const bf16x8*>(q + g * (2 * LB) + 8 * t);
    }
    // Waited for here: a use of loads that may still be under way makes the compiler wait
    // for every load, the ring's included, before the first products of each unit.
#pragma unroll
    for (int t = 0; t < LW; ++t) asm volatile("" : "+v"(qf[t]));
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = floatx4{};
    m = -INFINITY;
    lsum = 0.f;
  };
  auto flush = [&](const Cursor& x, bool whole) {
    if constexpr (PW > 0) return;
    lsum += __shfl_xor(lsum, 16, 64);
    lsum += __shfl_xor(lsum, 32, 64);
    if (!valid) return;
    if (whole) {
      const float inv = lsum != 0.f ? 1.0f / lsum : 0.f;  // a NaN sum stays one
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        bf16x4 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = f2bf(o[t][e] * inv);
        *reinterpret_cast<bf16x4*>(p.o + o_off + 16 * t + 4 * g) = r;
      }
    } else {
      float* rec = p.rec + ((int64_t)w + (int64_t)x.b * HS + x.hs) * rec_floats(D);
      if (g == 0) {
        rec[c] = m;
        rec[kCols + c] = lsum;
      }
#pragma unroll
      for (int t = 0; t < DT; ++t) *reinterpret_cast<floatx4*>(rec + 2 * kCols + c * D + 16 * t + 4 * g) = o[t];
    }
  };

  start(cc);  // its loads before the ring's: loads retire in order
  if constexpr (PW > 0) {
    if (cc.nb == 0) {  // an empty sequence: zeros
      if (valid && wave == 0)
#pragma unroll
        for (int t = 0; t < DT; ++t) *reinterpret_cast<bf16x4*>(p.o + o_off + 16 * t + 4 * g) = bf16x4{};
      return;
    }
  }
  open(ic);
  int issued = 0, islot = 0, slot_at = 0;
  auto issue_next = [&]() {
    issue(issued < count, islot);
    islot = islot == (kSlots - 1) * Lds::kSlot ? 0 : islot + Lds::kSlot;
    if (++issued < count && ++ic.tile == ic.nb) {
      advance(ic);
      open(ic);
    }
  };
#pragma unroll 1
  for (int i = 0; i < kSlots - 1; ++i) issue_next();
  int first = cc.tile;  // tile of the current pair at which this wave began
  for (int u = 0; u < count; ++u) {
    issue_next();
    vm_wait<(kSlots - 1) * LOADS>();  // this unit's loads have landed
    char* slot = mem + slot_at;
    slot_at = slot_at == (kSlots - 1) * Lds::kSlot ? 0 : slot_at + Lds::kSlot;
    const uint8_t* sc = reinterpret_cast<const uint8_t*>(slot + 2 * Lds::kCodes) + 4 * c + g * NB / 4;
    const words kw[2] = {codes_at(slot, 0), codes_at(slot, 1)};
    const words vw[2] = {codes_at(slot + Lds::kCodes, 0), codes_at(slot + Lds::kCodes, 1)};
    const uint32_t kb[2] = {sc[0], sc[64]}, vb[2] = {sc[128], sc[192]};
    asm volatile("" ::: "memory");  // read before V's rows take their place (the LDS works in a wave's order)
    bf16* tile = reinterpret_cast<bf16*>(slot);

    floatx4 s[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s[i] = floatx4{};
      const float ks = mx_scale(kb[i]);
#pragma unroll
      for (int t = 0; t < LW; ++t) s[i] = mfma16x16x32(mx_bf16x8(kw[i][t], ks), qf[t], s[i]);
    }
    const int seen = vis - cc.tile * kUnit - 4 * g;  // this lane's rows are 16 i + e
    if (__builtin_amdgcn_ballot_w64(seen < 20) != 0) {  // a unit that some column sees in part
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (16 * i + e >= seen) s[i][e] = -INFINITY;
    }

    // V^T fragments: rows 0-15, then 16-31 (the LDS of a wave works in order). A NaN
    // block (scale 255) counts as zeros here: a masked one must not reach a column
    // through 0 * NaN.
    const int rr = c >> 2, qq = c & 3;
    uint64_t bad[2];
    short4v vf[DT][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      bad[i] = __builtin_amdgcn_ballot_w64(vb[i] == 255);
      const float vs = mx_scale(vb[i] == 255 ? 0 : vb[i]);
#pragma unroll
      for (int t = 0; t < LW; ++t)
        *reinterpret_cast<bf16x8*>(tile + v_at<D>(c, g * (2 * LB) + 8 * t)) = mx_bf16x8(vw[i][t], vs);
#pragma unroll
      for (int t = 0; t < DT; ++t) vf[t][i] = read_tr16(tile + v_at<D>(4 * g + rr, 16 * t + 4 * qq));
    }

    float top = s[0][0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, s[i >> 2][i & 3]);
    top = max4(top) * p.scale_log2;
    const bool raise = top > m + kRescale;
    if (__builtin_amdgcn_ballot_w64(raise) != 0) {
      const float mn = raise ? top : m;
      const float alpha = mn == -INFINITY ? 1.f : exp2_(m - mn);
      lsum *= alpha;
#pragma unroll
      for (int t = 0; t < DT; ++t) o[t] *= alpha;
      m = mn;
    }
    const float base = m == -INFINITY ? 0.f : m;  // a column that has seen no row yet: weights 0, not NaN
    bf16x8 pb;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = exp2_(fmaf(s[i >> 2][i & 3], p.scale_log2, -base));
      lsum += e;
      pb[i] = f2bf(e);
    }
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      const short4v lo = vf[t][0], hi = vf[t][1];
      const short8v a8 = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      o[t] = mfma16x16x32(__builtin_bit_cast(bf16x8, a8), pb, o[t]);
    }
    if ((bad[0] | bad[1]) != 0) {  // rare: the NaN blocks of rows that a column sees
      uint32_t see[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) see[i] = (1u << min(max(seen - 16 * i, 0), 4)) - 1;
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const int at = 16 * (4 * n / NB) + 4 * g;  // bit of row 4 g in the ballot, among the lanes of block n
        const uint32_t hit = ((uint32_t)(bad[0] >> at) & see[0]) | ((uint32_t)(bad[1] >> at) & see[1]);
        float add = hit ? NAN : 0.f;
        add += __shfl_xor(add, 16, 64);
        add += __shfl_xor(add, 32, 64);
#pragma unroll
        for (int t = n * DT / NB; t < (n + 1) * DT / NB; ++t) o[t] += add;
      }
    }

    if (cc.tile + 1 == cc.nb || u + 1 == count) {
      flush(cc, first == 0 && cc.tile + 1 == cc.nb);
      if (u + 1 < count) {
        advance(cc);
        start(cc);
        first = 0;
      }
    } else {
      ++cc.tile;
    }
  }
  vm_wait<0>();  // no load may still target this block's LDS when the wave retires
  if constexpr (PW > 0) {  // this wave's statistics and sums over its slots: m[kCols], sum[kCols], o[kCols][D]
    constexpr int N = D / 64;  // outputs per lane
    typedef float outs __attribute__((ext_vector_type(N)));
    static_assert(rec_floats(D) * 4 <= Lds::kBytes, "a wave's sums take the place of its slots");
    lsum += __shfl_xor(lsum, 16, 64);
    lsum += __shfl_xor(lsum, 32, 64);
    asm volatile("" ::: "memory");
    float* rec = reinterpret_cast<float*>(mem);
    if (g == 0) {
      rec[c] = m;
      rec[kCols + c] = lsum;
    }
#pragma unroll
    for (int t = 0; t < DT; ++t) *reinterpret_cast<floatx4*>(rec + 2 * kCols + c * D + 16 * t + 4 * g) = o[t];
    __syncthreads();
    const int kvh = cc.hs / p.nset, col0 = (cc.hs - kvh * p.nset) * kCols;
    for (int col = wave; col < kCols; col += PW) {
      const int tok = (col0 + col) / p.groups, hd = col0 + col - tok * p.groups;
      if (tok >= p.Sq) break;
      auto rec_of = [&](int k) { return reinterpret_cast<const float*>(s_mem + k * Lds::kBytes); };
      float top = -INFINITY;
#pragma unroll
      for (int k = 0; k < PW; ++k) top = fmaxf(top, rec_of(k)[col]);
      if (top == -INFINITY) top = 0.f;  // no row seen: weights 0, not NaN
      float sum = 0.f;
      outs v{};
#pragma unroll
      for (int k = 0; k < PW; ++k) {
        const float r = exp2_(rec_of(k)[col] - top);
        sum += rec_of(k)[kCols + col] * r;
        v += *reinterpret_cast<const outs*>(rec_of(k) + 2 * kCols + col * D + N * lane) * r;
      }
      const float inv = sum != 0.f ? 1.0f / sum : 0.f;  // a NaN sum stays one
      bf16* y = p.o + cc.b * p.ob + ((int64_t)kvh * p.groups + hd) * p.oh + tok * p.os + N * lane;
#pragma unroll
      for (int e = 0; e < N; ++e) y[e] = f2bf(v[e] * inv);
    }
  }
}

// Advances the lengths, behind a launch whose blocks all read them.
__global__ void mx_advance_kernel(int* lens, int B, int inc) {
  const int b = blockIdx.x * 64 + threadIdx.x;
  if (b < B) lens[b] += inc;
}

// Merges the records of the pairs split between waves: a block per pair and column,
// its NW waves every NW-th record each, kBatch of them in flight together (the merge
// is bound by latency), and the waves' sums in wave order.
constexpr int kBatch = 4;

template <int D, int NW>
__global__ __launch_bounds__(64 * NW) void mx_decode_combine(const MxAttn p) {
  constexpr int N = D / 64;  // outputs per lane
  typedef float outs __attribute__((ext_vector_type(N)));
  __shared__ float s_m[NW], s_l[NW];
  __shared__ outs s_o[NW][64];
  const int HS = p.Hkv * p.nset, pair = blockIdx.x;
  const int b = pair / HS, hs = pair - b * HS;
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = blockIdx.y;
  if (p.lens_inc && hs == 0 && col == 0 && threadIdx.x == 0) p.lens_inc[b] += p.inc;
  const int u0 = p.hdr[b], u1 = p.hdr[b + 1], units = p.hdr[p.B];
  const int kvh = hs / p.nset, gc = (hs - kvh * p.nset) * kCols + col;
  const int tok = gc / p.groups, hd = gc - tok * p.groups;
  if (tok >= p.Sq) return;
  bf16* orow = p.o + b * p.ob + ((int64_t)kvh * p.groups + hd) * p.oh + tok * p.os + N * lane;
  auto store = [&](outs o) {
#pragma unroll
    for (int e = 0; e < N; ++e) orow[e] = f2bf(o[e]);
  };
  if (u0 == u1) {  // an empty sequence: zeros
    if (wv == 0) store(outs{});
    return;
  }
  const Split split(HS * units);
  const int first = HS * u0 + hs * (u1 - u0);
  const int w0 = split.wave_of(first), w1 = split.wave_of(first + (u1 - u0) - 1);
  if (w0 == w1) return;  // stored by its wave
  float m = -INFINITY, l = 0.f;
  outs o{};
  for (int wb = w0 + wv; wb <= w1; wb += NW * kBatch) {
    float mr[kBatch], lr[kBatch];
    outs orr[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int w = min(wb + NW * i, w1);
      const float* rec = p.rec + (int64_t)(w + pair) * rec_floats(D);
      mr[i] = rec[col];
      lr[i] = rec[kCols + col];
      orr[i] = *reinterpret_cast<const outs*>(rec + 2 * kCols + col * D + N * lane);
    }
    float mn = m;
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (wb + NW * i <= w1) mn = fmaxf(mn, mr[i]);
    const float base = mn == -INFINITY ? 0.f : mn;  // no row seen yet: weights 0, not NaN
    const float a = exp2_(m - base);
    l *= a;
    o *= a;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (wb + NW * i > w1) break;
      const float r = exp2_(mr[i] - base);
      l += lr[i] * r;
      o += orr[i] * r;
    }
    m = mn;
  }
  if (lane == 0) {
    s_m[wv] = m;
    s_l[wv] = l;
  }
  s_o[wv][lane] = o;
  __syncthreads();
  if (wv != 0) return;
#pragma unroll
  for (int i = 1; i < NW; ++i) m = fmaxf(m, s_m[i]);
  if (m == -INFINITY) m = 0.f;
  l = 0.f;
  o = outs{};
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const float r = exp2_(s_m[i] - m);
    l += s_l[i] * r;
    o += s_o[i][lane] * r;
  }
  store(o * (l != 0.f ? 1.0f / l : 0.f));
}

int64_t header_bytes(int64_t B) { return (B + 1 + 63) / 64 * 256; }

int64_t sets_of(int64_t groups, int64_t Sq) { return q3_cdiv(groups * Sq, kCols); }

// The streaming kernel takes single tokens, chunks of few pairs, and chunks of few column
// sets per KV head. Otherwise the cache is expanded to bf16 once and the chunk kernel of
// the bf16 cache runs.
//
// Few pairs: the chunk kernel shares each row among 256 columns but does not split the
// rows, so its time grows with the rows until the pairs fill the card, the streaming
// kernel's with pairs x rows. Microseconds, streaming / expanding, 8 KV heads of 4 query
// heads unless said otherwise: 8192 rows, 32 tokens (64 pairs) 38 / 209, 128 (256) 53 /
// 213, 512 (1024) 160 / 214, 700 (1400) 219 / 215, 1000 (2000) 279 / 216; 4 x 2000 rows,
// 64 tokens (512) 27 / 72, 200 (1600) 54 / 73, 300 (2432) 84 / 73; 1024 rows, 256 tokens
// (512) 20 / 41, 512 (1024) 34 / 42; 8 x 300 rows of 4 x 8 heads, 60 tokens (960) 21 / 28,
// 100 (1600) 28 / 29, 150 (2400) 37 / 30.
//
// Few sets: the streaming kernel reads and converts a row once per 16 columns of its KV
// head, while the expansion moves 4.8 times the bytes of the rows to make them bf16 and
// the chunk kernel reads those, however few columns there are. The same, by sets per KV
// head, 1 / 4 / 8 / 12 / 16: 256 sequences x 8 KV heads of 8192 rows 389 / 1258 / 2440 /
// 3403 / 4374 against 3776 / 3904 / 3921 / 4100 / 4121 (and 8.6 GB), of 300 rows 35 / 103 /
// 194 / 288 / 385 against 193 / 212 / 229 / 256 / 276; 32 x 8 of 2000, from 4 on: 57 / 95 /
// 127 / 163 against 124 / 126 / 141 / 154; D = 64, 256 x 8 of 2000: 59 / 186 / 363 / 539 /
// 684 against 596 / 573 / 591 / 624 / 632.
constexpr int64_t kStreamPairs = 1400, kStreamSets = 12;
bool streams(int64_t B, int64_t Hkv, int64_t groups, int64_t Sq) {
  const int64_t sets = sets_of(groups, Sq);
  return Sq == 1 || sets <= kStreamSets || B * Hkv * sets <= kStreamPairs;
}

// Waves of a block that takes one pair, or 0 to split all units between all waves and merge records. Pairs per
// block save the records and the merge, but each pair's rows go through few waves: right for few rows, for many pairs,
// and the more columns a pair has (its records are that much larger). Rows are the capacity, as the lengths are on the
// device. Both kernels, us, split / 8 waves / 4 waves: decode of 4 heads to a KV head, 8 pairs of 300 rows 11.0 / 10.3
// / 9.7, 1000 11.3 / 13.0 / 13.1; 64 pairs, 500 12.9 / 10.8 / 10.5, 1500 15.1 / 15.5 / 18.0; 256 pairs, 300 15.8 /
// 10.7 / 9.6, 2000 23.5 / 18.8 / 21.5; 512 pairs, 1000 24.6 / 22.3 / 18.5, 4000 42.7 / 48.9 / 44.0; 1024 pairs,
// 1000 30.6 / 39.5 / 28.5, 4000 67 / 83 / 71; chunks of 16 columns, 128 pairs of 1024 rows 27.7 / 14.7 / 14.5, 304 of
// 2000 31.9 / 24.8 / 25.0, 512 of 2000 37.6 / 32.5 / 26.1, 256 of 8192 58.7 / 49.9 / 65.6, 1024 of 8192 161 / 180 / 153.
int pair_waves(int64_t pairs, int64_t cap, int64_t cols) {
  if (cap > std::min<int64_t>(512 + 2 * cols * pairs, 640 * cols)) return 0;
  return pairs <= 320 && cap > 1024 ? 8 : 4;
}

int64_t stream_ws_bytes(int64_t B, int64_t Hkv, int64_t groups, int64_t Sq, int64_t D, int64_t cap) {
  const int64_t pairs = B * Hkv * sets_of(groups, Sq);
  if (pair_waves(pairs, cap, std::min<int64_t>(kCols, groups * Sq))) return 0;
  return header_bytes(B) + (kWaves + pairs) * (int64_t)rec_floats((int)D) * 4;
}

template <int D, int PW>
void launch_pairs(const MxAttn& p, int pairs, hipStream_t st) {
  if (p.nset == 1)  // every row is read once
    hipLaunchKernelGGL((mx_decode_kernel<D, true, PW>), dim3((unsigned)pairs), dim3(64 * PW), 0, st, p);
  else
    hipLaunchKernelGGL((mx_decode_kernel<D, false, PW>), dim3((unsigned)pairs), dim3(64 * PW), 0, st, p);
}

template <int D>
int launch_stream(const MxAttn& p, hipStream_t st) {
  const int pairs = p.B * p.Hkv * p.nset;
  const int cols = std::min(kCols, p.groups * p.Sq);
  if (const int waves = pair_waves(pairs, p.cap, cols)) {
    if (waves == 8)
      launch_pairs<D, 8>(p, pairs, st);
    else
      launch_pairs<D, 4>(p, pairs, st);
    Q3_LAUNCH_CHECK();
    if (p.lens_inc) {
      hipLaunchKernelGGL(mx_advance_kernel, dim3((unsigned)q3_cdiv(p.B, 64)), dim3(64), 0, st, p.lens_inc, p.B, p.inc);
      Q3_LAUNCH_CHECK();
    }
    return Q3_OK;
  }
  const dim3 grid(kBlocks), block(64 * kWavesPerBlock);
  if (p.nset == 1)  // every row is read once
    hipLaunchKernelGGL((mx_decode_kernel<D, true, 0>), grid, block, 0, st, p);
  else
    hipLaunchKernelGGL((mx_decode_kernel<D, false, 0>), grid, block, 0, st, p);
  Q3_LAUNCH_CHECK();
  const dim3 merge((unsigned)pairs, (unsigned)cols);
  // The merge is bound by latency: all of a pair's records should be in flight at once and all blocks resident.
  // A pair has up to kWaves / pairs records: 16 waves share more than 16 of them (8 pairs of one sequence's 1500
  // rows: 4.4 us against 6.3 on 4), 4 waves fewer (256 pairs of 32 sequences: 5.6 us, 8.5 on 16 and on 1), one wave
  // where 4 to each pair and column would not fit the card (320 pairs x 16 columns: 7.3 us against 10.2 on 4).
  if (kWaves / pairs > 16)
    hipLaunchKernelGGL((mx_decode_combine<D, 16>), merge, dim3(64 * 16), 0, st, p);
  else if ((int64_t)pairs * merge.y > 256 * 8)
    hipLaunchKernelGGL((mx_decode_combine<D, 1>), merge, dim3(64), 0, st, p);
  else
    hipLaunchKernelGGL((mx_decode_combine<D, 4>), merge, dim3(64 * 4), 0, st, p);
  Q3_LAUNCH_CHECK();
  return Q3_OK;
}

int launch_stream(const MxAttn& p, int64_t D, hipStream_t st) {
  return D == 128 ? launch_stream<128>(p, st) : launch_stream<64>(p, st);
}

// Arguments that both entry points take; strides = [qb, qh, qs, ob, oh, os] in
// elements, then [b, h] of k_codes, k_scales, v_codes, v_scales in bytes.
int check(const void* q, const void* kc, const void* ks, const void* vc, const void* vs, const int* lens,
          const void* o, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t D, int64_t cap,
          const int64_t* strides, float scale, int dtype) {
  Q3_REQUIRE(q && kc && ks && vc && vs && lens && o && strides, Q3_ERR_NULL);
  Q3_REQUIRE(B >= 0 && Hq >= 1 && Hkv >= 1 && Hq % Hkv == 0 && Sq >= 0 && D >= 1 && cap >= 0, Q3_ERR_SHAPE);
  // The kernels mask unscaled scores with -inf and take the running maximum of these: 0 would make a NaN of a masked
  // row, a negative scale an infinity.
  Q3_REQUIRE(scale > 0.f && scale < INFINITY, Q3_ERR_SHAPE);
  Q3_REQUIRE(dtype == Q3_BF16, Q3_ERR_DTYPE);
  Q3_REQUIRE((D == 64 || D == 128) && B <= kMaxBatch && (cap + kUnit) * D / 2 < (1ll << 31) && Sq < (1ll << 31) &&
                 Hq < (1ll << 16) && B * Hkv * sets_of(Hq / Hkv, streams(B, Hkv, Hq / Hkv, Sq) ? Sq : 1) * q3_cdiv(cap, kUnit) < (1ll << 31),
             Q3_ERR_UNSUPPORTED);
  bool ok = q3_aligned(q, 16) && q3_aligned(kc, 16) && q3_aligned(vc, 16) && q3_aligned(o, 8);
  for (int i = 0; i < 6; ++i) ok = ok && strides[i] % 8 == 0;
  for (int i : {6, 7, 10, 11}) ok = ok && strides[i] % 16 == 0;
  const int64_t row = D / kMxBlock;  // a row's scales are read at once
  ok = ok && q3_aligned(ks, row) && q3_aligned(vs, row);
  for (int i : {8, 9, 12, 13}) ok = ok && strides[i] % row == 0;
  return ok ? Q3_OK : Q3_ERR_ALIGN;
}

MxAttn arguments(const void* q, const void* kc, const void* ks, const void* vc, const void* vs, const int* lens,
                 void* o, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t cap, const int64_t* s, float scale) {
  MxAttn p{};
  p.q = static_cast<const bf16*>(q);
  p.kc = static_cast<const uint8_t*>(kc);
  p.ks = static_cast<const uint8_t*>(ks);
  p.vc = static_cast<const uint8_t*>(vc);
  p.vs = static_cast<const uint8_t*>(vs);
  p.o = static_cast<bf16*>(o);
  p.B = (int)B;
  p.Hkv = (int)Hkv;
  p.groups = (int)(Hq / Hkv);
  p.Sq = (int)Sq;
  p.nset = (int)sets_of(p.groups, Sq);
  p.cap = (int)cap;
  p.qb = s[0], p.qh = s[1], p.qs = s[2], p.ob = s[3], p.oh = s[4], p.os = s[5];
  p.kcb = s[6], p.kch = s[7], p.ksb = s[8], p.ksh = s[9];
  p.vcb = s[10], p.vch = s[11], p.vsb = s[12], p.vsh = s[13];
  p.lens = lens;
  p.scale_log2 = scale * kLog2e;
  return p;
}

void workspace_of(MxAttn& p, void* ws) {
  p.hdr = static_cast<int*>(ws);
  p.rec = reinterpret_cast<float*>(static_cast<char*>(ws) + header_bytes(p.B));
}

// 4.5 us for one sequence of 8192 rows x 8 heads, 1024 tokens, which reads 32 KB of scales.
// A NaN block of V in one of the chunk's own rows (the expansion made zeros of it, so
// that it does not reach the earlier tokens' 0 * NaN) into the outputs of the tokens
// from that row's on. lens[b] - off is the sequence's length before the chunk.
template <int D>
__global__ __launch_bounds__(256) void mx_chunk_nan_kernel(const MxAttn p, int off) {
  constexpr int NB = D / kMxBlock;
  __shared__ int s_first[NB];
  const int b = blockIdx.x / p.Hkv, kvh = blockIdx.x - b * p.Hkv;
  const int64_t len = max((int64_t)p.lens[b] - off, (int64_t)0);
  if (threadIdx.x < NB) s_first[threadIdx.x] = p.Sq;
  __syncthreads();
  typedef typename std::conditional<NB == 4, uint32_t, uint16_t>::type word;  // a row's scales
  const word* s = reinterpret_cast<const word*>(p.vs + b * p.vsb + kvh * p.vsh + len * NB);
  const int n = (int)max(min((int64_t)p.Sq, p.cap - len), (int64_t)0);
  for (int r0 = threadIdx.x; r0 < n; r0 += 4 * 256) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = s[min(r0 + 256 * i, n - 1)];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < NB; ++k)
        if ((w[i] >> (8 * k) & 255) == 255) atomicMin(&s_first[k], min(r0 + 256 * i, n - 1));
  }
  __syncthreads();
  for (int k = 0; k < NB; ++k)
    for (int64_t i = (int64_t)s_first[k] * p.groups + threadIdx.x / kMxBlock; i < (int64_t)p.Sq * p.groups;
         i += 256 / kMxBlock)
      p.o[b * p.ob + ((int64_t)kvh * p.groups + i % p.groups) * p.oh + (i / p.groups) * p.os + k * kMxBlock +
          threadIdx.x % kMxBlock] = f2bf(NAN);
}

}  // namespace

extern "C" {

int64_t q3_decode_attention_mxfp4_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t cap) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || cap < 0) return 0;
  return stream_ws_bytes(B, Hkv, Hq / Hkv, 1, D, cap);
}

int q3_decode_attention_mxfp4(const void* q, const void* k_codes, const void* k_scales, const void* v_codes,
                              const void* v_scales, int* kv_lens, int advance, void* o, int64_t B, int64_t Hq,
                              int64_t Hkv, int64_t D, int64_t cap, const int64_t* strides, float scale, int dtype,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check(q, k_codes, k_scales, v_codes, v_scales, kv_lens, o, B, Hq, Hkv, 1, D, cap, strides, scale,
                       dtype);
  if (rc != Q3_OK || B == 0) return rc;
  const int64_t need = q3_decode_attention_mxfp4_workspace_bytes(B, Hq, Hkv, D, cap);
  Q3_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), Q3_ERR_WORKSPACE);
  Q3_REQUIRE(need == 0 || q3_aligned(workspace, 16), Q3_ERR_ALIGN);
  MxAttn p = arguments(q, k_codes, k_scales, v_codes, v_scales, kv_lens, o, B, Hq, Hkv, 1, cap, strides, scale);
  p.len_add = advance ? 1 : 0;
  p.lens_inc = advance ? kv_lens : nullptr;
  p.inc = 1;
  workspace_of(p, workspace);
  return launch_stream(p, D, static_cast<hipStream_t>(stream));
}

int64_t q3_flash_attention_cache_mxfp4_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t D,
                                                       int64_t max_len) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Sq <= 0 || D <= 0 || max_len < 0) return 0;
  if (streams(B, Hkv, Hq / Hkv, Sq)) return stream_ws_bytes(B, Hkv, Hq / Hkv, Sq, D, max_len);
  return 2 * B * Hkv * max_len * D * 2;  // K and V in bf16
}

int q3_flash_attention_cache_mxfp4(const void* q, const void* k_codes, const void* k_scales, const void* v_codes,
                                   const void* v_scales, int* kv_lens, void* o, int64_t B, int64_t Hq, int64_t Hkv,
                                   int64_t Sq, int64_t D, int64_t max_len, const int64_t* strides, float scale,
                                   int advance, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  int rc =
      check(q, k_codes, k_scales, v_codes, v_scales, kv_lens, o, B, Hq, Hkv, Sq, D, max_len, strides, scale, dtype);
  if (rc != Q3_OK || B == 0 || Sq == 0) return rc;
  Q3_REQUIRE(Sq <= max_len, Q3_ERR_SHAPE);
  const int64_t need = q3_flash_attention_cache_mxfp4_workspace_bytes(B, Hq, Hkv, Sq, D, max_len);
  Q3_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), Q3_ERR_WORKSPACE);
  Q3_REQUIRE(need == 0 || q3_aligned(workspace, 16), Q3_ERR_ALIGN);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (streams(B, Hkv, Hq / Hkv, Sq)) {
    MxAttn p = arguments(q, k_codes, k_scales, v_codes, v_scales, kv_lens, o, B, Hq, Hkv, Sq, max_len, strides, scale);
    p.len_add = 1;
    p.lens_inc = advance ? kv_lens : nullptr;
    p.inc = (int)Sq;
    workspace_of(p, workspace);
    return launch_stream(p, D, st);
  }
  // A longer chunk reuses every row many times: the rows in use are expanded to
  // bf16 once (exact) and the chunk kernel of the bf16 cache runs on them.
  Q3_REQUIRE(B * Hkv <= 65535 && (max_len + 1) * D * 2 < 0x7fffffffLL, Q3_ERR_UNSUPPORTED);
  bf16* kx = static_cast<bf16*>(workspace);
  const bf16* vx = kx + B * Hkv * max_len * D;
  const int64_t cst[4] = {strides[6], strides[7], strides[10], strides[11]};
  const int64_t sst[4] = {strides[8], strides[9], strides[12], strides[13]};
  rc = mx_expand_cache(k_codes, k_scales, v_codes, v_scales, kx, B, Hkv, max_len, D, cst, sst, kv_lens,
                                (int)Sq, st);
  if (rc != Q3_OK) return rc;
  const int64_t rows[12] = {strides[0], strides[1], strides[2], Hkv * max_len * D, max_len * D, D,
                            Hkv * max_len * D, max_len * D, D, strides[3], strides[4], strides[5]};
  rc = q3_flash_attention_cache(q, kx, vx, kv_lens, o, B, Hq, Hkv, Sq, max_len, D, rows, scale, advance,
                                           dtype, stream);
  if (rc != Q3_OK) return rc;
  const MxAttn p =
      arguments(q, k_codes, k_scales, v_codes, v_scales, kv_lens, o, B, Hq, Hkv, Sq, max_len, strides, scale);
  const dim3 heads((unsigned)(B * Hkv));
  if (D == 128)
    hipLaunchKernelGGL((mx_chunk_nan_kernel<128>), heads, dim3(256), 0, st, p, advance ? (int)Sq : 0);
  else
    hipLaunchKernelGGL((mx_chunk_nan_kernel<64>), heads, dim3(256), 0, st, p, advance ? (int)Sq : 0);
  Q3_LAUNCH_CHECK();
  return Q3_OK;
}

}  // extern "C"
