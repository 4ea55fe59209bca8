// Attention over a KV cache held in MXFP4 (format: mxfp4.h): decode steps and
// prefill chunks. Keys and values are (B, Hkv, cap, D) with a row's codes (D / 2
// bytes) and scales (D / 32 bytes) packed, blocks along the head dim.
//
// Decode (q3_decode_attention_mxfp4): per query head
//   s_j = scale q . k_j,  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  m = max_j s_j
// over the sequence's rows, in one pass with a running m, sum and o in fp32.
//
//  * Work units are 32-row tiles of a (sequence, KV head) pair, listed pair-major;
//    each wave takes an equal contiguous range of all units, so ragged lengths
//    cost nothing. A pair that one wave finishes is stored at once; a pair split
//    between waves leaves a record (m, sum, o) per wave (record wave + pair, unique
//    and increasing in both), merged by mx_decode_combine.
//  * The up to 16 columns of a 16x16x32 MFMA are the query heads of the group
//    (times the tokens of a short chunk); larger groups take several columns
//    sets, each a pair of its own.
//  * 16 rows of K are 16 rows x D/2 bytes, contiguous: lane (r = l % 16, g = l / 16)
//    loads bytes [g D/8, (g + 1) D/8) of row r, which lie in one block of 32, and
//    converts them into A operands of S^T = K Q^T (the k index of a product is any
//    permutation of the head dim, the same for K and Q).
//  * V is needed transposed (A operand rows = head dim): a tile's values are
//    converted by the same lanes, written to the wave's LDS as bf16 rows and read
//    with ds_read_b64_tr_b16. P^T comes straight from the S^T accumulators (lane
//    (c, g) holds rows 4 g + i and 16 + 4 g + i of column c; V's fragment reads
//    follow that order).
//  * P is rounded to bf16 for the second product (relative 2^-9 each, averaged
//    over the rows: the output's own rounding to bf16 is larger); q, K and V enter
//    exactly; m, the sum and o are fp32.
#include <algorithm>

#include "gemm_tile.h"
#include "mxfp4.h"

namespace {

using namespace q3;

constexpr int kUnit = 32;        // rows of a unit
constexpr int kMaxBatch = 1024;  // sequences (their unit counts live in LDS)
constexpr int kCols = 16;        // MFMA columns
constexpr int kWavesPerBlock = 8;
constexpr int kBlocks = 512;
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

// Exclusive prefix of the sequences' unit counts in s_pre[0..B], their rows in s_len.
__device__ void unit_prefix(const MxAttn& p, int* s_pre, int* s_len, int* s_sum) {
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 63, wv = tid >> 6;
  const int per = (p.B + nt - 1) / nt;
  int local = 0;
  for (int i = 0; i < per; ++i) {
    const int b = tid * per + i;
    if (b < p.B) {
      const int n = rows_of(p, b);
      s_len[b] = n;
      local += (n + kUnit - 1) / kUnit;
    }
  }
  int incl = local;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(incl, o, 64);
    if (lane >= o) incl += v;
  }
  if (lane == 63) s_sum[wv] = incl;
  __syncthreads();
  int run = incl - local;
  for (int i = 0; i < wv; ++i) run += s_sum[i];
  for (int i = 0; i < per; ++i) {
    const int b = tid * per + i;
    if (b < p.B) {
      s_pre[b] = run;
      run += (s_len[b] + kUnit - 1) / kUnit;
    }
  }
  if (tid == nt - 1) s_pre[p.B] = run;
  __syncthreads();
}

// Unit u belongs to active wave ((u + 1) * n - 1) / U, n = min(U, waves) of them.
__device__ __forceinline__ int wave_of(int64_t u, int64_t U) {
  const int64_t n = min<int64_t>(U, kWaves);
  return (int)(((u + 1) * n - 1) / U);
}

struct Cursor {
  int b, hs, tile, nb;  // sequence, KV head and column set, tile, tiles of the sequence
};

// LDS element of value d of row r (0..31) in a wave's V tile. A row's 16-byte
// chunk c sits at slot c ^ swizzle(r), so that the 16 rows of a write (one chunk
// each) and of a transposed read (two neighbouring chunks each) use all banks.
template <int D>
__device__ __forceinline__ int v_at(int r, int d) {
  const int sw = D == 128 ? (((r & 7) << 1) | ((r >> 3) & 1)) : (r & 7);
  return r * D + ((((d >> 3) ^ sw) << 3) | (d & 7));
}

template <int D>
__global__ __launch_bounds__(64 * kWavesPerBlock, 2) void mx_decode_kernel(const MxAttn p) {
  constexpr int LB = D / 8;         // bytes of codes a lane takes of a row
  constexpr int LW = LB / 4;        // the same in words: A fragments of 8 values
  constexpr int DT = D / 16;        // output tiles along the head dim
  constexpr int NB = D / kMxBlock;  // blocks of a row
  typedef uint32_t words __attribute__((ext_vector_type(LW)));
  __shared__ int s_pre[kMaxBatch + 1];
  __shared__ int s_len[kMaxBatch];
  __shared__ int s_sum[kWavesPerBlock];
  __shared__ __attribute__((aligned(16))) bf16 s_v[kWavesPerBlock * kUnit * D];

  unit_prefix(p, s_pre, s_len, s_sum);
  if (blockIdx.x == 0)  // for the merge, which must not read the lengths
    for (int i = threadIdx.x; i <= p.B; i += blockDim.x) p.hdr[i] = s_pre[i];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int HS = p.Hkv * p.nset;
  const int64_t U = (int64_t)HS * s_pre[p.B];
  const int64_t nw = min<int64_t>(U, kWaves);
  const int w = blockIdx.x * kWavesPerBlock + wave;
  if (w >= nw) return;
  const int64_t u0 = (int64_t)w * U / nw, u1 = (int64_t)(w + 1) * U / nw;
  bf16* tile = s_v + wave * kUnit * D;

  Cursor cc;
  {
    int lo = 0, hi = p.B - 1;  // the largest b with HS * s_pre[b] <= u0
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((int64_t)HS * s_pre[mid] <= u0) lo = mid;
      else hi = mid - 1;
    }
    cc.b = lo;
    cc.nb = s_pre[lo + 1] - s_pre[lo];
    const int r = (int)(u0 - (int64_t)HS * s_pre[lo]);
    cc.hs = r / cc.nb;
    cc.tile = r - cc.hs * cc.nb;
  }
  auto advance = [&](Cursor& x) {
    if (++x.tile < x.nb) return;
    x.tile = 0;
    if (++x.hs < HS) return;
    x.hs = 0;
    do {
      ++x.b;
    } while (x.b < p.B && s_pre[x.b + 1] == s_pre[x.b]);
    x.nb = x.b < p.B ? s_pre[x.b + 1] - s_pre[x.b] : 0;
  };

  struct Tile {
    words k[2], v[2];
    uint32_t sk[2], sv[2];
  };
  // Rows past the sequence's end repeat its last row: read in bounds, masked below.
  auto load = [&](const Cursor& x, Tile& t) {
    const int n = s_len[x.b], kvh = x.hs / p.nset;
    const uint8_t* kc = p.kc + x.b * p.kcb + kvh * p.kch;
    const uint8_t* ks = p.ks + x.b * p.ksb + kvh * p.ksh;
    const uint8_t* vc = p.vc + x.b * p.vcb + kvh * p.vch;
    const uint8_t* vs = p.vs + x.b * p.vsb + kvh * p.vsh;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t row = min(x.tile * kUnit + 16 * i + c, n - 1);
      t.k[i] = __builtin_nontemporal_load(reinterpret_cast<const words*>(kc + row * (D / 2) + g * LB));
      t.v[i] = __builtin_nontemporal_load(reinterpret_cast<const words*>(vc + row * (D / 2) + g * LB));
      t.sk[i] = ks[row * NB + g * NB / 4];
      t.sv[i] = vs[row * NB + g * NB / 4];
    }
  };

  bf16x8 qf[LW];
  floatx4 o[DT];
  float m = -INFINITY, lsum = 0.f;
  int vis = 0;  // rows this lane's column sees
  bool valid = false;
  bf16* orow = nullptr;
  auto start = [&](const Cursor& x) {  // the query columns of a pair, and empty statistics
    const int kvh = x.hs / p.nset, col = (x.hs - kvh * p.nset) * kCols + c;
    const int tok = col / p.groups, hd = col - tok * p.groups;  // Sq = 1 or groups * Sq <= kCols
    valid = tok < p.Sq;
    const int64_t head = (int64_t)kvh * p.groups + hd;
    const bf16* q = p.q + x.b * p.qb + head * p.qh + tok * p.qs;
    orow = p.o + x.b * p.ob + head * p.oh + tok * p.os;
    vis = min((int)min((int64_t)p.lens[x.b] + p.len_add + tok, (int64_t)p.cap), s_len[x.b]);
#pragma unroll
    for (int t = 0; t < LW; ++t) {
      qf[t] = bf16x8{};
      if (valid) qf[t] = *reinterpret_cast<const bf16x8*>(q + g * (2 * LB) + 8 * t);
    }
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = floatx4{};
    m = -INFINITY;
    lsum = 0.f;
  };
  auto flush = [&](const Cursor& x, int64_t pair_u0) {
    lsum += __shfl_xor(lsum, 16, 64);
    lsum += __shfl_xor(lsum, 32, 64);
    if (pair_u0 >= u0 && pair_u0 + x.nb <= u1) {
      if (!valid) return;
      const float inv = lsum != 0.f ? 1.0f / lsum : 0.f;  // a NaN sum stays one
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        bf16x4 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = f2bf(o[t][e] * inv);
        *reinterpret_cast<bf16x4*>(orow + 16 * t + 4 * g) = r;
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

  int64_t pair_u0 = u0 - cc.tile;
  Tile cur, nxt;
  load(cc, cur);
  start(cc);
  for (int64_t u = u0; u < u1; ++u) {
    Cursor nc = cc;
    if (u + 1 < u1) advance(nc);
    load(nc, nxt);  // the last one's again past the range

    floatx4 s[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s[i] = floatx4{};
      const float ks = mx_scale(cur.sk[i]);
#pragma unroll
      for (int t = 0; t < LW; ++t) s[i] = mfma16x16x32(mx_bf16x8(cur.k[i][t], ks), qf[t], s[i]);
    }
    const int k0 = cc.tile * kUnit + 4 * g;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (k0 + 16 * i + e >= vis) s[i][e] = -INFINITY;
    // V rows whose block holds a NaN (scale 255) count as zeros in the product, and
    // the blocks become NaN in the columns that see such a row: a masked one must not
    // reach a column through 0 * NaN.
    uint64_t bad[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      bad[i] = __builtin_amdgcn_ballot_w64(cur.sv[i] == 255);
      const float vs = mx_scale(cur.sv[i]);
#pragma unroll
      for (int t = 0; t < LW; ++t) {
        bf16x8 v = mx_bf16x8(cur.v[i][t], vs);
        if (bad[i] != 0 && cur.sv[i] == 255) v = bf16x8{};
        *reinterpret_cast<bf16x8*>(tile + v_at<D>(16 * i + c, g * (2 * LB) + 8 * t)) = v;
      }
    }
    float top = s[0][0];
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, s[i >> 2][i & 3]);
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64)) * p.scale_log2;
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
    const int rr = c >> 2, qq = c & 3;
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((short4v __attribute__((address_space(3)))*)(
          reinterpret_cast<uintptr_t>(tile + v_at<D>(4 * g + rr, 16 * t + 4 * qq))));
      const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((short4v __attribute__((address_space(3)))*)(
          reinterpret_cast<uintptr_t>(tile + v_at<D>(16 + 4 * g + rr, 16 * t + 4 * qq))));
      const short8v a8 = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      o[t] = mfma16x16x32(__builtin_bit_cast(bf16x8, a8), pb, o[t]);
    }
    if ((bad[0] | bad[1]) != 0) {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        bool hit = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = 4 * g + (i & 3);
          // the lanes of block n of row r: l % 16 = r, l / 16 = 4 n / NB
          const bool nan = (bad[i >> 2] >> (r + 16 * (4 * n / NB))) & 1;
          hit = hit || (nan && k0 + 16 * (i >> 2) + (i & 3) < vis);
        }
        float add = hit ? NAN : 0.f;
        add += __shfl_xor(add, 16, 64);
        add += __shfl_xor(add, 32, 64);
#pragma unroll
        for (int t = n * DT / NB; t < (n + 1) * DT / NB; ++t) o[t] += add;
      }
    }

    const bool pair_end = cc.tile == cc.nb - 1;
    if (pair_end || u == u1 - 1) {
      flush(cc, pair_u0);
      if (pair_end) pair_u0 += cc.nb;
      if (u + 1 < u1) start(nc);
    }
    cc = nc;
    cur = nxt;
  }
}

// Merges the records of the pairs split between waves: a block per pair and
// column, its four waves every fourth record each, merged in wave order.
template <int D>
__global__ __launch_bounds__(256) void mx_decode_combine(const MxAttn p) {
  constexpr int N = D / 64;  // outputs per lane
  __shared__ float s_m[4], s_l[4], s_o[4][D];
  const int HS = p.Hkv * p.nset, pair = blockIdx.x, col = blockIdx.y;
  const int b = pair / HS, hs = pair - b * HS;
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (p.lens_inc && hs == 0 && col == 0 && threadIdx.x == 0) p.lens_inc[b] += p.inc;
  const int kvh = hs / p.nset, gc = (hs - kvh * p.nset) * kCols + col;
  const int tok = gc / p.groups, hd = gc - tok * p.groups;
  if (tok >= p.Sq) return;
  bf16* orow = p.o + b * p.ob + ((int64_t)kvh * p.groups + hd) * p.oh + tok * p.os;
  const int nb = p.hdr[b + 1] - p.hdr[b];
  if (nb == 0) {  // an empty sequence: zeros
    if (wv == 0)
#pragma unroll
      for (int e = 0; e < N; ++e) orow[N * lane + e] = f2bf(0.f);
    return;
  }
  const int64_t U = (int64_t)HS * p.hdr[p.B], first = (int64_t)HS * p.hdr[b] + (int64_t)hs * nb;
  const int w0 = wave_of(first, U), w1 = wave_of(first + nb - 1, U);
  if (w0 == w1) return;  // stored by its wave
  float m = -INFINITY, l = 0.f, o[N] = {};
  for (int w = w0 + wv; w <= w1; w += 4) {
    const float* rec = p.rec + ((int64_t)w + pair) * rec_floats(D);
    const float mr = rec[col], lr = rec[kCols + col];
    const float mn = fmaxf(m, mr), base = mn == -INFINITY ? 0.f : mn;
    const float a = exp2_(m - base), r = exp2_(mr - base);
    l = l * a + lr * r;
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = o[e] * a + rec[2 * kCols + col * D + N * lane + e] * r;
    m = mn;
  }
  if (lane == 0) {
    s_m[wv] = m;
    s_l[wv] = l;
  }
#pragma unroll
  for (int e = 0; e < N; ++e) s_o[wv][N * lane + e] = o[e];
  __syncthreads();
  if (wv != 0) return;
  m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  if (m == -INFINITY) m = 0.f;
  l = 0.f;
#pragma unroll
  for (int e = 0; e < N; ++e) o[e] = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float r = exp2_(s_m[i] - m);
    l += s_l[i] * r;
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] += s_o[i][N * lane + e] * r;
  }
  const float inv = l != 0.f ? 1.0f / l : 0.f;
#pragma unroll
  for (int e = 0; e < N; ++e) orow[N * lane + e] = f2bf(o[e] * inv);
}

int64_t header_bytes(int64_t B) { return (B + 1 + 63) / 64 * 256; }

int64_t sets_of(int64_t groups, int64_t Sq) { return q3_cdiv(groups * Sq, kCols); }

// The streaming kernel takes one token of any group, or a short chunk whose tokens and heads share the columns.
bool streams(int64_t groups, int64_t Sq) { return Sq == 1 || groups * Sq <= kCols; }

int64_t stream_ws_bytes(int64_t B, int64_t Hkv, int64_t groups, int64_t Sq, int64_t D) {
  return header_bytes(B) + (kWaves + B * Hkv * sets_of(groups, Sq)) * (int64_t)rec_floats((int)D) * 4;
}

int launch_stream(const MxAttn& p, int64_t D, hipStream_t st) {
  const dim3 grid(kBlocks), block(64 * kWavesPerBlock);
  const dim3 merge((unsigned)(p.B * p.Hkv * p.nset), (unsigned)std::min(kCols, p.groups * p.Sq));
  if (D == 128) {
    hipLaunchKernelGGL((mx_decode_kernel<128>), grid, block, 0, st, p);
    Q3_LAUNCH_CHECK();
    hipLaunchKernelGGL((mx_decode_combine<128>), merge, dim3(256), 0, st, p);
  } else {
    hipLaunchKernelGGL((mx_decode_kernel<64>), grid, block, 0, st, p);
    Q3_LAUNCH_CHECK();
    hipLaunchKernelGGL((mx_decode_combine<64>), merge, dim3(256), 0, st, p);
  }
  Q3_LAUNCH_CHECK();
  return Q3_OK;
}

// Arguments that both entry points take; strides = [qb, qh, qs, ob, oh, os] in
// elements, then [b, h] of k_codes, k_scales, v_codes, v_scales in bytes.
int check(const void* q, const void* kc, const void* ks, const void* vc, const void* vs, const int* lens,
          const void* o, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t D, int64_t cap,
          const int64_t* strides, int dtype) {
  Q3_REQUIRE(q && kc && ks && vc && vs && lens && o && strides, Q3_ERR_NULL);
  Q3_REQUIRE(B >= 0 && Hq >= 1 && Hkv >= 1 && Hq % Hkv == 0 && Sq >= 0 && D >= 1 && cap >= 0, Q3_ERR_SHAPE);
  Q3_REQUIRE(dtype == Q3_BF16, Q3_ERR_DTYPE);
  Q3_REQUIRE((D == 64 || D == 128) && B <= kMaxBatch && cap < (1ll << 31) - kUnit && Sq < (1ll << 31) &&
                 Hq < (1ll << 16) && B * Hkv * q3_cdiv(Hq / Hkv, kCols) < (1ll << 31),
             Q3_ERR_UNSUPPORTED);
  bool ok = q3_aligned(q, 16) && q3_aligned(kc, 16) && q3_aligned(vc, 16) && q3_aligned(o, 8);
  for (int i = 0; i < 6; ++i) ok = ok && strides[i] % 8 == 0;
  for (int i : {6, 7, 10, 11}) ok = ok && strides[i] % 16 == 0;
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

}  // namespace

extern "C" {

int64_t q3_decode_attention_mxfp4_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0) return 0;
  return stream_ws_bytes(B, Hkv, Hq / Hkv, 1, D);
}

int q3_decode_attention_mxfp4(const void* q, const void* k_codes, const void* k_scales, const void* v_codes,
                              const void* v_scales, int* kv_lens, int advance, void* o, int64_t B, int64_t Hq,
                              int64_t Hkv, int64_t D, int64_t cap, const int64_t* strides, float scale, int dtype,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check(q, k_codes, k_scales, v_codes, v_scales, kv_lens, o, B, Hq, Hkv, 1, D, cap, strides, dtype);
  if (rc != Q3_OK || B == 0) return rc;
  Q3_REQUIRE(workspace && workspace_bytes >= q3_decode_attention_mxfp4_workspace_bytes(B, Hq, Hkv, D),
             Q3_ERR_WORKSPACE);
  Q3_REQUIRE(q3_aligned(workspace, 16), Q3_ERR_ALIGN);
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
  if (streams(Hq / Hkv, Sq)) return stream_ws_bytes(B, Hkv, Hq / Hkv, Sq, D);
  return 2 * B * Hkv * max_len * D * 2;  // K and V in bf16
}

int q3_flash_attention_cache_mxfp4(const void* q, const void* k_codes, const void* k_scales, const void* v_codes,
                                   const void* v_scales, int* kv_lens, void* o, int64_t B, int64_t Hq, int64_t Hkv,
                                   int64_t Sq, int64_t D, int64_t max_len, const int64_t* strides, float scale,
                                   int advance, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc =
      check(q, k_codes, k_scales, v_codes, v_scales, kv_lens, o, B, Hq, Hkv, Sq, D, max_len, strides, dtype);
  if (rc != Q3_OK || B == 0 || Sq == 0) return rc;
  Q3_REQUIRE(Sq <= max_len, Q3_ERR_SHAPE);
  Q3_REQUIRE(workspace &&
                 workspace_bytes >= q3_flash_attention_cache_mxfp4_workspace_bytes(B, Hq, Hkv, Sq, D, max_len),
             Q3_ERR_WORKSPACE);
  Q3_REQUIRE(q3_aligned(workspace, 16), Q3_ERR_ALIGN);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (streams(Hq / Hkv, Sq)) {
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
  bf16* vx = kx + B * Hkv * max_len * D;
  int r = mx_expand(k_codes, k_scales, kx, B, Hkv, max_len * D, strides + 6, kv_lens, (int)Sq, D, Q3_BF16, st);
  if (r != Q3_OK) return r;
  const int64_t vst[4] = {strides[10], strides[11], strides[12], strides[13]};
  r = mx_expand(v_codes, v_scales, vx, B, Hkv, max_len * D, vst, kv_lens, (int)Sq, D, Q3_BF16, st);
  if (r != Q3_OK) return r;
  const int64_t rows[12] = {strides[0], strides[1], strides[2], Hkv * max_len * D, max_len * D, D,
                            Hkv * max_len * D, max_len * D, D, strides[3], strides[4], strides[5]};
  return q3_flash_attention_cache(q, kx, vx, kv_lens, o, B, Hq, Hkv, Sq, max_len, D, rows, scale, advance, dtype,
                                  stream);
}

}  // extern "C"
