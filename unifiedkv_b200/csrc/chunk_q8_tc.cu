// Attention of chunks of new tokens over 8-bit pages on the 5th-generation tensor
// cores (tcgen05.mma, TMEM accumulators), sm_100a, head_dim 64 and 128.
//
// The mathematics is page16_q8.cu's; the rows of a request and KV head (query token
// major, query head minor) are cut into tiles of 256 or 128.
//
// Design:
//  * Bound.  A chunk does 4 * head_dim FLOP per (row, visible token): with hundreds of
//    rows the tensor pipe and the exponentials bound it, not the pages' bytes.
//  * Codes become fp16 operands on the way into shared memory.  Eight converter warps
//    bring 16-code pieces in by cp.async (one tile ahead, each thread its own), turn them
//    into fp16 (cvt.rn.f16x2.e4m3x2 and one multiply per pair; e4m3 to bf16 takes five
//    instructions a pair and made the converters the bound) and store them in the
//    128-byte-swizzled layout of the UMMA descriptors, 128 tokens a tile, K and V each two
//    tiles deep.  A key takes its scale relative to the tile's largest, which joins the
//    softmax scale: one multiplier per tile.  A value takes its scale relative to a
//    reference that follows the largest seen (64 above it stays in range; O is rescaled in
//    the rare case that it moves).  Both are exact down to 2^-15 of the reference.  Where a
//    CTA meets a smaller scale (but for 0, that of rows of zeros) its rows are computed once
//    more, from the codes, in fp32 without tensor cores: a key or value 2^15 times the others
//    takes nothing from rows that do not see it, but time (2048 new of 32768 tokens 98 ms with
//    one such value per head, 1.35 ms without).
//  * q goes to fp16 with a power of two per row that brings the row into [2^14, 2^15):
//    exact down to 2^-29 of the row's largest element, off by 2^-40 of it below.
//  * Groups A and B of 8 softmax warps, 128 rows each, 2 threads per row.  The MMA warp
//    issues PV_A S_A' PV_B S_B' so that one group's softmax runs under the other's
//    MMAs.  With more than 128 rows A and B are two row tiles over the same K/V tiles;
//    with fewer (alternating) both hold the same rows and take every other K/V tile.
//  * Softmax: online in exp2, a reference maximum moved only when it lags by 2^4.  Weights
//    go to TMEM as fp16 in units of 2^-11 (off by 2^-11 of each, against 2^-8 for a bf16
//    output; nothing above 2^-35 of the row's largest vanishes); fp16 outputs take them as
//    a high and a low part.  (Exponentials on the FMA pipe, one in 4, 6 or 8: 1597, 1440,
//    1439 us for 2048 new of 32768 tokens against 1440 with none: the special function
//    unit is not what bounds the kernel.)
//  * The K/V tiles of row tiles are cut into shares where that fills the SMs better, a CTA
//    each: by the host for one request and for narrow tables, else by chunk_q8_plan_kernel
//    from the batch's lengths, which only the device knows.  Shares (and the two groups when
//    alternating) leave fp32 (o, lse) parts that chunk_q8_merge_kernel joins.
//  * Every wait is bounded (a poll count and 2 s); one that runs out ends in NaN rows.
//
// Measured (32 query heads, 8 KV heads, head_dim 128, bf16): 2048 new of 32768 tokens 1.35 to 1.37 ms
// from machine to machine, 780 TFLOP/s, 48 % of the measured cuBLAS burst; 8 x 512 over 900-16000 tokens
// 0.395 ms, 690.  Before row tiles were cut (1.45 ms) it took 1.35 with converters that store
// nothing and 1.17 with an eighth of the MMAs: the softmax chain (S, maximum, weights, P.V, next S) of two
// groups bounds it, and the converters' stores share the shared-memory port with the MMAs' operands.
#include <type_traits>

#include "chunk_q8.cuh"
#include "f32x2.cuh"
#include "tcgen05.cuh"

namespace bpkv {

namespace {

constexpr float kLn2 = 0.6931471805599453f;
constexpr int kBM = 128, kBN = 128;   // rows of a group, tokens of a K/V tile
constexpr int kRing = 2;              // K (and V) tiles in shared memory
constexpr int kGroupWarps = 8;        // softmax warps of a group: warps 0 .. 15
constexpr int kConvWarp = 16, kConvWarps = 8, kMmaWarp = 24, kScaleWarp = 25;
// Seven warpgroups are launched with 72 registers a thread (64,512 in all) and share them out anew:
// softmax 4 x 128 x 88, converters 2 x 128 x 56, MMA, scales (and two idle warps) 128 x 40 = 64,512.
constexpr int kThreads = 28 * 32;
constexpr int kRegsSoftmax = 88, kRegsConv = 56, kRegsMma = 40;
static_assert(128 * (4 * kRegsSoftmax + 2 * kRegsConv + kRegsMma) <= kThreads * 72, "register split");
constexpr int kMaxPages = 1024;       // block-table entries staged in shared memory
constexpr uint32_t kTmemCols = 512;
constexpr float kRescale = 4.f, kWOff = 11.f;  // weights <= 2^4, held times 2^11
constexpr int kVHead = 6;                      // values are held as code * 2^(byte - vref), byte <= vref + 6
constexpr int kExact = 15;                     // codes times 2^-15 are fp16 numbers still

// What a K/V tile's scales come to, worked out once by the scale warp: for the converters a factor per row
// (fp16 bits), for the softmax warps the rest.  A ring of 4; a slot is free again once P.V of its tile is done.
struct __align__(16) TileInfo {
  uint16_t kf[kBN], vf[kBN];
  float scale;       // softmax scale * log2(e) * 2^(largest key exponent)
  int vref;          // reference byte of the values
  uint32_t special;  // a token is missing (no page) or its value row is NaN
  uint32_t missing[4];
  uint32_t vnan[4];
};
constexpr int kInfo = 4;

template <int D, bool ALT>
struct Layout {
  static constexpr int kDB = D / 64;
  static constexpr int kQTiles = ALT ? 1 : 2;  // alternating groups share their rows
  // halves (the codes of one K or V tile) on their way to the converters: as many as fit.  Where few rows
  // read a long cache (alternating), memory's latency is what they have to cover.
  static constexpr int kDepth = D == 64 ? 6 : ALT ? 3 : 1;
  static constexpr int kQ = kDB * kBM * 128;   // bytes of a Q tile
  static constexpr int kKV = kDB * kBN * 128;  // bytes of a K or V tile
  static constexpr int kBars = kQTiles * kQ + 2 * kRing * kKV;
  static constexpr int kInfoOff = kBars + 256;
  static constexpr int kMx = kInfoOff + ((kInfo * static_cast<int>(sizeof(TileInfo)) + 15) / 16) * 16;
  static constexpr int kL = kMx + 4 * 2 * 2 * 2 * kBM;  // after the row maxima, [group][2 buffers][half][row]
  static constexpr int kQf = kL + 4 * 2 * 2 * kBM;      // after the row sums, [group][half][row]
  static constexpr int kStage = kQf + 4 * 2 * kBM;      // after q's row factors, [group][row]
  static constexpr int kPages = kStage + kDepth * kBN * D;
  static constexpr int kBytes = kPages + 4 * kMaxPages + 1024;  // + alignment
};

__device__ __forceinline__ uint32_t sw_off(int row, int chunk) {  // 16-byte chunk of a 128-byte swizzled row
  return static_cast<uint32_t>(row * 128 + ((chunk ^ (row & 7)) << 4));
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(N));
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// 2^e as an fp16 pair, e <= 15; 0 below the subnormals.
__device__ __forceinline__ uint32_t f16_pow2(int e) {
  const uint32_t x = e < -24 ? 0u : e < -14 ? 1u << (e + 24) : static_cast<uint32_t>(e + 15) << 10;
  return x | x << 16;
}

// The MMAs with their descriptors as two 32-bit words: only the low one (address, leading offset) varies, and
// an issuing thread with few registers keeps ahead of the tensor pipe.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 a, b;\n mov.b64 a, {%1, %3};\n mov.b64 b, {%2, %3};\n setp.ne.b32 p, %5, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n}\n" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 b;\n mov.b64 b, {%2, %3};\n setp.ne.b32 p, %5, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate));
}

// What a CTA needs to look at its scales once more (look: not all lie near one another), and to start over where they
// are too far apart for fp16 operands (wide).
struct Keep {
  int look, stuck, wide, vmin, vmax, item, tile0, n_tiles, share, shares;
};

// s += x, with what the additions so far rounded away in c.
__device__ __forceinline__ void add_exactly(float& s, float& c, float x) {
  const float y = x - c, t = s + y;
  c = (t - s) - y;
  s = t;
}

struct RowTile {
  int b, q0, n_q, n_rows, row0, kv_end;
};
template <bool ALT>
__device__ __forceinline__ RowTile row_tile(const ChunkQ8Params& p, int i) {
  RowTile r;
  const int rows = ALT ? kBM : 2 * kBM;
  r.b = i / p.tiles;
  r.row0 = (i % p.tiles) * rows;
  r.q0 = p.cu_q == nullptr ? r.b : __ldg(p.cu_q + r.b);
  r.n_q = p.cu_q == nullptr ? 1 : __ldg(p.cu_q + r.b + 1) - r.q0;
  r.n_rows = r.q0 < 0 ? 0 : min(r.n_q, p.total_q - r.q0) * p.n_rep;  // q has total_q rows, whatever cu_q says
  const int len = __ldg(p.lens + r.b);
  r.kv_end = 0;
  if (r.row0 < r.n_rows) {
    const int last = (min(r.row0 + rows, r.n_rows) - 1) / p.n_rep;
    r.kv_end = min(max(p.causal ? len - r.n_q + last + 1 : len, 0), p.max_blocks * kPage);
  }
  return r;
}

// The plan of a batch.  Candidates: the `whole` longest row tiles, none to two full waves of CTAs, stay whole; the
// tokens of each of the others are cut into s shares, or into shares of an s-th of the longest of them.  A candidate's
// time is the work over the SMs (as in page16_q8.cu, choose_shares), plus the idle end of the last wave, as long as the
// smallest piece, which starts last, but no less than the longest piece.
constexpr int kPlanThreads = 1024;
template <bool ALT>
__global__ void __launch_bounds__(kPlanThreads) chunk_q8_plan_kernel(const __grid_constant__ ChunkQ8Params p) {
  __shared__ int s_len[kMaxRanked], s_item[kMaxRanked], s_sorted[kMaxRanked], s_shares[kMaxRanked];
  __shared__ unsigned long long s_best[kPlanThreads / 32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n = p.B * p.tiles;
  if (tid < n) {
    const RowTile rt = row_tile<ALT>(p, tid);
    s_len[tid] = rt.row0 >= rt.n_rows ? -1 : (rt.kv_end + kBN - 1) / kBN;
  }
  __syncthreads();
  if (tid < n) {
    const int t = s_len[tid];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += (s_len[j] > t) || (s_len[j] == t && j < tid);
    s_item[rank] = tid;
    s_sorted[rank] = t;
  }
  __syncthreads();
  // candidate c: shares of an s-th (0) or s shares (1); full waves whole; s - 1
  const int m = p.max_shares;
  auto whole_of = [&](int c) { return min(n, c / m % 3 * p.sms / p.Hkv); };
  auto piece_of = [&](int c) {
    const int whole = whole_of(c), s = c % m + 1;
    return whole < n ? max(1, (s_sorted[whole] + s - 1) / s) : 1;
  };
  auto shares_of = [&](int j, int c, int whole, int piece) {
    const int t = s_sorted[j];
    return t < 0 ? 0 : j < whole ? 1 : c >= 3 * m ? c % m + 1 : max(1, (t + piece - 1) / piece);
  };
  unsigned long long best = ~0ull;
  for (int c = warp; c < 6 * m; c += kPlanThreads / 32) {
    const int whole = whole_of(c), piece = piece_of(c);
    if (c > 0 && (c % m == 0 || (c / m % 3 > 0 && (whole == 0 || whole >= n)))) continue;
    unsigned tiles = 0, count = 0, cut = 0;
    float least = INFINITY, longest = 0.f;
    for (int j = lane; j < n; j += 32) {
      const int k = shares_of(j, c, whole, piece);
      if (k == 0) break;
      const float size = static_cast<float>(s_sorted[j]) / k + (k > 1 ? 11.f : 9.f);
      tiles += s_sorted[j];
      count += k;
      if (k > 1) cut += k;
      least = fminf(least, size);
      longest = fmaxf(longest, size);
    }
    tiles = __reduce_add_sync(0xffffffffu, tiles);
    count = __reduce_add_sync(0xffffffffu, count);
    cut = __reduce_add_sync(0xffffffffu, cut);
    least = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(least)));  // not negative
    longest = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(longest)));
    if (c > 0 && (count == 0 || count > static_cast<unsigned>(p.n_pieces))) continue;  // 0, nothing cut, always fits
    const float per_sm = static_cast<float>(p.Hkv) / p.sms, idle = ceilf(count * per_sm) - count * per_sm;
    const float cost = fmaxf((tiles + 9.f * count + 2.f * cut) * per_sm + (idle > 0.f ? idle * least : 0.f), longest);
    best = min(best, static_cast<unsigned long long>(__float_as_uint(cost)) << 32 | static_cast<unsigned>(c));
  }
  if (lane == 0) s_best[warp] = best;
  __syncthreads();
  for (int i = 0; i < kPlanThreads / 32; ++i) best = min(best, s_best[i]);
  const int c = static_cast<int>(best & 0xffffffffu);
  const int shares = tid < n ? shares_of(tid, c, whole_of(c), piece_of(c)) : 0;
  if (tid < n) s_shares[tid] = shares;
  __syncthreads();
  // pieces in the order of their size
  int first = 0, total = 0;
  const int64_t t = tid < n ? s_sorted[tid] : 0;
  for (int j = 0; j < n; ++j) {
    const int k = s_shares[j];
    const int64_t d = s_sorted[j] * static_cast<int64_t>(shares) - t * k;
    if (d > 0 || (d == 0 && j < tid)) first += k;
    total += k;
  }
  if (tid < n) {
    const int item = s_item[tid];
    p.n_shares[item] = shares;
    for (int i = 0; i < shares; ++i) p.pieces[first + i] = make_int2(item, i | shares << 16);
  }
  for (int i = total + tid; i < p.n_pieces; i += kPlanThreads) p.pieces[i] = make_int2(-1, 0);
}

// Whether a tile of keys, or all the values, have scales too far apart; but for rows of zeros, NaN, and rows that are not
// there.  16 lanes a tile: keys of its 8 pages, then values.
template <bool ALT>
__device__ __forceinline__ void look_at_scales(const ChunkQ8Params& p, volatile Keep* keep) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hkv = static_cast<int>(blockIdx.x % p.Hkv);
  const RowTile rt = row_tile<ALT>(p, keep->item);
  const int32_t* bt_row = p.bt + static_cast<int64_t>(rt.b) * p.bt_sb;
  const int tile0 = keep->tile0, end = tile0 + keep->n_tiles;
  int vmax = 0, vmin = 255;
  for (int t0 = tile0 + 2 * warp; t0 < end; t0 += 4 * kGroupWarps) {
    const int t = t0 + lane / 16, first = t * kBN + lane % 8 * kPage, live = min(rt.kv_end, end * kBN) - first;
    const int page = live > 0 ? q8::page_of(bt_row, first / kPage, p.max_blocks, p.num_pages) : -1;
    int most = 0, least = 255;
    if (page >= 0) {
      const uint8_t* s = (lane & 8 ? p.vs : p.ks) + page * p.scale_stride + hkv * kPage;
      for (int i = 0; i < min(live, kPage); ++i) {
        const int b = __ldg(s + i);
        if (b != q8::kNanByte) most = max(most, b);
        if (b != 0) least = min(least, b);
      }
    }
    if (lane & 8) {
      vmax = max(vmax, most), vmin = min(vmin, least);
      most = 0;
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
      least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
    }
    if (least < most - kExact) keep->wide = 1;
  }
  vmax = __reduce_max_sync(0xffffffffu, vmax), vmin = __reduce_min_sync(0xffffffffu, vmin);
  if (lane == 0) {
    atomicMax(const_cast<int*>(&keep->vmax), vmax);
    atomicMin(const_cast<int*>(&keep->vmin), vmin);
  }
}

// The work of a CTA that met scales too far apart: two rows a warp, page by page, in fp32 from the codes.  For the dot
// products and the values a lane has D / 32 columns; the 2 x 16 sums of a page are exchanged so that lane 16 i + j has row
// i's of token j.  (What it needs it works out anew: the tensor-core path has no registers to keep it in.)
template <typename T, int D, bool ALT>
__device__ __forceinline__ void exact_rows(const ChunkQ8Params& p, const volatile Keep* keep) {
  constexpr int C = D / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, mine = lane / 16;
  const int tile0 = keep->tile0, n_tiles = keep->n_tiles, share = keep->share, hkv = static_cast<int>(blockIdx.x % p.Hkv);
  const bool whole = !ALT && keep->shares == 1;
  const RowTile rt = row_tile<ALT>(p, keep->item);
  const int len = __ldg(p.lens + rt.b);
  const int32_t* bt_row = p.bt + static_cast<int64_t>(rt.b) * p.bt_sb;
  const int64_t all_rows = static_cast<int64_t>(p.total_q) * p.Hq;
  auto codes = [](const uint8_t* src, float* y) {  // C of them
    uint32_t w;
    if constexpr (C == 4) w = __ldg(reinterpret_cast<const uint32_t*>(src));
    else w = __ldg(reinterpret_cast<const uint16_t*>(src));
    uint32_t lo, hi;
    q8::e4m3x4_to_f16x4(w, lo, hi);
    const float2 a = __half22float2(*reinterpret_cast<__half2*>(&lo)), b = __half22float2(*reinterpret_cast<__half2*>(&hi));
    y[0] = a.x, y[1] = a.y, y[2] = b.x, y[3] = b.y;
  };
  for (int first = 2 * warp; first < Layout<D, ALT>::kQTiles * kBM && rt.row0 + first < rt.n_rows; first += 4 * kGroupWarps) {
    float x[2][C], acc[2][C], acc_c[2][C], f = 0.f;
    int last[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int rr = min(rt.row0 + first + i, rt.n_rows - 1);
      const T* src = static_cast<const T*>(p.q) + static_cast<int64_t>(rt.q0 + rr / p.n_rep) * p.q_st +
                     static_cast<int64_t>(hkv * p.n_rep + rr % p.n_rep) * p.q_sh + lane * C;
      uint32_t amax = 0;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        x[i][c] = Elem<T>::to_f(src[c]);
        amax = max(amax, __float_as_uint(x[i][c]) & 0x7fffffffu);
        acc[i][c] = acc_c[i][c] = 0.f;
      }
      amax = __reduce_max_sync(0xffffffffu, amax);
      int qe = static_cast<int>(amax >> 23) - 127 - 14;
      qe = (amax == 0 || amax >= 0x7f800000u) ? 0 : max(qe, -100);
#pragma unroll
      for (int c = 0; c < C; ++c) x[i][c] *= q8::q_factor(amax, qe);
      if (mine == i) f = p.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 + qe) << 23);
      last[i] = min(min(p.causal ? len - rt.n_q + rr / p.n_rep : len - 1, rt.kv_end - 1), (tile0 + n_tiles) * kBN - 1);
    }
    float m = -INFINITY, sum = 0.f, sum_c = 0.f;  // of row `mine`; the sum over this lane's tokens
    for (int t0 = tile0 * kBN; t0 <= max(last[0], last[1]); t0 += kPage) {
      const int page = q8::page_of(bt_row, t0 / kPage, p.max_blocks, p.num_pages);
      if (page < 0) continue;
      const int64_t at = page * p.page_stride + static_cast<int64_t>(hkv) * D + lane * C, step = static_cast<int64_t>(p.Hkv) * D;
      const int64_t sat = page * p.scale_stride + hkv * kPage + lane % 16;
      float s[32];
#pragma unroll
      for (int j = 0; j < kPage; ++j) {
        float kx[4];
        codes(p.kc + at + j * step, kx);
        s[j] = s[16 + j] = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) s[j] += x[0][c] * kx[c], s[16 + j] += x[1][c] * kx[c];
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
        for (int j = 0; j < o; ++j) {
          const float give = lane & o ? s[j] : s[j + o], stay = lane & o ? s[j + o] : s[j];
          s[j] = stay + __shfl_xor_sync(0xffffffffu, give, o);
        }
      }
      const bool seen = t0 + lane % 16 <= (mine ? last[1] : last[0]);
      const float score = seen ? s[0] * fminf(f * q8::scale_of(__ldg(p.ks + sat)), 3.4028235e38f) : -INFINITY;
      float mn = score;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
      mn = fmaxf(m, mn);
      const float mu = mn == -INFINITY ? 0.f : mn, a = fast_exp2(m - mu), w = fast_exp2(score - mu);
      m = mn;
      sum *= a, sum_c *= a;
      add_exactly(sum, sum_c, w);
      // values times 2^-16, so that their sums stay in range
      const float wv = w * (q8::scale_of(__ldg(p.vs + sat)) * 0x1p-16f);
      float part[2][C] = {};
#pragma unroll
      for (int j = 0; j < kPage; ++j) {
        float vx[4];
        codes(p.vc + at + j * step, vx);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float wi = __shfl_sync(0xffffffffu, wv, 16 * i + j);
#pragma unroll
          for (int c = 0; c < C; ++c) part[i][c] += t0 + j <= last[i] ? wi * vx[c] : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float ai = __shfl_sync(0xffffffffu, a, 16 * i);
#pragma unroll
        for (int c = 0; c < C; ++c) {
          acc[i][c] *= ai, acc_c[i][c] *= ai;
          add_exactly(acc[i][c], acc_c[i][c], part[i][c]);
        }
      }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float l = __shfl_sync(0xffffffffu, sum, 16 * i), top = __shfl_sync(0xffffffffu, m, 16 * i);
      const int rr = rt.row0 + first + i;
      if (rr >= rt.n_rows) continue;
      const bool none = l == 0.f;
      const float inv = none ? 0.f : 1.f / l, lse = none ? -INFINITY : (top + log2f(l)) * kLn2;
      const int64_t o = static_cast<int64_t>(rt.q0 + rr / p.n_rep) * p.Hq + hkv * p.n_rep + rr % p.n_rep;
      if (whole) {
#pragma unroll
        for (int c = 0; c < C; c += 2)
          *reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + o * D + lane * C + c) =
              pack2<T>(none ? p.empty : acc[i][c] * inv * 65536.f, none ? p.empty : acc[i][c + 1] * inv * 65536.f);
        if (lane == 0 && p.lse_out != nullptr) p.lse_out[o] = lse;
      } else {  // alternating groups leave two parts: this is the first, and the second is empty
#pragma unroll
        for (int part = 0; part < (ALT ? 2 : 1); ++part) {
          const int64_t po = (ALT ? 2 * share + part : share) * all_rows + o;
#pragma unroll
          for (int c = 0; c < C; ++c) p.part_o[po * D + lane * C + c] = part == 0 ? acc[i][c] * inv * 65536.f : 0.f;
          if (lane == 0) p.part_lse[po] = part == 0 ? lse : -INFINITY;
        }
      }
    }
  }
}

template <typename T, int D, bool ALT>
__global__ void __launch_bounds__(kThreads, 1) chunk_q8_kernel(const __grid_constant__ ChunkQ8Params p) {
  using L = Layout<D, ALT>;
  static_assert(L::kBytes <= 232448, "shared memory");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t qs = smem_u32(smem), ks = qs + L::kQTiles * L::kQ, vs = ks + kRing * L::kKV;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
  constexpr int kBarCount = 4 * kRing + 7 + 2 * kInfo;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kBarCount);
  volatile Keep* keep = reinterpret_cast<Keep*>(tmem_slot + 2);
  static_assert((kBarCount + 1) * 8 + sizeof(Keep) <= 248, "barrier area");
  TileInfo* s_info = reinterpret_cast<TileInfo*>(smem + L::kInfoOff);
  float* s_mx = reinterpret_cast<float*>(smem + L::kMx);
  float* s_l = reinterpret_cast<float*>(smem + L::kL);
  float* s_qf = reinterpret_cast<float*>(smem + L::kQf);
  int* s_pages = reinterpret_cast<int*>(smem + L::kPages);

  constexpr bool kTwoParts = std::is_same<T, __half>::value;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // ---- work item: (row tile, share of its tokens, KV head) ----
  const int hkv = static_cast<int>(blockIdx.x % p.Hkv);
  int item = static_cast<int>(blockIdx.x / p.Hkv), share = 0, shares = 1;
  if (p.pieces != nullptr) {
    pdl_wait();
    const int2 piece = __ldcg(p.pieces + item);
    item = piece.x;
    share = piece.y & 0xffff;
    shares = piece.y >> 16;
    if (item < 0) return;  // uniform across the CTA
  } else if (item >= p.whole) {
    const int i = item - p.whole;
    item = p.whole + i / p.shares, share = i % p.shares, shares = p.shares;
  }
  if (p.B == 1) {
    item = p.tiles - 1 - item;
  } else if (p.ranked) {
    __shared__ int s_item;
    const int n_items = p.B * p.tiles;
    for (int i = tid; i < n_items; i += kThreads) s_pages[i] = row_tile<ALT>(p, i).kv_end;
    __syncthreads();
    for (int i = tid; i < n_items; i += kThreads) {
      const int wi = s_pages[i];
      int rank = 0;
      for (int j = 0; j < n_items; ++j) rank += (s_pages[j] > wi) || (s_pages[j] == wi && j < i);
      if (rank == item) s_item = i;
    }
    __syncthreads();
    item = s_item;
  }
  const RowTile rt = row_tile<ALT>(p, item);
  if (rt.row0 >= rt.n_rows) return;  // uniform across the CTA, before any barrier or TMEM use
  const int all_tiles = (rt.kv_end + kBN - 1) / kBN;
  const int tile0 = static_cast<int>(static_cast<int64_t>(all_tiles) * share / shares);
  const int n_tiles = static_cast<int>(static_cast<int64_t>(all_tiles) * (share + 1) / shares) - tile0;
  const int32_t* bt_row = p.bt + static_cast<int64_t>(rt.b) * p.bt_sb;

  auto k_full = [&](int t) { return smem_u32(&bars[t % kRing]); };
  auto v_full = [&](int t) { return smem_u32(&bars[kRing + t % kRing]); };
  auto k_free = [&](int t) { return smem_u32(&bars[2 * kRing + t % kRing]); };
  auto v_free = [&](int t) { return smem_u32(&bars[3 * kRing + t % kRing]); };
  auto s_full = [&](int g) { return smem_u32(&bars[4 * kRing + g]); };
  auto p_full = [&](int g) { return smem_u32(&bars[4 * kRing + 2 + g]); };
  auto o_done = [&](int g) { return smem_u32(&bars[4 * kRing + 4 + g]); };
  const uint32_t q_full = smem_u32(&bars[kBarCount - 1]);
  auto info_full = [&](int t) { return smem_u32(&bars[4 * kRing + 6 + t % kInfo]); };
  auto info_free = [&](int t) { return smem_u32(&bars[4 * kRing + 6 + kInfo + t % kInfo]); };

  if (warp == 0) {
    tc::tmem_alloc(smem_u32(tmem_slot), kTmemCols);
    tc::tmem_relinquish();
  }
  if (tid == 0) {
    for (int i = 0; i < kRing; ++i) {
      tc::mbar_init(k_full(i), 32u * kConvWarps);
      tc::mbar_init(v_full(i), 32u * kConvWarps);
      tc::mbar_init(k_free(i), 1u);
      tc::mbar_init(v_free(i), 1u);
    }
    for (int i = 0; i < kInfo; ++i) {
      tc::mbar_init(info_full(i), 32u);
      tc::mbar_init(info_free(i), 1u);
    }
    keep->look = keep->stuck = keep->wide = keep->vmax = 0;
    keep->vmin = 255;
    keep->item = item;
    keep->tile0 = tile0;
    keep->n_tiles = n_tiles;
    keep->share = share;
    keep->shares = shares;
    tc::mbar_init(q_full, 32u * 2 * kGroupWarps);
    for (int g = 0; g < 2; ++g) {
      tc::mbar_init(s_full(g), 1u);
      tc::mbar_init(p_full(g), 32u * kGroupWarps);
      tc::mbar_init(o_done(g), 1u);
    }
    tc::fence_mbar_init();
  }
  const int page0 = tile0 * (kBN / kPage);
  tc::tc_fence_before();
  __syncthreads();  // barriers initialised, TMEM address published; from here on every role goes its own way
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto t_s = [&](int g) { return tmem + static_cast<uint32_t>(g * 256); };
  auto t_o = [&](int g) { return tmem + static_cast<uint32_t>(g * 256 + 128); };
  const bool staged = n_tiles * (kBN / kPage) <= kMaxPages;
  auto page_at = [&](int idx) {  // idx from page0
    return staged || idx < kMaxPages ? s_pages[idx] : q8::page_of(bt_row, page0 + idx, p.max_blocks, p.num_pages);
  };
  // group g's tile number k is K/V tile tile_at(g, k)
  auto tile_at = [&](int g, int k) { return ALT ? 2 * k + g : k; };

  if (warp >= kConvWarp && warp < kMmaWarp) {
    // =================== converters ===================
    regs_dec<kRegsConv>();
    const int ct = tid - kConvWarp * 32;
    {
      const int np = min(n_tiles * (kBN / kPage), kMaxPages);
      for (int i = ct; i < np; i += 32 * kConvWarps) s_pages[i] = q8::page_of(bt_row, page0 + i, p.max_blocks, p.num_pages);
      asm volatile("bar.sync 1, %0;\n" ::"n"(32 * (kConvWarps + 1)) : "memory");  // with the scale warp
    }
    // Thread ct handles 16-code piece ct % 4 of each 64-code block of rows ct / 4 + RS i: a quarter warp then
    // stores whole swizzled rows of one block, without bank conflicts.
    constexpr int RS = 8 * kConvWarps, N = kBN / RS, DB = L::kDB;
    constexpr uint32_t kSlot = 32 * kConvWarps * 16;  // staging bytes of one piece of every thread
    const int ch = ct & 3, r0 = ct >> 2;
    const int64_t in_page = static_cast<int64_t>(r0 & 15) * p.Hkv * D + static_cast<int64_t>(hkv) * D + ch * 16;
    const uint8_t *kp = p.kc + in_page, *vp = p.vc + in_page;
    // Half 2t is K of tile t, half 2t + 1 its V; half h lies in slot h % kDepth of the staging area, where
    // each thread keeps its own pieces.  Row i of half h + kDepth is fetched when that of half h is stored.
    constexpr int kDepth = L::kDepth;
    const uint32_t stage = smem_u32(smem + L::kStage) + ct * 16;
    const int n_halves = 2 * n_tiles;
    auto slot_of = [&](int h, int i) { return stage + ((h % kDepth * N + i) * DB) * kSlot; };
    auto fetch = [&](int h, int i) {
      if (h < n_halves) {
        const int t = h >> 1;
        const int page = page_at(t * (kBN / kPage) + RS / 16 * i + (r0 >> 4));
        const bool ok = r0 + RS * i < rt.kv_end - (tile0 + t) * kBN && page >= 0;
        const uint8_t* src = (h & 1 ? vp : kp) + (ok ? page * p.page_stride : 0);
#pragma unroll
        for (int db = 0; db < DB; ++db) cp_async16(slot_of(h, i) + db * kSlot, src + db * 64, ok);
      }
      cp_async_commit();
    };
    // 16 values of row r0 + RS i, piece ch of block db: two 16-byte chunks of the swizzled tile
    auto store = [&](uint32_t tile, int i, int db, const uint32_t* x) {
      const uint32_t b = tile + db * (kBN * 128) + i * (RS * 128);
      sts128(b + sw_off(r0, 2 * ch), x[0], x[1], x[2], x[3]);
      sts128(b + sw_off(r0, 2 * ch + 1), x[4], x[5], x[6], x[7]);
    };
    // this thread's pieces of half h and the factors of their rows, all asked for before any is used
    auto take = [&](int h, const uint16_t* factors, uint4* c, uint32_t* f) {
      cp_async_wait<(kDepth - 1) * N>();  // half h has come
#pragma unroll
      for (int i = 0; i < N * DB; ++i) c[i] = lds128(slot_of(h, i / DB) + (i % DB) * kSlot);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t x = factors[r0 + RS * i];
        f[i] = x | x << 16;
      }
    };
    for (int h = 0; h < kDepth; ++h) {
#pragma unroll
      for (int i = 0; i < N; ++i) fetch(h, i);
    }
    // Are there scales below what the operands hold exactly?  Mostly all keys' bytes lie in 16 around that of a token in
    // the middle, and all values' too: then there are none.  (Here, while the first codes are on their way, the look
    // costs nothing that shows; 8 x 512 new tokens take 389 us, 397 to 408 with it in the softmax warps, 398 to 402 in a
    // warp of its own that follows the tiles.)
    {
      const int tokens = min(rt.kv_end - tile0 * kBN, n_tiles * kBN), n_pages = (tokens + kPage - 1) / kPage;
      const int mid = n_pages > 0 ? page_at(n_pages / 2) : -1;
      const uint8_t *ksp = p.ks + hkv * kPage, *vsp = p.vs + hkv * kPage;
      const int kref = mid < 0 ? 0 : __ldg(ksp + mid * p.scale_stride), vref = mid < 0 ? 0 : __ldg(vsp + mid * p.scale_stride);
      constexpr uint32_t kAll = 0x01010101u;
      uint32_t far = min(kref, vref) < 8 || max(kref, vref) > 246 ? ~0u : 0u;
      auto bytes_far = [&](const uint4& x, int ref, int live) {  // a byte + 8 - ref: 0 to 15, or an upper bit is set
        uint32_t w[4] = {x.x, x.y, x.z, x.w};
        if (live < kPage) {  // rows behind the last count as the one in the middle
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int n = min(max(live - 4 * v, 0), 4);
            const uint32_t there = n == 4 ? ~0u : (1u << (8 * n)) - 1;
            w[v] = (w[v] & there) | (ref * kAll & ~there);
          }
        }
        const uint32_t add = (8 - ref) * kAll;
        far |= (w[0] + add) | (w[1] + add) | (w[2] + add) | (w[3] + add);
      };
#pragma unroll 2
      for (int i = ct; i < n_pages; i += 32 * kConvWarps) {
        const int page = page_at(i);
        if (page >= 0) {
          const uint4 kw = __ldg(reinterpret_cast<const uint4*>(ksp + page * p.scale_stride));
          const uint4 vw = __ldg(reinterpret_cast<const uint4*>(vsp + page * p.scale_stride));
          bytes_far(kw, kref, tokens - i * kPage);
          bytes_far(vw, vref, tokens - i * kPage);
        }
      }
      if ((far & 0xf0 * kAll) != 0) keep->look = 1;
    }
    bool ok = true;
    for (int t = 0; ok && t < n_tiles; ++t) {
      const TileInfo& info = s_info[t % kInfo];
      ok = tc::mbar_wait(info_full(t), (t / kInfo) & 1);
      // ---- K ----
      if (ok && t >= kRing) ok = tc::mbar_wait(k_free(t), (t / kRing - 1) & 1);
      if (!__all_sync(0xffffffffu, ok)) break;
      {
        const uint32_t dst = ks + (t % kRing) * L::kKV;
        uint4 c[N * DB];
        uint32_t f[N];
        take(2 * t, info.kf, c, f);
#pragma unroll
        for (int i = 0; i < N * DB; ++i) {
          const uint32_t w[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
          uint32_t x[8];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            q8::e4m3x4_to_f16x4(w[u], x[2 * u], x[2 * u + 1]);  // NaN codes stay NaN
            x[2 * u] = hmul2(x[2 * u], f[i / DB]);
            x[2 * u + 1] = hmul2(x[2 * u + 1], f[i / DB]);
          }
          store(dst, i / DB, i % DB, x);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) fetch(2 * t + kDepth, i);
      }
      tc::fence_proxy_async_smem();
      asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(k_full(t)) : "memory");
      // ---- V ----
      if (t >= kRing) ok = tc::mbar_wait(v_free(t), (t / kRing - 1) & 1);
      if (!__all_sync(0xffffffffu, ok)) break;
      {
        const uint32_t dst = vs + (t % kRing) * L::kKV;
        uint4 c[N * DB];
        uint32_t f[N];
        take(2 * t + 1, info.vf, c, f);
#pragma unroll
        for (int i = 0; i < N * DB; ++i) {
          const uint32_t keep = f[i / DB] == 0x7fff7fffu ? 0u : 0xffffffffu;  // a NaN row: its codes are taken out
          const uint32_t w[4] = {c[i].x & keep, c[i].y & keep, c[i].z & keep, c[i].w & keep};
          uint32_t x[8];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            q8::e4m3x4_to_f16x4(w[u], x[2 * u], x[2 * u + 1]);
            x[2 * u] = hmul2(x[2 * u], f[i / DB] & keep);
            x[2 * u + 1] = hmul2(x[2 * u + 1], f[i / DB] & keep);
          }
          store(dst, i / DB, i % DB, x);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) fetch(2 * t + 1 + kDepth, i);
      }
      tc::fence_proxy_async_smem();
      asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(v_full(t)) : "memory");
    }
    cp_async_wait<0>();
    asm volatile("bar.sync 10, %0;\n" ::"n"(32 * (2 * kGroupWarps + kConvWarps)) : "memory");  // with the softmax warps
  } else if (warp >= kMmaWarp) {
    // =================== MMA issue, scales (the first two warps of the group) ===================
    regs_dec<kRegsMma>();
    const uint32_t id_s = tc::idesc_f16(false, false, false, kBM, kBN);
    const uint32_t id_o = tc::idesc_f16(false, false, true, kBM, D);
    const uint64_t dv = tc::smem_desc_sw128(vs, kBN * 128, 1024);  // the high words are all alike
    const uint32_t hi = static_cast<uint32_t>(dv >> 32), v_lo = static_cast<uint32_t>(dv);
    const uint32_t q_lo = static_cast<uint32_t>(tc::smem_desc_sw128(qs, 16, 1024));
    constexpr uint32_t kToK = (L::kQTiles * L::kQ) >> 4;  // from Q's descriptor to K's
    auto issue_s = [&](int g, int t) {
      tc::tc_fence_after();
      const uint32_t qb = q_lo + (ALT ? 0u : static_cast<uint32_t>(g * (L::kQ >> 4)));
      const uint32_t kb = q_lo + kToK + static_cast<uint32_t>((t % kRing) * (L::kKV >> 4));
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint32_t off = static_cast<uint32_t>(((kk >> 2) * (kBM * 128) + (kk & 3) * 32) >> 4);
        mma_ss(t_s(g), qb + off, kb + off, hi, id_s, kk > 0 ? 1u : 0u);
      }
      tc::mma_commit(s_full(g));
      if (ALT || g == 1) tc::mma_commit(k_free(t));
    };
    auto issue_o = [&](int g, int k, int t) {
      tc::tc_fence_after();
      const uint32_t vb = v_lo + static_cast<uint32_t>((t % kRing) * (L::kKV >> 4));
#pragma unroll
      for (int part = 0; part < (kTwoParts ? 2 : 1); ++part) {
#pragma unroll
        for (int kk = 0; kk < kBN / 16; ++kk) {
          const uint32_t pa = t_s(g) + (kk >> 1) * 32 + part * 16 + (kk & 1) * 8;
          mma_ts(t_o(g), pa, vb + static_cast<uint32_t>((kk * 16 * 128) >> 4), hi, id_o, (k > 0 || part > 0 || kk > 0) ? 1u : 0u);
        }
      }
      tc::mma_commit(o_done(g));
      if (ALT || g == 1) {
        tc::mma_commit(v_free(t));
        tc::mma_commit(info_free(t));
      }
    };
    if (warp == kScaleWarp) {
      asm volatile("bar.sync 1, %0;\n" ::"n"(32 * (kConvWarps + 1)) : "memory");  // s_pages is there
      auto fetch_scales = [&](const uint8_t* scales, int t) -> uint32_t {  // bytes of tokens 4 lane .. 4 lane + 3
        const int page = lane * 4 < rt.kv_end - (tile0 + t) * kBN ? page_at(t * (kBN / kPage) + lane / 4) : -1;
        return page < 0 ? 0u : __ldg(reinterpret_cast<const uint32_t*>(scales + page * p.scale_stride + hkv * kPage) + lane % 4);
      };
      int vref = -1;
      uint32_t ksc = 0, vsc = 0, ksc_next = 0, vsc_next = 0;  // of tiles t, t + 1
      if (n_tiles > 0) ksc = fetch_scales(p.ks, 0), vsc = fetch_scales(p.vs, 0);
      if (n_tiles > 1) ksc_next = fetch_scales(p.ks, 1), vsc_next = fetch_scales(p.vs, 1);
      for (int t = 0; t < n_tiles; ++t) {
        if (t >= kInfo && !__all_sync(0xffffffffu, tc::mbar_wait(info_free(t), (t / kInfo - 1) & 1))) break;
        const int left = rt.kv_end - (tile0 + t) * kBN;
        const bool there = lane * 4 < left && page_at(t * (kBN / kPage) + lane / 4) >= 0;
        int emax = 0, vmax = 0;  // over live and finite rows
        uint32_t miss = 0, vnan = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int kb = ksc >> (8 * i) & 0xff, vb = vsc >> (8 * i) & 0xff;
          const bool live = there && lane * 4 + i < left;
          if (live && kb != q8::kNanByte) emax = max(emax, kb);
          if (live && vb != q8::kNanByte) vmax = max(vmax, vb);
          if (lane * 4 + i < left && !there) miss |= 1u << i;
          if (live && vb == q8::kNanByte) vnan |= 1u << i;
        }
        emax = __reduce_max_sync(0xffffffffu, emax);
        vmax = __reduce_max_sync(0xffffffffu, vmax);
        // the reference moves when the largest scale leaves fp16's range above it
        if (vref < 0 || vmax > vref + kVHead) vref = max(vmax - kVHead, 0);
        const bool special = __any_sync(0xffffffffu, (miss | vnan) != 0);
        TileInfo& info = s_info[t % kInfo];
        uint32_t kf[2] = {0, 0}, vf[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int kb = ksc >> (8 * i) & 0xff, vb = vsc >> (8 * i) & 0xff;
          kf[i >> 1] |= (f16_pow2(min(kb - emax, 0)) & 0xffffu) << (16 * (i & 1));
          vf[i >> 1] |= (vb == q8::kNanByte ? 0x7fffu : f16_pow2(min(vb - vref, kVHead)) & 0xffffu) << (16 * (i & 1));
        }
        *reinterpret_cast<uint2*>(info.kf + 4 * lane) = make_uint2(kf[0], kf[1]);
        *reinterpret_cast<uint2*>(info.vf + 4 * lane) = make_uint2(vf[0], vf[1]);
        if (lane == 0) {
          info.scale = p.scale_log2 * q8::scale_of(emax);
          info.vref = vref;
          info.special = special;
        }
        if (special) {  // bits of tokens 4 lane .. + 3 into words of 32
          miss <<= (lane & 7) * 4, vnan <<= (lane & 7) * 4;
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) {
            miss |= __shfl_xor_sync(0xffffffffu, miss, o);
            vnan |= __shfl_xor_sync(0xffffffffu, vnan, o);
          }
          if ((lane & 7) == 0) info.missing[lane >> 3] = miss, info.vnan[lane >> 3] = vnan;
        }
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(info_full(t)) : "memory");
        ksc = ksc_next, vsc = vsc_next;
        if (t + 2 < n_tiles) ksc_next = fetch_scales(p.ks, t + 2), vsc_next = fetch_scales(p.vs, t + 2);
      }
    }
    bool ok = warp == kMmaWarp && tc::mbar_wait(q_full, 0);
    for (int g = 0; ok && g < 2; ++g) {
      const int t = tile_at(g, 0);
      if (t >= n_tiles) break;
      ok = tc::mbar_wait(k_full(t), (t / kRing) & 1);
      if (ok && lane == 0) issue_s(g, t);
      __syncwarp();
    }
    for (int k = 0; ok && tile_at(0, k) < n_tiles; ++k) {
      for (int g = 0; ok && g < 2; ++g) {
        const int t = tile_at(g, k), tn = tile_at(g, k + 1);
        if (t >= n_tiles) break;
        ok = tc::mbar_wait(p_full(g), k & 1) && tc::mbar_wait(v_full(t), (t / kRing) & 1);
        if (!ok) break;
        if (lane == 0) issue_o(g, k, t);
        __syncwarp();
        if (tn < n_tiles) {  // S_g overwrites P_g: once PV_g has read it
          ok = tc::mbar_wait(k_full(tn), (tn / kRing) & 1) && tc::mbar_wait(o_done(g), k & 1);
          if (!ok) break;
          if (lane == 0) issue_s(g, tn);
          __syncwarp();
        }
      }
    }
    if (warp == kMmaWarp && !ok) keep->stuck = 1;
  } else {
    // =================== softmax ===================
    regs_inc<kRegsSoftmax>();
    const int g = warp / kGroupWarps;
    const int half = (warp % kGroupWarps) / 4, rq = warp % 4;
    const int row = rq * 32 + lane;  // of the group, and TMEM lane
    const int r = rt.row0 + (ALT ? 0 : g * kBM) + row;
    const bool valid = r < rt.n_rows;
    const int tok = valid ? r / p.n_rep : 0;
    const int len = __ldg(p.lens + rt.b);
    // last visible token, from the split's first
    const int lim = (valid ? min(p.causal ? len - rt.n_q + tok : len - 1, rt.kv_end - 1) : rt.kv_end - 1) - tile0 * kBN;
    const uint32_t lane_base = static_cast<uint32_t>(rq * 32) << 16;
    constexpr int kSC = kBN / 2, kOC = D / 2;
    const int sc0 = half * kSC, oc0 = half * kOC;
    const uint32_t ts = t_s(g) + lane_base + sc0, to = t_o(g) + lane_base + oc0;
    const uint32_t bar_id = 2 + g * 4 + rq;  // the two warps that share these rows
    float* mxg = s_mx + g * 4 * kBM;
    // ---- Q tiles -> shared memory as fp16, swizzled K-major; D / 8 neighbouring lanes share a row ----
    {
      constexpr int CPR = D / 8, kPieces = L::kQTiles * kBM * CPR / (32 * 2 * kGroupWarps);  // per thread
      uint4 raw[kPieces];
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int e = tid + i * (32 * 2 * kGroupWarps), ch = e % CPR, qr = rt.row0 + e / CPR;
        raw[i] = make_uint4(0, 0, 0, 0);
        if (qr < rt.n_rows)
          raw[i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) +
                                                        static_cast<int64_t>(rt.q0 + qr / p.n_rep) * p.q_st +
                                                        static_cast<int64_t>(hkv * p.n_rep + qr % p.n_rep) * p.q_sh) + ch);
      }
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int e = tid + i * (32 * 2 * kGroupWarps), m = e / CPR, ch = e % CPR;
        const T* x = reinterpret_cast<const T*>(&raw[i]);
        uint32_t amax = 0;
#pragma unroll
        for (int u = 0; u < 8; ++u) amax = max(amax, __float_as_uint(Elem<T>::to_f(x[u])) & 0x7fffffffu);
#pragma unroll
        for (int o = 1; o < CPR; o <<= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        // rows of zeros stay as they are, rows that are not finite become NaN
        int qe = static_cast<int>(amax >> 23) - 127 - 14;
        qe = (amax == 0 || amax >= 0x7f800000u) ? 0 : max(qe, -100);
        const float inv = q8::q_factor(amax, qe);
        uint32_t y[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) y[u] = pack2<__half>(Elem<T>::to_f(x[2 * u]) * inv, Elem<T>::to_f(x[2 * u + 1]) * inv);
        sts128(qs + (m / kBM) * L::kQ + (ch >> 3) * (kBM * 128) + sw_off(m % kBM, ch & 7), y[0], y[1], y[2], y[3]);
        if (ch == 0) s_qf[m] = __uint_as_float(static_cast<uint32_t>(127 + qe) << 23);
      }
      tc::fence_proxy_async_smem();
      asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(q_full) : "memory");
    }
    float qf = 1.f;  // this row's q factor: there once the first S is
    float m_ref = -INFINITY, l_run = 0.f;
    int vref = -1;  // reference of the values in O
    bool failed = false, row_nan = false;
    // a wait that runs out only sets `failed`: every warp still reaches every barrier
    auto wait = [&](uint32_t bar, uint32_t parity) {
      if (failed) return;
      if (!__all_sync(0xffffffffu, tc::mbar_wait(bar, parity))) failed = true;
    };
    int k = 0;
    for (; tile_at(g, k) < n_tiles; ++k) {
      const int t = tile_at(g, k);
      wait(s_full(g), k & 1);
      tc::tc_fence_after();
      if (k == 0) qf = s_qf[(ALT ? 0 : g * kBM) + row];
      const TileInfo& info = s_info[t % kInfo];
      // Not below the smallest normal number, 2^-126: a tile whose keys are all zero or absent would bring it to 0, and
      // a masked score of -inf times 0 is NaN.  |S| <= 2^31, so what real scores gain by this is below 2^-95.
      const float scale = fmaf(info.scale, qf, 0x1p-126f);
      const int tbase = t * kBN + sc0;
      const bool crosses = tbase + kSC - 1 > lim;
      const bool special = info.special != 0;
      auto mask32 = [&](float* s, int c0) {  // columns c0 .. c0 + 31 of this thread's half
        if (crosses) {
#pragma unroll
          for (int c = 0; c < 32; ++c) s[c] = (tbase + c0 + c <= lim) ? s[c] : -INFINITY;
        }
        if (special) {
          const uint32_t miss = info.missing[(sc0 + c0) >> 5];
#pragma unroll
          for (int c = 0; c < 32; ++c) s[c] = (miss >> c & 1) ? -INFINITY : s[c];
        }
      };
      // pass 1: row maximum; columns [32, 64) stay in registers for pass 2
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      float s1[32];
      {
        float s0[32];
        tc::tmem_ld32x2(ts, ts + 32, s0, s1);
        mask32(s0, 0);
        mask32(s1, 32);
        if (special) {  // rows that see a NaN value row
          const uint32_t n0 = info.vnan[sc0 >> 5], n1 = info.vnan[(sc0 + 32) >> 5];
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            row_nan |= (n0 >> c & 1) && s0[c] != -INFINITY;
            row_nan |= (n1 >> c & 1) && s1[c] != -INFINITY;
          }
        }
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          mx4[c & 3] = fmaxf(mx4[c & 3], s0[c]);
          mx4[c & 3] = fmaxf(mx4[c & 3], s1[c]);
        }
      }
      const float mxh = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
      mxg[((k & 1) * 2 + half) * kBM + row] = mxh;
      asm volatile("bar.sync %0, %1;\n" ::"r"(bar_id), "n"(64) : "memory");
      const float mx = fmaxf(mxg[((k & 1) * 2) * kBM + row], mxg[((k & 1) * 2 + 1) * kBM + row]) * scale;
      const bool need = mx > m_ref + kRescale;
      float alpha = 1.f;
      bool rescale = false;
      if (need) {
        alpha = fast_exp2(m_ref - mx);
        m_ref = mx;
        l_run *= alpha;
      }
      if (info.vref != vref) {  // the same for the whole warp
        if (k > 0) alpha *= exp2f(static_cast<float>(vref - info.vref));
        rescale = k > 0;
        vref = info.vref;
      }
      const float m_use = m_ref == -INFINITY ? 0.f : m_ref - kWOff;
      const uint64_t sc2 = pk2(scale, scale), nm2 = pk2(-m_use, -m_use);
      uint64_t sum2[2] = {0ull, 0ull};
      // pass 2: S columns [c0, c0 + 32) -> weights, high then low parts, in the same TMEM columns
      auto emit = [&](int c0, float* s) {
        uint32_t hi[16];
        [[maybe_unused]] uint32_t lo[16];
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          const uint64_t x2 = fma2(pk2(s[c], s[c + 1]), sc2, nm2);
          float ea, eb;
          up2(x2, ea, eb);
          ea = fast_exp2(ea), eb = fast_exp2(eb);
          sum2[(c >> 1) & 1] = add2(sum2[(c >> 1) & 1], pk2(ea, eb));
          if constexpr (kTwoParts) {
            split2<__half>(ea, eb, hi[c >> 1], lo[c >> 1]);
          } else {
            hi[c >> 1] = pack2<__half>(ea, eb);
          }
        }
        tc::tmem_st16_nowait(ts + c0, hi);
        if constexpr (kTwoParts) tc::tmem_st16_nowait(ts + c0 + 16, lo);
      };
      emit(32, s1);
      {
        float s0[32];
        tc::tmem_ld32(ts, s0);
        mask32(s0, 0);
        emit(0, s0);
      }
      if (rescale || (k > 0 && __any_sync(0xffffffffu, need))) {
#pragma unroll
        for (int c0 = 0; c0 < kOC; c0 += 32) {
          float o[32];
          tc::tmem_ld32(to + c0, o);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] *= alpha;
          tc::tmem_st32u(to + c0, reinterpret_cast<const uint32_t*>(o));
        }
      }
      tc::tmem_st_wait();
      {
        float sa, sb;
        up2(add2(sum2[0], sum2[1]), sa, sb);
        l_run += sa + sb;
      }
      tc::tc_fence_before();
      asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(p_full(g)) : "memory");
    }
    if (k > 0) wait(o_done(g), (k - 1) & 1);
    // ---- epilogue ----
    float* lg = s_l + g * 2 * kBM;
    lg[half * kBM + row] = l_run;
    mxg[((k & 1) * 2 + half) * kBM + row] = row_nan ? 1.f : 0.f;  // the buffer the last tile did not use
    asm volatile("bar.sync %0, %1;\n" ::"r"(bar_id), "n"(64) : "memory");
    const float l_row = lg[row] + lg[kBM + row];
    const bool bad = mxg[((k & 1) * 2) * kBM + row] + mxg[((k & 1) * 2 + 1) * kBM + row] > 0.f;
    const bool all_ok = __all_sync(0xffffffffu, !failed);
    const bool none = l_row == 0.f;  // this part sees no token
    const float nan = __int_as_float(0x7fc00000);
    // l holds 2^kWOff times the sum; O the same times 2^-(vref - 127)
    const float inv = none ? 0.f : (bad || !all_ok) ? nan : 1.f / l_row;
    const float lse = !all_ok ? nan : none ? -INFINITY : (m_ref - kWOff + log2f(l_row)) * kLn2;
    const float vf = vref < 0 ? 0.f : q8::scale_of(vref);
    const int64_t o = static_cast<int64_t>(rt.q0 + tok) * p.Hq + hkv * p.n_rep + (valid ? r % p.n_rep : 0);
    const int64_t all_rows = static_cast<int64_t>(p.total_q) * p.Hq;
    const int part = ALT ? 2 * share + g : share;
    const bool whole = !ALT && shares == 1;
    if (all_ok && k > 0) tc::tc_fence_after();
#pragma unroll
    for (int c0 = 0; c0 < kOC; c0 += 32) {
      float acc[32];
      if (all_ok && k > 0) {
        tc::tmem_ld32(to + c0, acc);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) acc[i] = 0.f;
      }
      if (valid) {
        if (whole) {
          T* dst = static_cast<T*>(p.out) + o * D + oc0 + c0;
          uint32_t y[16];
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            const bool blank = none && all_ok;
            y[c >> 1] = pack2<T>(blank ? p.empty : acc[c] * inv * vf, blank ? p.empty : acc[c + 1] * inv * vf);
          }
          if ((reinterpret_cast<uintptr_t>(p.out) & 31) == 0) {
            q8::stg256(dst, y);
            q8::stg256(dst + 16, y + 8);
          } else {
#pragma unroll
            for (int c = 0; c < 16; c += 4) *reinterpret_cast<uint4*>(dst + 2 * c) = make_uint4(y[c], y[c + 1], y[c + 2], y[c + 3]);
          }
        } else {
          float* dst = p.part_o + (part * all_rows + o) * D + oc0 + c0;
#pragma unroll
          for (int c = 0; c < 32; ++c) acc[c] = acc[c] * inv * vf;
#pragma unroll
          for (int c = 0; c < 32; c += 8) q8::stg256(dst + c, reinterpret_cast<const uint32_t*>(acc + c));
        }
      }
    }
    if (valid && half == 0) {
      if (!whole) p.part_lse[part * all_rows + o] = lse;
      else if (p.lse_out != nullptr) p.lse_out[o] = lse;
    }
    asm volatile("bar.sync 10, %0;\n" ::"n"(32 * (2 * kGroupWarps + kConvWarps)) : "memory");  // with the converters: keep->look is final
    if (keep->look != 0) {
      look_at_scales<ALT>(p, keep);
      asm volatile("bar.sync 11, %0;\n" ::"n"(32 * 2 * kGroupWarps) : "memory");
      if (keep->wide != 0 || keep->vmin < keep->vmax - kExact) exact_rows<T, D, ALT>(p, keep);  // over what was stored above
    }
  }
  if (warp == kMmaWarp && keep->stuck != 0) {  // a wait ran out: the MMAs under way end before their TMEM is given back
    const uint32_t drained = smem_u32(smem + L::kBars + 248);
    if (lane == 0) {
      tc::mbar_init(drained, 1u);
      tc::fence_mbar_init();
      tc::mma_commit(drained);
    }
    __syncwarp();
    tc::mbar_wait(drained, 0);
  }
  // the merge may be scheduled from here on; it waits for this grid itself
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, kTmemCols);
  }
}

// Joins the parts of every row that has some; one warp per row, D / 32 columns a lane.  The lanes of a warp
// first look up 32 of its rows, most of which may have been written by their CTA.
constexpr int kMergeWarps = 8;
template <typename T, int D, bool ALT>
__global__ void __launch_bounds__(32 * kMergeWarps) chunk_q8_merge_kernel(const __grid_constant__ ChunkQ8Params p) {
  constexpr int C = D / 32;
  pdl_wait();
  const int64_t all_rows = static_cast<int64_t>(p.total_q) * p.Hq;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kMergeWarps;
  const int lane = threadIdx.x & 31;
  auto parts_of = [&](int64_t o) {
    if (o >= all_rows) return 0;
    const int tok = static_cast<int>(o / p.Hq), b = p.cu_q == nullptr ? tok : q8::request_of(p.cu_q, p.B, tok);
    if (b < 0) return 0;
    const int r = (p.cu_q == nullptr ? 0 : tok - __ldg(p.cu_q + b)) * p.n_rep + static_cast<int>(o % p.Hq) % p.n_rep;
    const int tile = r / (ALT ? kBM : 2 * kBM);
    if (tile >= p.tiles) return 0;
    const int shares = p.pieces != nullptr ? __ldcg(p.n_shares + b * p.tiles + tile)
                       : tile < p.tiles - p.whole ? p.shares : 1;
    return ALT ? 2 * shares : shares > 1 ? shares : 0;
  };
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kMergeWarps + (threadIdx.x >> 5); first < all_rows; first += 32 * step) {
    const int my_parts = parts_of(first + lane * step);
    for (uint32_t left = __ballot_sync(0xffffffffu, my_parts > 0); left != 0; left &= left - 1) {
      const int src_lane = __ffs(left) - 1;
      const int parts = __shfl_sync(0xffffffffu, my_parts, src_lane);
      const int64_t o = first + src_lane * step;
      // lane i holds the log-sum-exp, then the weight, of parts i, i + 32, ... (at most kMaxParts of them)
      float w[kMaxParts / 32], M = -INFINITY;
      bool nan = false;
#pragma unroll
      for (int u = 0; u < kMaxParts / 32; ++u) {
        w[u] = u * 32 + lane < parts ? p.part_lse[(u * 32 + lane) * all_rows + o] : -INFINITY;
        nan |= w[u] != w[u];
        M = fmaxf(M, w[u]);
      }
      for (int s = 16; s > 0; s >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, s));
      nan = __any_sync(0xffffffffu, nan);
      float a[C] = {}, W = 0.f;
#pragma unroll
      for (int u = 0; u < kMaxParts / 32; ++u) {
        w[u] = w[u] == -INFINITY ? 0.f : exp2f((w[u] - M) * 1.4426950408889634f);
        W += w[u];
      }
      for (int s = 16; s > 0; s >>= 1) W += __shfl_xor_sync(0xffffffffu, W, s);
      const bool blank = M == -INFINITY && !nan;
      const float inv = nan ? __int_as_float(0x7fc00000) : blank ? 0.f : 1.f / W;
#pragma unroll
      for (int u = 0; u < kMaxParts / 32; ++u) {
        w[u] *= inv;  // before the sums: those of the largest values stay in range
        const int n = min(32, parts - u * 32);
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
          const float wi = __shfl_sync(0xffffffffu, w[u], i);
          const float* src = p.part_o + ((u * 32 + i) * all_rows + o) * D + lane * C;  // a part without tokens holds zeros
#pragma unroll
          for (int k = 0; k < C; ++k) a[k] += wi * src[k];
        }
      }
      T* dst = static_cast<T*>(p.out) + o * D + lane * C;
#pragma unroll
      for (int k = 0; k < C; k += 2) *reinterpret_cast<uint32_t*>(dst + k) = pack2<T>(blank ? p.empty : a[k], blank ? p.empty : a[k + 1]);
      if (lane == 0 && p.lse_out != nullptr) p.lse_out[o] = nan ? inv : M == -INFINITY ? -INFINITY : M + logf(W);
    }
  }
}

template <typename T, int D, bool ALT>
int launch_chunk(const ChunkQ8Params& p, cudaStream_t st) {
  auto kern = chunk_q8_kernel<T, D, ALT>;
  constexpr int kBytes = Layout<D, ALT>::kBytes;
  static bool raised[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !raised[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes) != cudaSuccess) {
      set_error("q8_attention_launch:smem_attr");
      return BPKV_ERR_CUDA;
    }
    if (dev >= 0 && dev < 64) raised[dev] = true;
  }
  const dim3 grid(static_cast<unsigned>(p.n_pieces) * p.Hkv);
  cudaError_t e = cudaSuccess;
  if (p.pieces != nullptr) {
    chunk_q8_plan_kernel<ALT><<<1, kPlanThreads, 0, st>>>(p);
    e = launch_pdl(kern, grid, dim3(kThreads), kBytes, st, p);
  } else {
    kern<<<grid, kThreads, kBytes, st>>>(p);
  }
  if (e == cudaSuccess && (ALT || p.max_shares > 1)) {
    const int64_t rows = static_cast<int64_t>(p.total_q) * p.Hq;
    const int64_t blocks = (rows + kMergeWarps - 1) / kMergeWarps, most = 8 * p.sms;
    e = launch_pdl(chunk_q8_merge_kernel<T, D, ALT>, dim3(static_cast<unsigned>(blocks < most ? blocks : most)), dim3(32 * kMergeWarps), 0, st, p);
  }
  if (e != cudaSuccess) {
    set_error("q8_attention_launch:%s", cudaGetErrorString(e));
    return BPKV_ERR_CUDA;
  }
  BPKV_RETURN_LAUNCH("q8_attention_launch");
}

template <typename T, int D>
int launch(const ChunkQ8Params& p, cudaStream_t st) {
  return p.alt ? launch_chunk<T, D, true>(p, st) : launch_chunk<T, D, false>(p, st);
}

}  // namespace

int chunk_q8_tc_launch(const ChunkQ8Params& p, int head_dim, int dtype, cudaStream_t st) {
  if (dtype == BPKV_BF16) return head_dim == 64 ? launch<__nv_bfloat16, 64>(p, st) : launch<__nv_bfloat16, 128>(p, st);
  return head_dim == 64 ? launch<__half, 64>(p, st) : launch<__half, 128>(p, st);
}

}  // namespace bpkv
