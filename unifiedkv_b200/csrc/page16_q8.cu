// Attention of a few query rows per KV head over 8-bit pages: one-token decode,
// drafted tokens, and short or narrow chunks (sm_100a, mma.sync).
//
// For one request and KV head the rows are its (query token, query head) pairs,
// token-major, cut into tiles of R = 8 * NT rows; an item is one tile.  With
// x[t, r] = scale * q_r . k_t and p = exp(x - max),
//   out_r = sum_t p[t, r] v_t / sum_t p[t, r],   t <= limit(r)
// where k_t = code * 2^(byte - 127) and v_t likewise.
//
// Design:
//  * Bound.  Decode reads 2 * (head_dim + 1) bytes per token and KV head and does
//    4 * head_dim * n_rep FLOP on them: HBM-bound, half the bytes of 16-bit pages, so
//    half the instructions per token may be spent to stay so.
//  * No dequantised copy.  e4m3 codes are exact in fp16 (cvt.rn.f16x2.e4m3x2, one
//    instruction per pair), so the MMAs run on raw codes: the key's scale multiplies
//    the score in fp32, the value's scale multiplies the weight in fp32 before it is
//    rounded to fp16 (off by 2^-11 of it at most, against 2^-8 for the bf16 output).
//    fp16 outputs keep 11 bits themselves: their weights go in as a high and a low
//    part, two MMAs.  Weights are kept in units of 2^(reference value scale - 12): they
//    reach 2^15 at most.  The reference follows the pages' scales, and a page whose scales
//    span 2^8 and more is walked once per span, so that a weight holds 11 bits down to
//    2^-18 of the row's largest and vanishes at 2^-30 of it whatever else the page or the
//    request holds: a huge value that a row does not see, or gives no weight to, takes
//    nothing from it (up to a ratio of 2^72).
//  * q is scaled per row by a power of two into [2^14, 2^15) and rounded to fp16:
//    exact for fp16 and bf16 elements down to 2^-29 of the row's largest, and off by
//    at most 2^-40 of it below that.
//  * Tokens are the M rows of the MMA and query rows its N columns (S^T = K Q^T,
//    O^T = V^T P^T): 8 columns hold the n_rep <= 8 query heads of a GQA group, where
//    16-row query tiles would leave three quarters of the tensor work empty.  A lane
//    loads its K fragment as 16-byte pieces of one row (the dot product does not mind
//    the order of head_dim, q is loaded in the same order), V^T comes by
//    ldmatrix.trans on code pairs, and movmatrix transposes the weights.
//  * Work split.  All items' pages form one list, cut into equal ranges for W workers;
//    a worker is one warp per KV head (HP warps), and a CTA has several workers when
//    there are few KV heads.  A worker's first and last item may be shared with its
//    neighbours: it leaves (o, lse) in its slot 0 or 1, and q8_combine_kernel merges
//    them.  With very many items (long chunks) no item is split: worker w takes items
//    w, w + W, ... and there is no merge.
//  * Loads: a ring of NS pages per warp filled by cp.async, no block barriers.
//  * head_dim 256: two warps share a head, half its dimensions each, and exchange scores through shared
//    memory: half the accumulators a warp (15 x 7-58 new over 58-174 tokens 118 us with one warp a
//    head, 91 so; decode, latency-bound, unchanged).
//
// Measured (8 KV heads, head_dim 128, 32 query heads, bf16; attention / combine kernel, each launch by
// itself with a cold cache): 32 requests of 4K-32K tokens 165 / 9 us for 972 MB (5.9 TB/s, 90 % of the
// measured copy rate; the call 176 us), one of 131072 52 / 11 for 271 MB (61); 16 requests with 16 rows
// each 67 / 13 for 200 MB (68): two MMA columns of tiles double the arithmetic per byte and leave
// 8 warps an SM, whose dependent chains bound it (issue slots 44 % active).  What mattered most beside
// the MMA layout was code size: exact power-of-two factors in place of scalbnf took 16 rows from 94 to
// 69 us a call and head_dim 256 from 43 to 38.  Following the value scales costs 32 requests 0 to
// 3 us of 173, from machine to machine.
#include <math.h>
#include <string.h>

#include <type_traits>

#include "chunk_q8.cuh"
#include "q8.cuh"

namespace bpkv {

struct Q8Params {
  const void* q;
  const uint8_t* kc;
  const uint8_t* vc;
  const uint8_t* ks;
  const uint8_t* vs;
  const int32_t* bt;
  const int32_t* lens;  // cached tokens of a request, the new ones included
  const int32_t* cu_q;  // null: request b has the one query row b
  void* out;            // [total_q, Hq, D] contiguous
  float* lse_out;       // [total_q, Hq] or null
  int32_t* g_prefix;    // workspace: [items + 1]
  float* part_lse;      // workspace: [2 W][Hkv][R]
  float* part_o;        // workspace: [2 W][Hkv][R][D]
  int B, total_q, Hq, Hkv, n_rep, max_blocks, num_pages, tiles, n_items, split, causal, rows_max, hp, pl;
  float empty;          // value of a row that sees no key
  int64_t q_st, q_sh, page_stride, scale_stride, bt_sb;
  float scale_log2;
};

namespace {

constexpr float kLn2 = 0.6931471805599453f;
constexpr float kMaxLazy = 3.f;  // a row's reference may lag its maximum by this (log2): p <= 2^3
constexpr int kWOff = 12;        // weights are held as p * 2^(byte - vref + 12) <= 2^15
constexpr int kVSpan = 8;        // of the value scales that one reference serves: bytes in (vref - 8, vref]
constexpr int kVDeep = 72;       // the reference stays within this of its highest: O * 2^72 does not overflow
constexpr int kAllBytes = 255;

struct Item {
  int b, q0, row0, n_rows, len, n_q;  // rows [row0, row0 + R) of n_rows; first packed token q0
};

template <int R>
__device__ __forceinline__ Item item_of(const Q8Params& p, int i) {
  Item it;
  it.b = i / p.tiles;
  it.row0 = (i % p.tiles) * R;
  it.q0 = p.cu_q == nullptr ? it.b : __ldg(p.cu_q + it.b);
  it.n_q = p.cu_q == nullptr ? 1 : __ldg(p.cu_q + it.b + 1) - it.q0;
  it.n_rows = it.q0 < 0 ? 0 : min(it.n_q, p.total_q - it.q0) * p.n_rep;  // q has total_q rows, whatever cu_q says
  it.len = __ldg(p.lens + it.b);
  return it;
}
// Tokens that query token i of the request sees (before the table's width cuts them).
__device__ __forceinline__ int visible(const Q8Params& p, const Item& it, int i) {
  return p.causal ? it.len - it.n_q + i + 1 : it.len;
}
template <int R>
__device__ __forceinline__ int item_tokens(const Q8Params& p, const Item& it) {
  if (it.row0 >= it.n_rows) return 0;
  const int last = (min(it.row0 + R, it.n_rows) - 1) / p.n_rep;
  return min(max(visible(p, it, last), 0), p.max_blocks * kPage);
}
template <int R>
__device__ __forceinline__ int item_pages(const Q8Params& p, int i) {
  return (item_tokens<R>(p, item_of<R>(p, i)) + kPage - 1) / kPage;
}

// Block-wide exclusive scan of the items' page counts into prefix[0..n_items].
template <int R>
__device__ void build_item_prefix(const Q8Params& p, int* prefix) {
  __shared__ int wsum[32];
  const int nt = blockDim.x, tid = threadIdx.x, n = p.n_items;
  const int lane = tid & 31, warp = tid >> 5;
  const int per = (n + nt - 1) / nt;
  const int beg = min(tid * per, n), end = min(beg + per, n);
  int local = 0;
  for (int i = beg; i < end; ++i) {
    const int c = item_pages<R>(p, i);
    prefix[i] = c;
    local += c;
  }
  int incl = local;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) wsum[warp] = incl;
  __syncthreads();
  int before = 0;
  for (int w = 0; w < warp; ++w) before += wsum[w];
  int run = before + incl - local;
  for (int i = beg; i < end; ++i) {
    const int c = prefix[i];
    prefix[i] = run;
    run += c;
  }
  if (tid == nt - 1) prefix[n] = run;
  __syncthreads();
}

// Largest i with prefix[i] <= s (s < prefix[n]): the item that owns flattened page s.
__device__ __forceinline__ int find_item(const int* prefix, int n, int s) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= s) lo = mid; else hi = mid;
  }
  return lo;
}
// Equal shares of `total` pages for W workers: the first total % W take one more.  With fewer pages than
// workers the first `total` workers have a page each.
struct Shares {
  int per, more;
  __device__ __forceinline__ Shares(int total, int W) : per(total / W), more(total % W) {}
  __device__ __forceinline__ int start(int c) const { return c * per + min(c, more); }
  __device__ __forceinline__ int owner(int page) const {
    const int big = more * (per + 1);
    return page < big ? page / (per + 1) : more + (page - big) / per;  // per > 0 where a page lies past `big`
  }
};

// A worker's walk over its pages: item by item, pages [page, end) of each.
template <int R>
struct Walk {
  int item, page, end, next;  // next: first flattened page not yet visited (split), or next item (not split)
  int tokens, ids, ids_next, k;  // loader only: tokens of the item; lane l's ids are pages page - k + l, and 32 on
  const int32_t* bt_row;
  __device__ __forceinline__ bool live() const { return item >= 0; }
};
template <int R>
__device__ __forceinline__ void walk_next(const Q8Params& p, const int* prefix, int worker, int W, int s_end, Walk<R>& w) {
  if (p.split) {
    if (w.next >= s_end) {
      w.item = -1;
      return;
    }
    if (w.item < 0) w.item = find_item(prefix, p.n_items, w.next);
    else do { ++w.item; } while (prefix[w.item + 1] == prefix[w.item]);
    w.page = w.next - prefix[w.item];
    const int stop = min(s_end, prefix[w.item + 1]);
    w.end = stop - prefix[w.item];
    w.next = stop;
  } else {
    // longest items last in the list: take them first
    for (;;) {
      if (w.next >= p.n_items) {
        w.item = -1;
        return;
      }
      w.item = p.n_items - 1 - w.next;
      w.next += W;
      w.page = 0;
      w.end = item_pages<R>(p, w.item);
      if (w.end > 0) return;
    }
  }
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ int lds_u8(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];\n" : "=r"(v) : "r"(addr));
  return static_cast<int>(v);
}

// Position of 16-byte piece ch of row r inside a tile, such that both the row-wise reads of K and the
// 8-row ldmatrix of V touch all banks once.
template <int D>
__device__ __forceinline__ uint32_t piece(int r, int ch) {
  const int x = D == 64 ? (r >> 1) & 3 : r & 7;
  return static_cast<uint32_t>(r * D + ((ch ^ x) << 4));
}

// D: head_dim; DS: warps that share a KV head, DW dimensions each (2 for head_dim 256, whose accumulators would
// take a warp's registers twice over).  They add their halves of every score through shared memory.
template <typename T, int D, int DS, int NT, int NW, int NS>
__global__ void __launch_bounds__(NW * 32, 1) q8_attend_kernel(Q8Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int R = 8 * NT, DW = D / DS;
  constexpr int TILEB = 16 * DW;
  constexpr int STAGEB = 2 * TILEB + 64;  // K, V, 16 + 16 scale bytes, number of live rows
  constexpr int CH = DW / 16;             // 16-byte pieces per row
  constexpr int KS = DW / 16;             // MMA k-steps of S
  constexpr int MT = DW / 16;             // 16-row tiles of O^T

  float4* s_pair = reinterpret_cast<float4*>(smem + NW * NS * STAGEB);  // DS == 2: [2 buffers][NW][NT][32]
  int* prefix = reinterpret_cast<int*>(s_pair + (DS == 2 ? 2 * NW * NT * 32 : 0));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int W = gridDim.x * p.pl;
  if (p.split) {
    build_item_prefix<R>(p, prefix);
    if (blockIdx.x == 0 && blockIdx.y == 0)
      for (int i = threadIdx.x; i <= p.n_items; i += blockDim.x) p.g_prefix[i] = prefix[i];
  }
  // rows that see no key
  for (int i = blockIdx.x; i < p.n_items; i += gridDim.x) {
    if (p.split ? prefix[i + 1] != prefix[i] : item_pages<R>(p, i) != 0) continue;
    const Item it = item_of<R>(p, i);
    const int rows = min(R, it.n_rows - it.row0);
    const int hb = blockIdx.y * p.hp, nh = min(p.hp, p.Hkv - hb);
    for (int e = threadIdx.x; e < rows * nh * D; e += blockDim.x) {
      const int d = e % D, r = it.row0 + (e / D) % rows, h = hb + e / (D * rows);
      const int64_t o = static_cast<int64_t>(it.q0 + r / p.n_rep) * p.Hq + h * p.n_rep + r % p.n_rep;
      static_cast<T*>(p.out)[o * D + d] = Elem<T>::from_f(p.empty);
      if (d == 0 && p.lse_out != nullptr) p.lse_out[o] = -INFINITY;
    }
  }
  const int part = warp % DS, hw = warp / DS;
  const int h = blockIdx.y * p.hp + hw % p.hp;
  const int worker = blockIdx.x * p.pl + hw / p.hp;
  if (hw / p.hp >= p.pl || h >= p.Hkv) return;
  // the two warps of a head meet here (DS == 2); they walk over the same pages
  auto meet = [&]() { asm volatile("bar.sync %0, 64;\n" ::"r"(1 + hw) : "memory"); };
  int turn = 0;  // buffer of s_pair
  int s_beg = 0, s_end = 0;
  if (p.split) {
    const Shares sh(prefix[p.n_items], W);
    s_beg = sh.start(worker), s_end = sh.start(worker + 1);
  }

  const uint32_t ring = smem_u32(smem + warp * NS * STAGEB);
  const int g = lane >> 2, c = lane & 3;

  // ---- loader: one page of this head into a ring stage ----
  const int64_t row_stride = static_cast<int64_t>(p.Hkv) * D;
  // this lane's pieces are ch0 of rows tok0, tok0 + 32 / CH, ...
  const int tok0 = lane / CH, ch0 = lane % CH;
  const int64_t lane_off = static_cast<int64_t>(h) * D + part * DW + tok0 * row_stride + ch0 * 16;
  auto issue = [&](const Walk<R>& w, int stage) {
    const int page = __shfl_sync(0xffffffffu, w.ids, w.k);
    // rows past the item's last visible token are zero-filled, so that what a page holds there never
    // reaches the MMAs
    const int live = page < 0 ? 0 : min(kPage, w.tokens - w.page * kPage);
    const int64_t off = page < 0 ? 0 : page * p.page_stride + lane_off;
    const uint8_t *kp = p.kc + off, *vp = p.vc + off;
    const uint32_t sk = ring + stage * STAGEB;
#pragma unroll
    for (int r = 0; r < CH / 2; ++r) {
      const int tok = tok0 + r * (32 / CH);
      const bool ok = tok < live;
      const int64_t o = ok ? r * (32 / CH) * row_stride : 0;
      const uint32_t so = piece<DW>(tok, ch0);
      cp_async16(sk + so, kp + o, ok);
      cp_async16(sk + TILEB + so, vp + o, ok);
    }
    if (lane < 2) {
      const uint8_t* sp = (lane == 0 ? p.ks : p.vs) + (page < 0 ? 0 : page * p.scale_stride + h * kPage);
      cp_async16(sk + 2 * TILEB + 16 * lane, sp, page >= 0);
    } else if (lane == 2) {
      asm volatile("st.shared.b32 [%0], %1;\n" ::"r"(sk + 2 * TILEB + 32), "r"(live) : "memory");
    }
  };

  Walk<R> ld, cs;
  ld.item = cs.item = -1;
  ld.page = cs.page = ld.end = cs.end = 0;
  ld.next = cs.next = p.split ? s_beg : worker;
  // 32 block-table entries a load, the next 32 under way: one dependent load per item, not per page
  auto ids_at = [&](int page) { return page + lane < ld.end ? q8::page_of(ld.bt_row, page + lane, p.max_blocks, p.num_pages) : -1; };
  auto load_seek = [&]() {  // the loader's next item
    walk_next<R>(p, prefix, worker, W, s_end, ld);
    if (ld.live()) {
      const Item it = item_of<R>(p, ld.item);
      ld.tokens = item_tokens<R>(p, it);
      ld.bt_row = p.bt + static_cast<int64_t>(it.b) * p.bt_sb;
      ld.ids = ids_at(ld.page);
      ld.ids_next = ids_at(ld.page + 32);
      ld.k = 0;
    }
  };
  load_seek();
  auto load_one = [&](int stage) {
    if (ld.live()) {
      issue(ld, stage);
      if (++ld.page == ld.end) {
        load_seek();
      } else if (++ld.k == 32) {
        ld.ids = ld.ids_next;
        ld.ids_next = ids_at(ld.page + 32);
        ld.k = 0;
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) load_one(i);

  int it_stage = 0;
  bool first_segment = true;
  for (walk_next<R>(p, prefix, worker, W, s_end, cs); cs.live(); walk_next<R>(p, prefix, worker, W, s_end, cs)) {
    const Item it = item_of<R>(p, cs.item);
    const int tokens = item_tokens<R>(p, it);
    const bool whole = cs.page == 0 && cs.end * kPage >= tokens;
    // ---- q: fragment column g of every N tile is row row0 + 8 nt + g, pieces 2c + (j & 1) + 8 (j >> 1) ----
    uint32_t qb[NT][KS][2];
    float rf[NT][2];   // scale * log2(e) * 2^(row exponent) of columns 2c, 2c + 1
    int lim[NT][2];    // last visible token of those rows
    int lim_min = 0x7fffffff;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = it.row0 + 8 * nt + g;
      const bool ok = r < it.n_rows;
      const T* qr = static_cast<const T*>(p.q) + static_cast<int64_t>(it.q0 + (ok ? r / p.n_rep : 0)) * p.q_st +
                    static_cast<int64_t>(h * p.n_rep + (ok ? r % p.n_rep : 0)) * p.q_sh + part * DW;
      uint4 raw[2 * (CH / 4)];
      uint32_t amax = 0;
#pragma unroll
      for (int j = 0; j < CH / 4; ++j) {
        const int ch = DW == 64 ? c : 2 * c + (j & 1) + 8 * (j >> 1);
        const uint4* src = reinterpret_cast<const uint4*>(qr + ch * 16);
        raw[2 * j] = ok ? __ldg(src) : make_uint4(0, 0, 0, 0);
        raw[2 * j + 1] = ok ? __ldg(src + 1) : make_uint4(0, 0, 0, 0);
      }
      const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
      for (int i = 0; i < DW / 4; ++i) amax = max(amax, __float_as_uint(Elem<T>::to_f(e[i])) & 0x7fffffffu);
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      if constexpr (DS == 2) {  // one exponent for the whole row
        // in the warp's own part of the buffer, as below: only the two warps wait for each other
        uint32_t* x = reinterpret_cast<uint32_t*>(s_pair + turn * NW * NT * 32);
        x[warp * NT * 128 + lane] = amax;
        meet();
        amax = max(amax, x[(warp ^ 1) * NT * 128 + lane]);
        turn ^= 1;
      }
      // exponent that brings the largest element into [2^14, 2^15); rows of zeros stay as they are, rows that are not
      // finite become NaN
      int qe = static_cast<int>(amax >> 23) - 127 - 14;
      qe = (amax == 0 || amax >= 0x7f800000u) ? 0 : max(qe, -100);
      const float inv = q8::q_factor(amax, qe);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const T* x = e + 4 * s;
        qb[nt][s][0] = pack2<__half>(Elem<T>::to_f(x[0]) * inv, Elem<T>::to_f(x[1]) * inv);
        qb[nt][s][1] = pack2<__half>(Elem<T>::to_f(x[2]) * inv, Elem<T>::to_f(x[3]) * inv);
      }
      const float f = p.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 + qe) << 23);
#pragma unroll
      for (int e2 = 0; e2 < 2; ++e2) {
        rf[nt][e2] = __shfl_sync(0xffffffffu, f, (2 * c + e2) * 4);
        const int rr = it.row0 + 8 * nt + 2 * c + e2;
        lim[nt][e2] = rr < it.n_rows ? visible(p, it, rr / p.n_rep) - 1 : 0x7fffffff;
        lim_min = min(lim_min, lim[nt][e2]);
      }
    }
    lim_min = __reduce_min_sync(0xffffffffu, lim_min);

    float acc[NT][MT][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) acc[nt][mt][0] = acc[nt][mt][1] = acc[nt][mt][2] = acc[nt][mt][3] = 0.f;
    }
    int vref = 0, vtop = 0;  // value-scale byte whose unit the weights and O are in; the highest so far
    int below = kAllBytes;   // less: the page is walked again, for its tokens with value-scale bytes up to this

    while (cs.page < cs.end) {
      if (below == kAllBytes) {
        load_one((it_stage + NS - 1) % NS);
        cp_async_wait<NS - 1>();
        __syncwarp();
      }
      const uint32_t sk = ring + (it_stage % NS) * STAGEB;
      const uint32_t sv = sk + TILEB, ss = sk + 2 * TILEB;
      int live;
      asm volatile("ld.shared.b32 %0, [%1];\n" : "=r"(live) : "r"(ss + 32));
      const int t0 = cs.page * kPage;
      // V codes: lane (mi, row) of ldmatrix addresses token (row + 8 (mi & 1)), piece mt + (mi >> 1)
      auto load_v = [&](int mt, uint32_t* r) {
        const int tok = (lane & 7) + 8 * ((lane >> 3) & 1);
        ldmatrix_x4_trans(sv + piece<DW>(tok, mt + (lane >> 4)), r[0], r[1], r[2], r[3]);
      };
      uint32_t vr[MT / 2][4];  // into registers before the softmax, which hides their latency
#pragma unroll
      for (int mt = 0; mt < MT; mt += 2) load_v(mt, vr[mt / 2]);
      const bool ok0 = g < live, ok1 = g + 8 < live;
      const int kb0 = lds_u8(ss + g), kb1 = lds_u8(ss + g + 8);
      int vb0 = ok0 ? lds_u8(ss + 16 + g) : 0, vb1 = ok1 ? lds_u8(ss + 16 + g + 8) : 0;
      // ---- S^T = K Q^T: rows tokens g, g + 8; columns query rows; two chains of MMAs ----
      float s[NT][4];
      {
        float s2[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][e] = s2[nt][e] = 0.f;
#pragma unroll
        for (int j = 0; j < CH / 4; ++j) {
          const int ch = DW == 64 ? c : 2 * c + (j & 1) + 8 * (j >> 1);
          const uint4 ka = lds128(sk + piece<DW>(g, ch)), kb = lds128(sk + piece<DW>(g + 8, ch));
          const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t a[4];
            q8::e4m3x4_to_f16x4(wa[w], a[0], a[2]);
            q8::e4m3x4_to_f16x4(wb[w], a[1], a[3]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816<__half>(w & 1 ? s2[nt] : s[nt], a, qb[nt][4 * j + w][0], qb[nt][4 * j + w][1]);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][e] += s2[nt][e];
        if constexpr (DS == 2) {
          float4* x = s_pair + turn * NW * NT * 32;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) x[(warp * NT + nt) * 32 + lane] = make_float4(s[nt][0], s[nt][1], s[nt][2], s[nt][3]);
          meet();
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float4 y = x[((warp ^ 1) * NT + nt) * 32 + lane];  // the sum of two has no order
            s[nt][0] += y.x, s[nt][1] += y.y, s[nt][2] += y.z, s[nt][3] += y.w;
          }
          turn ^= 1;
        }
      }
      // ---- scores, online softmax in log2 ----
      const float kf0 = q8::scale_of(kb0), kf1 = q8::scale_of(kb1);
      const bool edge = live < kPage || t0 + kPage - 1 > lim_min;
      // Rare, and looked for with one vote: a row whose maximum outgrew its reference, a value scale above the
      // reference (byte 255, not finite, among them) or far below it (byte 0, zeros, apart), a further walk.
      bool rare = max(vb0, vb1) > vref || static_cast<int>(min(vb0 - 1u, vb1 - 1u) & 0x7fffffffu) < vref - kVSpan ||
                  below < kAllBytes;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[nt][e] *= rf[nt][e] * kf0;
          s[nt][2 + e] *= rf[nt][e] * kf1;
          if (edge) {
            s[nt][e] = (ok0 && t0 + g <= lim[nt][e]) ? s[nt][e] : -INFINITY;
            s[nt][2 + e] = (ok1 && t0 + g + 8 <= lim[nt][e]) ? s[nt][2 + e] : -INFINITY;
          }
          rare |= fmaxf(s[nt][e], s[nt][2 + e]) > m[nt][e] + kMaxLazy;
        }
      }
      if (__any_sync(0xffffffffu, rare)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(s[nt][e], s[nt][2 + e]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float mn = fmaxf(m[nt][e], mx);
            const float a = mn == -INFINITY ? 1.f : fast_exp2(m[nt][e] - mn);
            m[nt][e] = mn;
            l[nt][e] *= a;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              acc[nt][mt][e] *= a;
              acc[nt][mt][2 + e] *= a;
            }
          }
        }
        // a value row that is not finite: its codes are taken out, and the rows that see it become NaN
        if (__any_sync(0xffffffffu, vb0 == q8::kNanByte || vb1 == q8::kNanByte)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              bool bad = (vb0 == q8::kNanByte && s[nt][e] != -INFINITY) || (vb1 == q8::kNanByte && s[nt][2 + e] != -INFINITY);
              uint32_t who = __ballot_sync(0xffffffffu, bad);
              who |= who >> 16, who |= who >> 8, who |= who >> 4;
              if (who >> c & 1) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) acc[nt][mt][e] = acc[nt][mt][2 + e] = __int_as_float(0x7fc00000);
              }
            }
          }
          for (int t = 0; t < kPage; ++t) {
            const bool bad = t < live && lds_u8(ss + 16 + t) == q8::kNanByte;
            if (bad && lane < CH)
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n" ::"r"(sv + piece<DW>(t, lane)), "r"(0) : "memory");
          }
          if (vb0 == q8::kNanByte) vb0 = 0;
          if (vb1 == q8::kNanByte) vb1 = 0;
          __syncwarp();
#pragma unroll
          for (int mt = 0; mt < MT; mt += 2) load_v(mt, vr[mt / 2]);
        }
        // The unit follows the page's largest value scale (of the tokens not yet taken) up, or down when that is
        // far below.  What then still lies below the span waits for another walk over the page: one unit would
        // round those tokens' weights away, although a row may see none of the larger ones.
        int vmax = __reduce_max_sync(0xffffffffu, max(vb0 <= below ? vb0 : 0, vb1 <= below ? vb1 : 0));
        vmax = vmax == 0 ? vref : max(vmax, vtop - kVDeep);
        if (vmax > vref || vmax <= vref - kVSpan) {
          // 2^(vref - vmax), exact; far below: nothing of the old sum is left
          const float a = vmax - vref > 126 ? 0.f : __uint_as_float(static_cast<uint32_t>(127 + vref - vmax) << 23);
          vref = vmax;
          vtop = max(vtop, vref);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[nt][mt][e] *= a;
        }
        // (a walk's unit is at or below the last one's cut, so there are at most kVDeep / kVSpan + 1 of them)
        const int cut = vref - kVSpan >= vtop - kVDeep ? vref - kVSpan : 0;
        const bool later0 = vb0 > 0 && vb0 <= cut, later1 = vb1 > 0 && vb1 <= cut;
        const bool again = __any_sync(0xffffffffu, later0 || later1);
        if (again || below < kAllBytes) {
          const bool out0 = later0 || vb0 > below || (vb0 == 0 && below < kAllBytes);
          const bool out1 = later1 || vb1 > below || (vb1 == 0 && below < kAllBytes);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              s[nt][e] = out0 ? -INFINITY : s[nt][e];
              s[nt][2 + e] = out1 ? -INFINITY : s[nt][2 + e];
            }
          }
        }
        below = again ? cut : kAllBytes;
      }
      const int ve0 = vb0 - vref + kWOff + 127, ve1 = vb1 - vref + kWOff + 127;
      const float vf0 = ve0 > 0 ? __uint_as_float(static_cast<uint32_t>(ve0) << 23) : 0.f;
      const float vf1 = ve1 > 0 ? __uint_as_float(static_cast<uint32_t>(ve1) << 23) : 0.f;
      constexpr bool kTwoParts = std::is_same<T, __half>::value;
      uint32_t pb[NT][2], pl[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float mu = m[nt][e] == -INFINITY ? 0.f : m[nt][e];
          const float p0 = fast_exp2(s[nt][e] - mu), p1 = fast_exp2(s[nt][2 + e] - mu);
          l[nt][e] += p0 + p1;
          w[e] = p0 * vf0;
          w[2 + e] = p1 * vf1;
        }
        if constexpr (kTwoParts) {
          split2<__half>(w[0], w[1], pb[nt][0], pl[nt][0]);
          split2<__half>(w[2], w[3], pb[nt][1], pl[nt][1]);
          pl[nt][0] = movmatrix_trans(pl[nt][0]);
          pl[nt][1] = movmatrix_trans(pl[nt][1]);
        } else {
          pb[nt][0] = pack2<__half>(w[0], w[1]);
          pb[nt][1] = pack2<__half>(w[2], w[3]);
        }
        pb[nt][0] = movmatrix_trans(pb[nt][0]);
        pb[nt][1] = movmatrix_trans(pb[nt][1]);
      }
      // ---- O^T += V^T P^T ----
#pragma unroll
      for (int mt = 0; mt < MT; mt += 2) {
        const uint32_t* r = vr[mt / 2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          // bytes (token 2c: d, d + 1; token 2c + 1: d, d + 1) -> (d: both tokens), (d + 1: both tokens)
          uint32_t a[4];
          q8::e4m3x4_to_f16x4(__byte_perm(r[2 * u], 0, 0x3120), a[0], a[1]);
          q8::e4m3x4_to_f16x4(__byte_perm(r[2 * u + 1], 0, 0x3120), a[2], a[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma16816<__half>(acc[nt][mt + u], a, pb[nt][0], pb[nt][1]);
            if constexpr (kTwoParts) mma16816<__half>(acc[nt][mt + u], a, pl[nt][0], pl[nt][1]);
          }
        }
      }
      __syncwarp();
      if (below == kAllBytes) {
        it_stage = it_stage + 1 == NS ? 0 : it_stage + 1;
        ++cs.page;
      }
    }

    // ---- finish the item (or this worker's share of it) ----
    const int slot = 2 * worker + (first_segment ? 0 : 1);
    first_segment = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float L = l[nt][e];
        L += __shfl_xor_sync(0xffffffffu, L, 4);
        L += __shfl_xor_sync(0xffffffffu, L, 8);
        L += __shfl_xor_sync(0xffffffffu, L, 16);
        const int rl = 8 * nt + 2 * c + e, r = it.row0 + rl;
        if (r >= it.n_rows) continue;
        const bool none = m[nt][e] == -INFINITY && L == 0.f;
        const float inv = none ? 0.f : 1.f / L;
        const float vf = q8::scale_of(vref), vd = 1.f / (1 << kWOff);  // the weights' unit, in two exact steps
        const float lse = none ? -INFINITY : (m[nt][e] + log2f(L)) * kLn2;
        const int64_t o = static_cast<int64_t>(it.q0 + r / p.n_rep) * p.Hq + h * p.n_rep + r % p.n_rep;
        const int64_t po = (static_cast<int64_t>(slot) * p.Hkv + h) * R + rl;
        if (whole) {
          T* dst = static_cast<T*>(p.out) + o * D + part * DW + 2 * g;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            const float y0 = none ? p.empty : acc[nt][mt][e] * inv * vd * vf;
            const float y1 = none ? p.empty : acc[nt][mt][2 + e] * inv * vd * vf;
            *reinterpret_cast<uint32_t*>(dst + mt * 16) = pack2<T>(y0, y1);
          }
          if (g == 0 && part == 0 && p.lse_out != nullptr) p.lse_out[o] = lse;
        } else {
          float* dst = p.part_o + po * D + part * DW + 2 * g;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            *reinterpret_cast<float2*>(dst + mt * 16) =
                make_float2(acc[nt][mt][e] * inv * vd * vf, acc[nt][mt][2 + e] * inv * vd * vf);
          if (g == 0 && part == 0) p.part_lse[po] = lse;
        }
      }
    }
  }
  cp_async_wait<0>();
  // the combine may be scheduled from here on; it waits for this grid itself
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Merges the items that several workers share.  CTA = (unit, one query row); a unit is an
// item when there are no more items than workers, otherwise the boundary between workers
// u and u + 1.  The weights of the parts are formed once, in shared memory; warp w then sums
// parts w, w + warps, ..., a lane D / 32 columns.  (Every warp scanning all log-sum-exps for
// itself needs one barrier less and gains nothing for a few parts, 5.8 against 5.6 us, but takes
// 17.6 against 8.5 for 296 of them.)
constexpr int kCombMaxWarps = 32;
constexpr int kMaxWorkers = 2560;  // parts of one item: their weights fit in shared memory

template <typename T, int D, int R>
__global__ void __launch_bounds__(kCombMaxWarps * 32) q8_combine_kernel(Q8Params p, int W, int by_item) {
  extern __shared__ float s_w[];  // [parts], at most W
  __shared__ float s_red[2][kCombMaxWarps];
  __shared__ float s_acc[kCombMaxWarps][D];
  constexpr int C = D / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
  // what the caller gave is there already: this grid starts after the attention kernel has
  Item it{};
  if (by_item) it = item_of<R>(p, blockIdx.x);
  pdl_wait();
  const int total = p.g_prefix[p.n_items];
  int item = blockIdx.x;
  int first = by_item ? p.g_prefix[item] : 0, last = by_item ? p.g_prefix[item + 1] : 0;
  if (total == 0) return;
  const Shares sh(total, W);
  if (!by_item) {
    const int s = sh.start(blockIdx.x + 1);
    if (s >= total) return;
    item = find_item(p.g_prefix, p.n_items, s);
    // this boundary is the item's first one: worker blockIdx.x has its first page
    const int first0 = p.g_prefix[item];
    if (first0 >= s || sh.start(blockIdx.x) > first0) return;
    it = item_of<R>(p, item);
    first = first0, last = p.g_prefix[item + 1];
  }
  if (first == last) return;  // written by the attention kernel
  const int c_lo = sh.owner(first), n = sh.owner(last - 1) - c_lo + 1;
  if (n == 1) return;  // one worker had all of it
  const int h = blockIdx.y / p.rows_max, rl = blockIdx.y % p.rows_max;
  const int r = it.row0 + rl;
  if (r >= it.n_rows) return;
  // The item is the last one of worker c_lo (slot 1, or slot 0 if that worker begins with it) and the
  // first one of the workers after it (slot 0).
  const int64_t step = 2 * static_cast<int64_t>(p.Hkv) * R;
  const int64_t part0 = (static_cast<int64_t>(2 * c_lo) * p.Hkv + h) * R + rl;
  const int64_t lead = sh.start(c_lo) < first ? static_cast<int64_t>(p.Hkv) * R : 0;
  auto part = [&](int i) { return part0 + i * step + (i == 0 ? lead : 0); };
  const float nan = __int_as_float(0x7fc00000);
  float M = -INFINITY;  // NaN once any part is (fmaxf alone would drop it)
  auto over_warp = [&](float x) {
    for (int o = 16; o > 0; o >>= 1) {
      const float y = __shfl_xor_sync(0xffffffffu, x, o);
      x = (x != x || y != y) ? nan : fmaxf(x, y);
    }
    return x;
  };
  for (int i = tid; i < n; i += blockDim.x) {
    const float x = p.part_lse[part(i)];
    s_w[i] = x;
    M = (x != x || M != M) ? nan : fmaxf(M, x);
  }
  M = over_warp(M);
  if (lane == 0) s_red[0][warp] = M;
  __syncthreads();
  M = over_warp(lane < nw ? s_red[0][lane] : -INFINITY);
  float L = 0.f;
  for (int i = tid; i < n; i += blockDim.x) {
    const float w = M == -INFINITY ? 0.f : exp2f((s_w[i] - M) * 1.4426950408889634f);
    s_w[i] = w;
    L += w;
  }
  for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
  if (lane == 0) s_red[1][warp] = L;
  __syncthreads();
  L = lane < nw ? s_red[1][lane] : 0.f;
  for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
  const float inv = M == -INFINITY ? 0.f : 1.f / L;  // into the weights: sums of the largest values stay in range
  float a[C] = {};
#pragma unroll 8
  for (int i = warp; i < n; i += nw) {
    const float w = s_w[i] * inv;
    const float* src = p.part_o + part(i) * D + lane * C;
    float x[C];
    if constexpr (C == 2) *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(src);
    else
#pragma unroll
      for (int k = 0; k < C; k += 4) *reinterpret_cast<float4*>(x + k) = *reinterpret_cast<const float4*>(src + k);
    // a part of a worker that saw none of its tokens (w = 0) holds zeros; NaN parts stay NaN
#pragma unroll
    for (int k = 0; k < C; ++k) a[k] += w * x[k];
  }
#pragma unroll
  for (int k = 0; k < C; ++k) s_acc[warp][lane * C + k] = a[k];
  __syncthreads();
  const int64_t o = static_cast<int64_t>(it.q0 + r / p.n_rep) * p.Hq + h * p.n_rep + r % p.n_rep;
  for (int d = tid; d < D; d += blockDim.x) {
    float y = 0.f;
#pragma unroll 8
    for (int w = 0; w < nw; ++w) y += s_acc[w][d];
    static_cast<T*>(p.out)[o * D + d] = Elem<T>::from_f(M == -INFINITY ? p.empty : y);
  }
  if (tid == 0 && p.lse_out != nullptr) p.lse_out[o] = M == -INFINITY ? -INFINITY : M + logf(L);
}

// ---- host side ----------------------------------------------------------------
inline size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// Items whose page counts fit beside the rings in shared memory.
constexpr int max_split_items(int D) { return D == 256 ? 2048 : 4096; }

// Rows per request and KV head above which the tensor-core chunk kernel takes over (head_dim 64 and 128,
// positive softmax scale).  Measured, 16 requests of 8192 tokens, 8 KV heads, this kernel / that one: head_dim
// 128: 32 rows 141 / 192 us, 64 rows 250 / 196; head_dim 64: 108 / 149, 189 / 153.
constexpr int kTcRows = 32;

// The chunk kernel may cut the tokens of a row tile into shares, a CTA each.  Estimated in K/V tiles of 128
// tokens: a CTA costs its tiles and about nine more (start, first tile, last output), and two more where it leaves
// a part to be joined.
//
// One request: the host chooses, as if it were as long as the table is wide (over a table much wider than the request
// its shares are short).  Candidates are
// zero to two full waves of CTAs whole, the rest in s shares.  Measured (32 heads, 8 KV heads, head_dim
// 128), 1 share / chosen: 512 new tokens of 32768 732 / 389 us, 128 new of 32768 718 / 117, 2048 new of 32768
// (256 CTAs; 144 whole, 112 in 4 shares) 1461 / 1326.
//
// A batch over a wide table: chunk_q8_plan_kernel, which knows the lengths, chooses.  Over a narrow one all row tiles
// are cut into s shares, 2 at least if they fit one wave, since the longest request sets the time.  What decides is how
// unequal the lengths are, which the host does not know: it goes by the table's width, below which the plan's time
// (about 6 us, and the CTAs left over some more) is won back by very unequal lengths only.  Measured, s shares /
// planned: 8 x 64 new over 2048 tokens each 52 / 58 us, over 3900 77 / 86, 6 x 1-333 over 170-3000 59 / 72 (but over
// 100-3900 76 / 54); above it 4 x 64 over 200-8000 73 / 55, 16 x 16 over 2000-16000 173 / 174, 16 x 32 over 8192 each
// 196 / 179.
constexpr int kPlanTokens = 4096;
void choose_shares(int row_tiles, int Hkv, int64_t tokens, int most, bool batch, int& whole, int& shares) {
  const int sms = sm_count();
  const float tiles = static_cast<float>(tokens) / 128.f;
  const int fewest = batch && static_cast<int64_t>(row_tiles) * Hkv <= sms ? min(2, most) : 1;
  float least = 1e30f;
  for (int w = 0; w < (batch ? 1 : 3); ++w) {
    const int n = static_cast<int>(min(static_cast<int64_t>(row_tiles), static_cast<int64_t>(w) * sms / Hkv));
    if (w > 0 && (n == 0 || n == row_tiles)) continue;
    for (int s = w == 0 ? fewest : 2; s <= most; ++s) {
      const float pieces = n + static_cast<float>(s) * (row_tiles - n), waves = pieces * Hkv / sms;
      const float cut = tiles / s + (s > 1 ? 11.f : 9.f), first = n > 0 ? tiles + 9.f : cut;
      const float t = fmaxf(first, (n * (tiles + 9.f) + s * (row_tiles - n) * cut) * Hkv / sms + (ceilf(waves) - waves) * cut);
      if (t < least) least = t, whole = n, shares = s;
    }
  }
}

// Shares that a row tile may be cut into: this bounds the CTAs and the parts' memory (8 x 256 rows per SM).  A
// share is 512 tokens at least.
int most_shares(int64_t ctas, int64_t tokens, int most) {
  const int64_t sms = sm_count();
  const int64_t s = ctas <= sms / 2 ? 2 * sms / ctas : ctas <= 2 * sms ? max(static_cast<int64_t>(4), 4 * sms / ctas) : 1;
  return static_cast<int>(max(static_cast<int64_t>(1), min(min(s, static_cast<int64_t>(most)), (tokens + 511) / 512)));
}

struct Plan {
  int tc, alt, planned, ranked, whole, max_shares, n_pieces;  // chunk_q8_tc.cu's, else the rest
  int nt, nw, groups, hp, pl, grid, tiles, n_items, split;
  size_t shares_off, lse_off, o_off, bytes;
};

Plan make_plan(int B, int total_q, int Hkv, int n_rep, int D, int max_q, int max_blocks, float scale) {
  Plan pl{};
  const int64_t rows = static_cast<int64_t>(max_q) * n_rep;
  if (D <= 128 && rows > kTcRows && scale > 0.f) {
    pl.tc = 1;
    pl.alt = rows <= 128;
    const int64_t tiles = (rows + (pl.alt ? 127 : 255)) / (pl.alt ? 128 : 256);
    const int64_t ctas = tiles * B * Hkv;
    pl.tiles = static_cast<int>(tiles);
    pl.n_items = tiles * B < (1LL << 30) && ctas < (1LL << 30) ? static_cast<int>(tiles * B) : -1;
    const int sms = sm_count();
    const int64_t tokens = static_cast<int64_t>(max_blocks) * kPage;
    pl.n_pieces = pl.n_items;
    pl.max_shares = most_shares(ctas, tokens, pl.alt ? kMaxParts / 2 : kMaxParts);
    if (pl.n_items <= 0) {
      pl.max_shares = 1;
    } else if (B > 1 && tokens >= kPlanTokens && pl.n_items <= kMaxRanked && pl.max_shares > 1) {
      pl.planned = 1;
      pl.n_pieces = min(pl.n_items * pl.max_shares, pl.n_items + 2 * sms / Hkv);
      pl.shares_off = up256(sizeof(int2) * pl.n_pieces);
      pl.bytes = pl.lse_off = pl.shares_off + up256(sizeof(int32_t) * pl.n_items);
    } else {
      choose_shares(pl.n_items, Hkv, tokens, pl.max_shares, B > 1, pl.whole, pl.max_shares);
      pl.n_pieces = pl.whole + (pl.n_items - pl.whole) * pl.max_shares;
      pl.ranked = B > 1 && pl.n_items <= kMaxRanked && static_cast<int64_t>(pl.n_pieces) * Hkv > sms;
    }
    const int parts = pl.max_shares * (pl.alt ? 2 : 1);
    if (parts > 1) {
      const size_t all_rows = static_cast<size_t>(total_q) * Hkv * n_rep;
      pl.o_off = pl.lse_off + up256(sizeof(float) * parts * all_rows);
      pl.bytes = pl.o_off + sizeof(float) * parts * all_rows * D;
    }
    return pl;
  }
  pl.nt = rows <= 8 ? 1 : 2;
  pl.nw = pl.nt == 1 ? 16 : 8;
  const int per_head = D == 256 ? 2 : 1, heads = min(8, pl.nw / per_head);  // warps of a head, heads of a CTA
  pl.groups = (Hkv + heads - 1) / heads;
  pl.hp = (Hkv + pl.groups - 1) / pl.groups;
  pl.pl = pl.nw / per_head / pl.hp;
  const int sms = sm_count();
  pl.grid = max(1, min(sms / pl.groups, kMaxWorkers / pl.pl));
  const int64_t tiles = (rows + 8 * pl.nt - 1) / (8 * pl.nt);
  const int64_t items = tiles * B;
  pl.tiles = static_cast<int>(tiles);
  pl.n_items = items < (1LL << 30) ? static_cast<int>(items) : -1;
  pl.split = items <= max_split_items(D);
  if (pl.split) {
    const size_t slots = 2 * static_cast<size_t>(pl.grid) * pl.pl * Hkv * 8 * pl.nt;
    pl.lse_off = up256(sizeof(int32_t) * (items + 1));
    pl.o_off = pl.lse_off + up256(sizeof(float) * slots);
    pl.bytes = pl.o_off + sizeof(float) * slots * D;
  }
  return pl;
}

template <typename T, int D, int NT, int NW, int NS>
int launch_attend(Q8Params& p, const Plan& pl, cudaStream_t st) {
  constexpr int DS = D == 256 ? 2 : 1;
  constexpr size_t ring = static_cast<size_t>(NW) * NS * (2 * 16 * (D / DS) + 64) + (DS == 2 ? 2 * NW * NT * 512 : 0);
  const size_t smem = ring + (pl.split ? sizeof(int) * (pl.n_items + 1) : 0);
  static_assert(ring + 4 * (max_split_items(D) + 1) + 1024 <= 232448, "shared memory");
  auto kern = q8_attend_kernel<T, D, DS, NT, NW, NS>;
  static bool raised[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !raised[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(ring + sizeof(int) * (max_split_items(D) + 1))) != cudaSuccess) {
      set_error("q8_attention_launch:smem_attr");
      return BPKV_ERR_CUDA;
    }
    if (dev >= 0 && dev < 64) raised[dev] = true;
  }
  kern<<<dim3(pl.grid, pl.groups), NW * 32, smem, st>>>(p);
  if (pl.split) {
    const int W = pl.grid * pl.pl;
    const int by_item = pl.n_items <= W;
    const dim3 grid(by_item ? pl.n_items : W - 1, p.Hkv * p.rows_max);
    if (W > 1) {
      // about as many warps as an item has parts, 2 to 32, but no more than the SMs hold at once
      int warps = 2;
      while (warps < kCombMaxWarps && static_cast<int64_t>(warps) * pl.n_items < W &&
             static_cast<int64_t>(2 * warps) * grid.x * grid.y <= 64LL * sm_count())
        warps *= 2;
      const cudaError_t e = launch_pdl(q8_combine_kernel<T, D, 8 * NT>, grid, dim3(warps * 32), sizeof(float) * W, st, p, W, by_item);
      if (e != cudaSuccess) {
        set_error("q8_attention_launch:%s", cudaGetErrorString(e));
        return BPKV_ERR_CUDA;
      }
    }
  }
  BPKV_RETURN_LAUNCH("q8_attention_launch");
}

template <typename T>
int dispatch(Q8Params& p, const Plan& pl, int D, cudaStream_t st) {
  if (D == 64) {
    if (pl.nt == 1) return launch_attend<T, 64, 1, 16, 5>(p, pl, st);
    return launch_attend<T, 64, 2, 8, 8>(p, pl, st);
  }
  if (D == 128) {
    if (pl.nt == 1) return launch_attend<T, 128, 1, 16, 3>(p, pl, st);
    return launch_attend<T, 128, 2, 8, 5>(p, pl, st);
  }
  if (pl.nt == 1) return launch_attend<T, 256, 1, 16, 3>(p, pl, st);
  return launch_attend<T, 256, 2, 8, 5>(p, pl, st);
}

}  // namespace
}  // namespace bpkv

using namespace bpkv;

extern "C" BPKV_API size_t bpkv_q8_attention_workspace_size(int batch, int total_q, int num_q_heads, int num_kv_heads,
                                                            int head_dim, int max_blocks, int max_seqlen_q,
                                                            float softmax_scale) {
  if (batch <= 0 || total_q <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads || max_seqlen_q <= 0 ||
      !(head_dim == 64 || head_dim == 128 || head_dim == 256))
    return 0;
  return make_plan(batch, total_q, num_kv_heads, num_q_heads / num_kv_heads, head_dim, max_seqlen_q, max_blocks, softmax_scale)
      .bytes;
}

extern "C" BPKV_API int bpkv_q8_attention(const void* q, const void* k_codes, const void* v_codes,
                                          const uint8_t* k_scales, const uint8_t* v_scales, const int32_t* block_table,
                                          const int32_t* cu_seqlens_q, const int32_t* seqlens_k, void* out,
                                          float* lse_out, int batch, int total_q, int num_q_heads, int num_kv_heads, int head_dim,
                                          int max_blocks, int num_pages, int max_seqlen_q, int64_t q_stride_t,
                                          int64_t q_stride_h, int64_t page_stride, int64_t scale_stride,
                                          int64_t bt_stride_b, float softmax_scale, int causal, int empty_nan,
                                          int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  const char* what = "q8_attention_shape_unsupported";
  BPKV_CHECK_ARG(batch >= 0 && total_q >= 0 && num_q_heads > 0 && max_blocks >= 0 && num_pages >= 0, "%s:empty", what);
  BPKV_CHECK_ARG(num_kv_heads > 0 && num_q_heads % num_kv_heads == 0, "%s:gqa", what);
  BPKV_CHECK_ARG(num_kv_heads <= 1024, "%s:kv_heads_%d", what, num_kv_heads);
  BPKV_CHECK_ARG(head_dim == 64 || head_dim == 128 || head_dim == 256, "%s:head_dim_%d", what, head_dim);
  BPKV_CHECK_ARG(dtype == BPKV_F16 || dtype == BPKV_BF16, "%s:dtype_%d", what, dtype);
  BPKV_CHECK_ARG(cu_seqlens_q != nullptr || (max_seqlen_q == 1 && total_q == batch), "%s:max_seqlen_q", what);
  if (batch == 0 || total_q == 0 || max_seqlen_q <= 0) return BPKV_OK;
  BPKV_CHECK_ARG(q && k_codes && v_codes && k_scales && v_scales && seqlens_k && out && (block_table || max_blocks == 0),
                 "%s:null_pointer", what);
  BPKV_CHECK_ARG(aligned16(q) && aligned16(k_codes) && aligned16(v_codes) && aligned16(k_scales) && aligned16(v_scales) &&
                     aligned16(out) && q_stride_t % 8 == 0 && q_stride_h % 8 == 0 && page_stride % 16 == 0 &&
                     scale_stride % 16 == 0,
                 "%s:alignment", what);
  BPKV_CHECK_ARG(max_blocks <= (1 << 26), "%s:max_blocks_%d", what, max_blocks);
  const int n_rep = num_q_heads / num_kv_heads;
  const Plan pl = make_plan(batch, total_q, num_kv_heads, n_rep, head_dim, max_seqlen_q, max_blocks, softmax_scale);
  BPKV_CHECK_ARG(pl.n_items > 0, "%s:max_seqlen_q", what);
  // the flattened page list is indexed in 31 bits
  BPKV_CHECK_ARG(pl.tc || !pl.split || static_cast<int64_t>(pl.n_items) * max_blocks < (1LL << 31), "%s:max_blocks_%d", what, max_blocks);
  if (pl.bytes > 0 && (workspace == nullptr || workspace_bytes < pl.bytes)) {
    set_error("q8_attention_workspace:need_%zu_bytes", pl.bytes);
    return BPKV_ERR_WORKSPACE;
  }
  BPKV_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 31) == 0, "%s:workspace_alignment", what);
  if (pl.tc) {
    ChunkQ8Params c{};
    c.q = q;
    c.kc = static_cast<const uint8_t*>(k_codes);
    c.vc = static_cast<const uint8_t*>(v_codes);
    c.ks = k_scales;
    c.vs = v_scales;
    c.bt = block_table;
    c.cu_q = cu_seqlens_q;
    c.lens = seqlens_k;
    c.out = out;
    c.lse_out = lse_out;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    if (pl.planned) {
      c.pieces = reinterpret_cast<int2*>(ws);
      c.n_shares = reinterpret_cast<int32_t*>(ws + pl.shares_off);
    }
    c.part_lse = reinterpret_cast<float*>(ws + pl.lse_off);
    c.part_o = reinterpret_cast<float*>(ws + pl.o_off);
    c.B = batch;
    c.Hq = num_q_heads;
    c.Hkv = num_kv_heads;
    c.n_rep = n_rep;
    c.tiles = pl.tiles;
    c.whole = pl.whole;
    c.shares = c.max_shares = pl.max_shares;
    c.ranked = pl.ranked;
    c.n_pieces = pl.n_pieces;
    c.sms = sm_count();
    c.alt = pl.alt;
    c.causal = causal;
    c.max_blocks = max_blocks;
    c.num_pages = num_pages;
    c.total_q = total_q;
    c.q_st = q_stride_t;
    c.q_sh = q_stride_h;
    c.page_stride = page_stride;
    c.scale_stride = scale_stride;
    c.bt_sb = bt_stride_b;
    c.scale_log2 = softmax_scale * 1.4426950408889634f;
    c.empty = empty_nan ? NAN : 0.f;
    return chunk_q8_tc_launch(c, head_dim, dtype, static_cast<cudaStream_t>(stream));
  }
  Q8Params p{};
  p.q = q;
  p.kc = static_cast<const uint8_t*>(k_codes);
  p.vc = static_cast<const uint8_t*>(v_codes);
  p.ks = k_scales;
  p.vs = v_scales;
  p.bt = block_table;
  p.lens = seqlens_k;
  p.cu_q = cu_seqlens_q;
  p.out = out;
  p.lse_out = lse_out;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.g_prefix = reinterpret_cast<int32_t*>(ws);
  p.part_lse = reinterpret_cast<float*>(ws + pl.lse_off);
  p.part_o = reinterpret_cast<float*>(ws + pl.o_off);
  p.B = batch;
  p.total_q = total_q;
  p.Hq = num_q_heads;
  p.Hkv = num_kv_heads;
  p.n_rep = n_rep;
  p.max_blocks = max_blocks;
  p.num_pages = num_pages;
  p.tiles = pl.tiles;
  p.n_items = pl.n_items;
  p.split = pl.split;
  p.causal = causal;
  const int64_t rows = static_cast<int64_t>(max_seqlen_q) * n_rep;
  p.rows_max = rows < 8 * pl.nt ? static_cast<int>(rows) : 8 * pl.nt;
  p.hp = pl.hp;
  p.pl = pl.pl;
  p.empty = empty_nan ? NAN : 0.f;
  p.q_st = q_stride_t;
  p.q_sh = q_stride_h;
  p.page_stride = page_stride;
  p.scale_stride = scale_stride;
  p.bt_sb = bt_stride_b;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == BPKV_BF16 ? dispatch<__nv_bfloat16>(p, pl, head_dim, st) : dispatch<__half>(p, pl, head_dim, st);
}
