// Writing rows of K and V into 8-bit pages, and reading ranges of them back.
//
// Both are bound by HBM: a row is read once and written once, with a handful of
// instructions per element.  A block takes a few tokens with all their heads: it looks
// their slots up once (request, page, position), into shared memory, and its threads then
// walk over the (token, head, 16-element piece) items.  head_dim / 16 neighbouring threads
// share a row, so a warp touches whole 128-byte lines.  Measured at 32768 tokens, 8 KV heads,
// head_dim 128, bf16 (201.9 MB): write 36 us, 86 % of the measured copy rate (8 elements a
// thread, maxima in fp32: 50 us), read back 37.5 us, 82 % (stores of half sectors: 43 us).
#include "q8.cuh"

namespace bpkv {
namespace {

struct AppendParams {
  const void* k_new;
  const void* v_new;
  uint8_t* kc;
  uint8_t* vc;
  uint8_t* ks;
  uint8_t* vs;
  const int32_t* bt;
  const int32_t* cu_q;  // null: token b is request b's
  const int32_t* seqlens_k;
  int batch, total, Hkv, max_blocks, num_pages, tokens;
  int64_t k_st, k_sh, v_st, v_sh, page_stride, scale_stride, bt_sb;
};

// Sixteen consecutive elements as loaded.
template <typename T>
struct Raw {
  uint4 q[sizeof(T)];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) q[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  }
  // Bits of the largest magnitude, as a float's.  16-bit magnitudes compare as integers too (a NaN above an
  // infinity above every number), two at a time.
  __device__ __forceinline__ uint32_t amax() const {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(q);
    uint32_t m = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 16; ++i) m = max(m, w[i] & 0x7fffffffu);
      return m;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
      const uint16_t b = static_cast<uint16_t>(max(m & 0xffffu, m >> 16));
      return __float_as_uint(Elem<T>::to_f(*reinterpret_cast<const T*>(&b)));
    }
  }
  __device__ __forceinline__ uint32_t codes4(int i, float scale) const {  // elements 4 i .. 4 i + 3
    const T* e = reinterpret_cast<const T*>(q) + 4 * i;
    return q8::to_e4m3x2(Elem<T>::to_f(e[0]) * scale, Elem<T>::to_f(e[1]) * scale) |
           q8::to_e4m3x2(Elem<T>::to_f(e[2]) * scale, Elem<T>::to_f(e[3]) * scale) << 16;
  }
};

// Quantises a row that G neighbouring lanes hold.
template <int G, typename T>
__device__ __forceinline__ void store_row(const Raw<T>& x, uint8_t* codes, uint8_t* scale, int lane_in_row, bool live) {
  uint32_t amax = x.amax();
#pragma unroll
  for (int o = 1; o < G; o <<= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  const int byte = q8::scale_byte(amax);
  uint4 c;
  if (byte == q8::kNanByte) {
    c = make_uint4(0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu);
  } else {
    // 2^-e, e = byte - 127 in [-127, 119]: a normal number, so the products are exact (or far below the
    // smallest code)
    const float inv = __uint_as_float(static_cast<uint32_t>(254 - byte) << 23);
    c = make_uint4(x.codes4(0, inv), x.codes4(1, inv), x.codes4(2, inv), x.codes4(3, inv));
  }
  if (live) {
    *reinterpret_cast<uint4*>(codes + lane_in_row * 16) = c;
    if (lane_in_row == 0) *scale = static_cast<uint8_t>(byte);
  }
}

constexpr int kMaxTokens = 64;  // of a block

// Slot of a token: its page (-1: none) and position in it.
struct Slots {
  int page[kMaxTokens], slot[kMaxTokens];
};

template <typename T, int D>
__global__ void __launch_bounds__(256) q8_append_kernel(AppendParams p) {
  constexpr int G = D / 16;
  __shared__ Slots s;
  const int t0 = blockIdx.x * p.tokens, n_tok = min(p.tokens, p.total - t0);
  const int items = n_tok * p.Hkv * G;
  // the lookups of the first threads run beside everybody's first loads
  if (threadIdx.x < n_tok) {
    const int i = t0 + threadIdx.x;
    const int b = p.cu_q == nullptr ? i : q8::request_of(p.cu_q, p.batch, i);
    int page = -1, pos = 0;
    if (b >= 0) {
      pos = __ldg(p.seqlens_k + b) - (p.cu_q == nullptr ? 1 : __ldg(p.cu_q + b + 1) - i);
      if (pos >= 0) page = q8::page_of(p.bt + static_cast<int64_t>(b) * p.bt_sb, pos / kPage, p.max_blocks, p.num_pages);
    }
    s.page[threadIdx.x] = page;
    s.slot[threadIdx.x] = pos & (kPage - 1);
  }
  const int lr = threadIdx.x % G;
  bool looked_up = false;
  for (int e0 = 0; e0 < items; e0 += 256) {
    const int e = e0 + threadIdx.x;
    const int row = min(e, items - 1) / G, t = row / p.Hkv, h = row % p.Hkv;
    Raw<T> k{}, v{};
    if (e < items) {
      k.load(static_cast<const T*>(p.k_new) + (t0 + t) * p.k_st + h * p.k_sh + lr * 16);
      v.load(static_cast<const T*>(p.v_new) + (t0 + t) * p.v_st + h * p.v_sh + lr * 16);
    }
    if (!looked_up) {
      __syncthreads();
      looked_up = true;
    }
    const int page = s.page[t], slot = s.slot[t];
    // the lanes of a row agree on `live`; the others only take part in the shuffles
    const bool live = e < items && page >= 0;
    const int64_t off = live ? page * p.page_stride + (static_cast<int64_t>(slot) * p.Hkv + h) * D : 0;
    const int64_t soff = live ? page * p.scale_stride + h * kPage + slot : 0;
    store_row<G>(k, p.kc + off, p.ks + soff, lr, live);
    store_row<G>(v, p.vc + off, p.vs + soff, lr, live);
  }
}

struct ReadParams {
  const uint8_t* kc;
  const uint8_t* vc;
  const uint8_t* ks;
  const uint8_t* vs;
  const int32_t* bt;
  const int32_t* cu;
  const int32_t* starts;  // null: every range starts at token 0
  void* k_out;
  void* v_out;
  int batch, total, Hkv, max_blocks, num_pages, tokens, wide;
  int64_t page_stride, scale_stride, bt_sb, o_st, o_sh;
};

// Sixteen values in one go: whole 32-byte sectors where the output is aligned to them (`wide`).
template <typename T>
__device__ __forceinline__ void store16(T* p, const float* x, bool wide) {
  constexpr int kWords = 4 * sizeof(T);
  uint32_t y[kWords];
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    if constexpr (sizeof(T) == 4) y[i] = __float_as_uint(x[i]);
    else y[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
  }
  uint32_t* dst = reinterpret_cast<uint32_t*>(p);
  if (wide) {
#pragma unroll
    for (int i = 0; i < kWords; i += 8) q8::stg256(dst + i, y + i);
  } else {
#pragma unroll
    for (int i = 0; i < kWords; i += 4) *reinterpret_cast<uint4*>(dst + i) = make_uint4(y[i], y[i + 1], y[i + 2], y[i + 3]);
  }
}

__device__ __forceinline__ void values16(const uint4& c, float s, float* x) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t lo, hi;
    q8::e4m3x4_to_f16x4(w[i], lo, hi);
    const float2 a = __half22float2(*reinterpret_cast<__half2*>(&lo)), b = __half22float2(*reinterpret_cast<__half2*>(&hi));
    x[4 * i] = a.x * s;  // exact: s is a power of two
    x[4 * i + 1] = a.y * s;
    x[4 * i + 2] = b.x * s;
    x[4 * i + 3] = b.y * s;
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(256) q8_read_kernel(ReadParams p) {
  constexpr int G = D / 16, kUnroll = 2;
  __shared__ Slots s;
  const int t0 = blockIdx.x * p.tokens, n_tok = min(p.tokens, p.total - t0);
  const int items = n_tok * p.Hkv * G;
  if (threadIdx.x < n_tok) {
    const int i = t0 + threadIdx.x;
    const int b = q8::request_of(p.cu, p.batch, i);
    int page = -2, pos = 0;  // rows outside every sequence stay as they were
    if (b >= 0) {
      pos = (p.starts == nullptr ? 0 : __ldg(p.starts + b)) + i - __ldg(p.cu + b);
      page = pos < 0 ? -1 : q8::page_of(p.bt + static_cast<int64_t>(b) * p.bt_sb, pos / kPage, p.max_blocks, p.num_pages);
    }
    s.page[threadIdx.x] = page;
    s.slot[threadIdx.x] = pos & (kPage - 1);
  }
  __syncthreads();
  const int lr = threadIdx.x % G;
  for (int e0 = threadIdx.x; e0 < items; e0 += 256 * kUnroll) {
    uint4 k[kUnroll], v[kUnroll];
    float sk[kUnroll], sv[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int e = e0 + u * 256;
      k[u] = v[u] = make_uint4(0, 0, 0, 0);  // a token without a page reads as zeros
      sk[u] = sv[u] = 0.f;
      if (e >= items) continue;
      const int row = e / G, t = row / p.Hkv, h = row % p.Hkv, page = s.page[t], slot = s.slot[t];
      if (page < 0) continue;
      const int64_t off = page * p.page_stride + (static_cast<int64_t>(slot) * p.Hkv + h) * D + lr * 16;
      const int64_t soff = page * p.scale_stride + h * kPage + slot;
      k[u] = __ldg(reinterpret_cast<const uint4*>(p.kc + off));
      v[u] = __ldg(reinterpret_cast<const uint4*>(p.vc + off));
      sk[u] = q8::scale_of(__ldg(p.ks + soff));
      sv[u] = q8::scale_of(__ldg(p.vs + soff));
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int e = e0 + u * 256;
      if (e >= items) break;
      const int row = e / G, t = row / p.Hkv, h = row % p.Hkv;
      if (s.page[t] == -2) continue;
      const int64_t o = (t0 + t) * p.o_st + h * p.o_sh + lr * 16;
      float x[16];
      values16(k[u], sk[u], x);
      store16(static_cast<T*>(p.k_out) + o, x, p.wide);
      values16(v[u], sv[u], x);
      store16(static_cast<T*>(p.v_out) + o, x, p.wide);
    }
  }
}

// Tokens of a block: two items a thread (one, four, eight: 38, 37, 42 us for the write that takes 36 with
// two), but no fewer blocks than the SMs can hold twice over.
int block_tokens(int total, int items_per_token) {
  const int fill = max(1, 512 / items_per_token);
  return min(min(fill, kMaxTokens), max(1, total / (2 * sm_count())));
}

int check_pages(const char* what, const void* kc, const void* vc, const void* ks, const void* vs, int Hkv, int D,
                int num_pages, int64_t page_stride, int64_t scale_stride) {
  BPKV_CHECK_ARG(Hkv > 0 && num_pages >= 0, "%s_shape_unsupported:empty", what);
  BPKV_CHECK_ARG(Hkv <= 1024, "%s_shape_unsupported:kv_heads_%d", what, Hkv);
  BPKV_CHECK_ARG(D == 64 || D == 128 || D == 256, "%s_shape_unsupported:head_dim_%d", what, D);
  BPKV_CHECK_ARG(kc && vc && ks && vs, "%s_shape_unsupported:null_pointer", what);
  BPKV_CHECK_ARG(aligned16(kc) && aligned16(vc) && aligned16(ks) && aligned16(vs) && page_stride % 16 == 0 &&
                     scale_stride % 16 == 0,
                 "%s_shape_unsupported:alignment", what);
  return BPKV_OK;
}

}  // namespace
}  // namespace bpkv

using namespace bpkv;

extern "C" BPKV_API int bpkv_q8_append(const void* k_new, const void* v_new, void* k_codes, void* v_codes,
                                       uint8_t* k_scales, uint8_t* v_scales, const int32_t* block_table,
                                       const int32_t* cu_seqlens_q, const int32_t* seqlens_k, int batch, int total_q,
                                       int num_kv_heads, int head_dim, int max_blocks, int num_pages,
                                       int64_t k_stride_t, int64_t k_stride_h, int64_t v_stride_t, int64_t v_stride_h,
                                       int64_t page_stride, int64_t scale_stride, int64_t bt_stride_b, int dtype,
                                       void* stream) {
  clear_error();
  const int rc = check_pages("q8_append", k_codes, v_codes, k_scales, v_scales, num_kv_heads, head_dim, num_pages,
                             page_stride, scale_stride);
  if (rc != BPKV_OK) return rc;
  BPKV_CHECK_ARG(batch >= 0 && total_q >= 0 && max_blocks >= 0, "q8_append_shape_unsupported:empty");
  BPKV_CHECK_ARG(dtype == BPKV_F32 || dtype == BPKV_F16 || dtype == BPKV_BF16, "q8_append_shape_unsupported:dtype_%d", dtype);
  BPKV_CHECK_ARG(cu_seqlens_q != nullptr || total_q == batch, "q8_append_shape_unsupported:seqlens");
  if (batch == 0 || total_q == 0 || max_blocks == 0) return BPKV_OK;
  BPKV_CHECK_ARG(k_new && v_new && block_table && seqlens_k, "q8_append_shape_unsupported:null_pointer");
  const int64_t per16 = dtype == BPKV_F32 ? 4 : 8;
  BPKV_CHECK_ARG(aligned16(k_new) && aligned16(v_new) && k_stride_t % per16 == 0 && k_stride_h % per16 == 0 &&
                     v_stride_t % per16 == 0 && v_stride_h % per16 == 0,
                 "q8_append_shape_unsupported:alignment");
  AppendParams p{k_new, v_new, static_cast<uint8_t*>(k_codes), static_cast<uint8_t*>(v_codes), k_scales, v_scales,
                 block_table, cu_seqlens_q, seqlens_k, batch, total_q, num_kv_heads, max_blocks, num_pages,
                 block_tokens(total_q, num_kv_heads * (head_dim / 16)), k_stride_t, k_stride_h, v_stride_t, v_stride_h, page_stride, scale_stride, bt_stride_b};
  const unsigned grid = static_cast<unsigned>((total_q + p.tokens - 1) / p.tokens);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define BPKV_APPEND(T)                                                        \
  do {                                                                        \
    if (head_dim == 64) q8_append_kernel<T, 64><<<grid, 256, 0, st>>>(p);     \
    else if (head_dim == 128) q8_append_kernel<T, 128><<<grid, 256, 0, st>>>(p); \
    else q8_append_kernel<T, 256><<<grid, 256, 0, st>>>(p);                   \
  } while (0)
  if (dtype == BPKV_F32) BPKV_APPEND(float);
  else if (dtype == BPKV_F16) BPKV_APPEND(__half);
  else BPKV_APPEND(__nv_bfloat16);
#undef BPKV_APPEND
  BPKV_RETURN_LAUNCH("q8_append_launch");
}

extern "C" BPKV_API int bpkv_q8_dequantize(const void* k_codes, const void* v_codes, const uint8_t* k_scales,
                                           const uint8_t* v_scales, const int32_t* block_table,
                                           const int32_t* cu_seqlens, const int32_t* starts, void* k_out, void* v_out,
                                           int batch, int total, int num_kv_heads, int head_dim, int max_blocks,
                                           int num_pages, int64_t page_stride, int64_t scale_stride,
                                           int64_t bt_stride_b, int64_t out_stride_t, int64_t out_stride_h, int dtype,
                                           void* stream) {
  clear_error();
  const int rc = check_pages("q8_dequantize", k_codes, v_codes, k_scales, v_scales, num_kv_heads, head_dim, num_pages,
                             page_stride, scale_stride);
  if (rc != BPKV_OK) return rc;
  BPKV_CHECK_ARG(batch >= 0 && total >= 0 && max_blocks >= 0, "q8_dequantize_shape_unsupported:empty");
  BPKV_CHECK_ARG(dtype == BPKV_F32 || dtype == BPKV_F16 || dtype == BPKV_BF16, "q8_dequantize_shape_unsupported:dtype_%d", dtype);
  if (batch == 0 || total == 0) return BPKV_OK;
  BPKV_CHECK_ARG(cu_seqlens && k_out && v_out && (block_table || max_blocks == 0), "q8_dequantize_shape_unsupported:null_pointer");
  const int64_t per16 = dtype == BPKV_F32 ? 4 : 8;
  BPKV_CHECK_ARG(aligned16(k_out) && aligned16(v_out) && out_stride_t % per16 == 0 && out_stride_h % per16 == 0,
                 "q8_dequantize_shape_unsupported:alignment");
  const int64_t per32 = 2 * per16;
  const int wide = reinterpret_cast<uintptr_t>(k_out) % 32 == 0 && reinterpret_cast<uintptr_t>(v_out) % 32 == 0 &&
                   out_stride_t % per32 == 0 && out_stride_h % per32 == 0;
  ReadParams p{static_cast<const uint8_t*>(k_codes), static_cast<const uint8_t*>(v_codes), k_scales, v_scales, block_table,
               cu_seqlens, starts, k_out, v_out, batch, total, num_kv_heads, max_blocks, num_pages,
               block_tokens(total, num_kv_heads * (head_dim / 16)), wide, page_stride,
               scale_stride, bt_stride_b, out_stride_t, out_stride_h};
  const unsigned grid = static_cast<unsigned>((total + p.tokens - 1) / p.tokens);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define BPKV_READ(T)                                                        \
  do {                                                                      \
    if (head_dim == 64) q8_read_kernel<T, 64><<<grid, 256, 0, st>>>(p);     \
    else if (head_dim == 128) q8_read_kernel<T, 128><<<grid, 256, 0, st>>>(p); \
    else q8_read_kernel<T, 256><<<grid, 256, 0, st>>>(p);                   \
  } while (0)
  if (dtype == BPKV_F32) BPKV_READ(float);
  else if (dtype == BPKV_F16) BPKV_READ(__half);
  else BPKV_READ(__nv_bfloat16);
#undef BPKV_READ
  BPKV_RETURN_LAUNCH("q8_dequantize_launch");
}
