// Writing rows of K and V into 8-bit pages, and reading ranges of them back.
//
// Both are bound by HBM: a row is read once and written once, with a handful of
// instructions per element.  head_dim / 8 (write) or head_dim / 16 (read back)
// neighbouring threads share a row, so a warp touches whole 128-byte lines, and
// every thread handles the K and the V row of its (token, head), which keeps two
// independent loads in flight.
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
  int batch, total, Hkv, max_blocks, num_pages;
  int64_t k_st, k_sh, v_st, v_sh, page_stride, scale_stride, bt_sb;
};

// Eight consecutive elements as floats.
__device__ __forceinline__ void load8(const float* p, float* x) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, float* x) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = Elem<T>::to_f(e[i]);
}

template <int G>  // G neighbouring lanes share a row
__device__ __forceinline__ void store_row(const float* x, uint8_t* codes, uint8_t* scale, int lane_in_row, bool live) {
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = max(amax, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
  for (int o = 1; o < G; o <<= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  const int byte = q8::scale_byte(amax);
  uint2 c;
  if (byte == q8::kNanByte) {
    c = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
  } else {
    // 2^-e, e = byte - 127 in [-127, 119]: a normal number, so the products are exact (or far
    // below the smallest code)
    const float inv = __uint_as_float(static_cast<uint32_t>(254 - byte) << 23);
    c.x = q8::to_e4m3x2(x[0] * inv, x[1] * inv) | q8::to_e4m3x2(x[2] * inv, x[3] * inv) << 16;
    c.y = q8::to_e4m3x2(x[4] * inv, x[5] * inv) | q8::to_e4m3x2(x[6] * inv, x[7] * inv) << 16;
  }
  if (live) {
    *reinterpret_cast<uint2*>(codes + lane_in_row * 8) = c;
    if (lane_in_row == 0) *scale = static_cast<uint8_t>(byte);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(256) q8_append_kernel(AppendParams p) {
  constexpr int G = D / 8;
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / G;
  const int lr = threadIdx.x % G;
  const int64_t rows = static_cast<int64_t>(p.total) * p.Hkv;
  const int i = row < rows ? static_cast<int>(row / p.Hkv) : 0;
  const int h = row < rows ? static_cast<int>(row % p.Hkv) : 0;
  // the token's slot: position len - n_new + (index in the request)
  int page = -1, slot = 0;
  if (row < rows) {
    const int b = p.cu_q == nullptr ? i : q8::request_of(p.cu_q, p.batch, i);
    if (b >= 0) {
      const int pos = __ldg(p.seqlens_k + b) - (p.cu_q == nullptr ? 1 : __ldg(p.cu_q + b + 1) - i);
      if (pos >= 0) page = q8::page_of(p.bt + static_cast<int64_t>(b) * p.bt_sb, pos / kPage, p.max_blocks, p.num_pages);
      slot = pos & (kPage - 1);
    }
  }
  const bool live = page >= 0;  // the lanes of a row agree; the others only take part in the shuffles
  float k[8] = {}, v[8] = {};
  if (live) {
    load8(static_cast<const T*>(p.k_new) + i * p.k_st + h * p.k_sh + lr * 8, k);
    load8(static_cast<const T*>(p.v_new) + i * p.v_st + h * p.v_sh + lr * 8, v);
  }
  const int64_t off = live ? page * p.page_stride + (static_cast<int64_t>(slot) * p.Hkv + h) * D : 0;
  const int64_t soff = live ? page * p.scale_stride + h * kPage + slot : 0;
  store_row<G>(k, p.kc + off, p.ks + soff, lr, live);
  store_row<G>(v, p.vc + off, p.vs + soff, lr, live);
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
  int batch, total, Hkv, max_blocks, num_pages;
  int64_t page_stride, scale_stride, bt_sb, o_st, o_sh;
};

// Sixteen values in one go.
__device__ __forceinline__ void store16(float* p, const float* x) {
#pragma unroll
  for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
}
template <typename T>
__device__ __forceinline__ void store16(T* p, const float* x) {
#pragma unroll
  for (int i = 0; i < 16; i += 8)
    *reinterpret_cast<uint4*>(p + i) = make_uint4(pack2<T>(x[i], x[i + 1]), pack2<T>(x[i + 2], x[i + 3]),
                                                  pack2<T>(x[i + 4], x[i + 5]), pack2<T>(x[i + 6], x[i + 7]));
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
  constexpr int G = D / 16;
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / G;
  const int lr = threadIdx.x % G;
  if (row >= static_cast<int64_t>(p.total) * p.Hkv) return;
  const int i = static_cast<int>(row / p.Hkv), h = static_cast<int>(row % p.Hkv);
  const int b = q8::request_of(p.cu, p.batch, i);
  if (b < 0) return;  // rows behind the last sequence stay as they were
  const int pos = (p.starts == nullptr ? 0 : __ldg(p.starts + b)) + i - __ldg(p.cu + b);
  const int page =
      pos < 0 ? -1 : q8::page_of(p.bt + static_cast<int64_t>(b) * p.bt_sb, pos / kPage, p.max_blocks, p.num_pages);
  uint4 kq = make_uint4(0, 0, 0, 0), vq = kq;  // a token without a page reads as zeros
  float sk = 0.f, sv = 0.f;
  if (page >= 0) {
    const int slot = pos & (kPage - 1);
    const int64_t off = page * p.page_stride + (static_cast<int64_t>(slot) * p.Hkv + h) * D + lr * 16;
    const int64_t soff = page * p.scale_stride + h * kPage + slot;
    kq = __ldg(reinterpret_cast<const uint4*>(p.kc + off));
    vq = __ldg(reinterpret_cast<const uint4*>(p.vc + off));
    sk = q8::scale_of(__ldg(p.ks + soff));
    sv = q8::scale_of(__ldg(p.vs + soff));
  }
  float x[16];
  const int64_t o = i * p.o_st + h * p.o_sh + lr * 16;
  values16(kq, sk, x);
  store16(static_cast<T*>(p.k_out) + o, x);
  values16(vq, sv, x);
  store16(static_cast<T*>(p.v_out) + o, x);
}

int check_pages(const char* what, const void* kc, const void* vc, const void* ks, const void* vs, int Hkv, int D,
                int num_pages, int64_t page_stride, int64_t scale_stride) {
  BPKV_CHECK_ARG(Hkv > 0 && num_pages >= 0, "%s_shape_unsupported:empty", what);
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
                 k_stride_t, k_stride_h, v_stride_t, v_stride_h, page_stride, scale_stride, bt_stride_b};
  const int64_t blocks = (static_cast<int64_t>(total_q) * num_kv_heads * (head_dim / 8) + 255) / 256;
  BPKV_CHECK_ARG(blocks < (1LL << 31), "q8_append_shape_unsupported:total_%d", total_q);
  const unsigned grid = static_cast<unsigned>(blocks);
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
  ReadParams p{static_cast<const uint8_t*>(k_codes), static_cast<const uint8_t*>(v_codes), k_scales, v_scales, block_table,
               cu_seqlens, starts, k_out, v_out, batch, total, num_kv_heads, max_blocks, num_pages, page_stride,
               scale_stride, bt_stride_b, out_stride_t, out_stride_h};
  const int64_t blocks = (static_cast<int64_t>(total) * num_kv_heads * (head_dim / 16) + 255) / 256;
  BPKV_CHECK_ARG(blocks < (1LL << 31), "q8_dequantize_shape_unsupported:total_%d", total);
  const unsigned grid = static_cast<unsigned>(blocks);
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
