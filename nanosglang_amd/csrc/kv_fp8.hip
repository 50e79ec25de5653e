// Writes into and reads from the 8-bit KV pool (format: fp8_kv.hpp).
//
// nsg_kv_write_fp8 / nsg_rope_kv_write_fp8 are the 8-bit counterparts of
// nsg_kv_write / nsg_rope_kv_write (the scatter at
// nano_sglang/model/causal_lm.py:335-338, after apply_rope at :300-301 for the
// second), nsg_kv_read_fp8 the gather of such rows as bf16.  All three move
// each byte once and are bound by memory for long inputs, by the launch for a
// decode step's.
#include <algorithm>

#include "fp8_kv.hpp"

namespace nsg {
namespace {

constexpr int kThreads = 256;

// A lane holds 16 values of a head's row: chunk l of each half of the row, so
// that it has both members of 8 rotary pairs.
struct Half16 {
  fp8_u32x4 a, b;
};

__device__ __forceinline__ uint32_t abs_bits_max(uint32_t m, uint32_t packed) {
  const uint32_t lo = packed << 16 & 0x7fff0000u, hi = packed & 0x7fff0000u;
  return max(m, max(lo, hi));
}

__device__ __forceinline__ Half16 load16(const uint16_t* row, int l, int half) {
  return {*reinterpret_cast<const fp8_u32x4*>(row + 8 * l),
          *reinterpret_cast<const fp8_u32x4*>(row + half + 8 * l)};
}

// The row (D / 16 neighbouring lanes) quantised into its slot.
template <int D>
__device__ __forceinline__ void store_row(const Half16& x, int l, bool is_v, uint8_t* codes,
                                          uint8_t* scale) {
  constexpr int LPR = D / 16;
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) m = abs_bits_max(abs_bits_max(m, x.a[i]), x.b[i]);
#pragma unroll
  for (int o = 1; o < LPR; o <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
  const uint32_t e = e8m0_of(m);
  const float s = e8m0_scale(e == kE8M0NaN ? 127 : e);
  fp8_u32x2 ca = {to_fp8x4(x.a[0], x.a[1], s), to_fp8x4(x.a[2], x.a[3], s)};
  fp8_u32x2 cb = {to_fp8x4(x.b[0], x.b[1], s), to_fp8x4(x.b[2], x.b[3], s)};
  if (e == kE8M0NaN) ca = cb = is_v ? fp8_u32x2{0u, 0u} : fp8_u32x2{0x7f7f7f7fu, 0x7f7f7f7fu};
  *reinterpret_cast<fp8_u32x2*>(codes + 8 * l) = ca;
  *reinterpret_cast<fp8_u32x2*>(codes + D / 2 + 8 * l) = cb;
  if (l == 0) *scale = (uint8_t)e;
}

struct WriteParams {
  const uint16_t *k, *v;
  int64_t k_stride, v_stride;  // elements between tokens
  const int64_t* slots;
  int num_tokens, Hkv, log2P;
  int64_t num_slots;
  uint8_t *kc, *vc, *scale;
};

// One group of D / 16 lanes per (token, K or V, head) row.
template <int D>
__global__ __launch_bounds__(kThreads) void kv_write_fp8_kernel(WriteParams p) {
  constexpr int LPR = D / 16;
  const int64_t gid = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int l = (int)(gid % LPR);
  const int64_t row = gid / LPR;
  const int rows = 2 * p.Hkv;
  const int64_t t = row / rows;
  if (t >= p.num_tokens) return;  // whole groups of lanes: the shuffles stay within one
  const int r = (int)(row - t * rows);
  const bool is_v = r >= p.Hkv;
  const int h = is_v ? r - p.Hkv : r;
  const int64_t slot = p.slots[t];
  if (slot < 0 || slot >= p.num_slots) return;
  const uint16_t* src = is_v ? p.v + t * p.v_stride : p.k + t * p.k_stride;
  const Half16 x = load16(src + (int64_t)h * D, l, D / 2);
  store_row<D>(x, l, is_v, (is_v ? p.vc : p.kc) + (slot * p.Hkv + h) * D,
               p.scale + scale_at(slot, p.log2P, p.Hkv, h, is_v));
}

struct RopeParams {
  const uint16_t* qkv;
  int64_t stride;
  const int64_t* positions;
  const float *cos_t, *sin_t;
  int max_pos;
  const int64_t* slots;
  int num_tokens, Hq, Hkv, log2P, heads_per_thread;
  int64_t num_slots;
  uint16_t* q_out;
  uint8_t *kc, *vc, *scale;
  int* flags;
};

__device__ __forceinline__ float bf16_lo(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

// Two rotary pairs packed: y1 = bf16(bf16(x1 c) + bf16(-x2 s)), y2 = bf16(bf16(
// x2 c) + bf16(x1 s)) with c, s rounded to bf16 -- the roundings of
// nsg_rope_kv_write (the arithmetic of bf16 tensors in
// nano_sglang/model/causal_lm.py:181-206), so that q and the K rows before
// quantisation are the same bits whichever pool is written.
__device__ __forceinline__ void rotate(uint32_t& x1, uint32_t& x2, uint32_t c, uint32_t s) {
  const uint32_t a = pack_bf16x2(bf16_lo(x1) * bf16_lo(c), bf16_hi(x1) * bf16_hi(c));
  const uint32_t b = pack_bf16x2(-bf16_lo(x2) * bf16_lo(s), -bf16_hi(x2) * bf16_hi(s));
  const uint32_t d = pack_bf16x2(bf16_lo(x2) * bf16_lo(c), bf16_hi(x2) * bf16_hi(c));
  const uint32_t e = pack_bf16x2(bf16_lo(x1) * bf16_lo(s), bf16_hi(x1) * bf16_hi(s));
  x1 = pack_bf16x2(bf16_lo(a) + bf16_lo(b), bf16_hi(a) + bf16_hi(b));
  x2 = pack_bf16x2(bf16_lo(d) + bf16_lo(e), bf16_hi(d) + bf16_hi(e));
}

// A group of D / 16 lanes takes heads_per_thread consecutive heads (blockIdx.y
// picks which) of one token: the token's 8 cosines and sines per lane are
// loaded once for them.
template <int D>
__global__ __launch_bounds__(kThreads) void rope_kv_write_fp8_kernel(RopeParams p) {
  constexpr int LPR = D / 16;
  const int64_t gid = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int l = (int)(gid % LPR);
  const int64_t t = gid / LPR;
  if (t >= p.num_tokens) return;
  const int heads = p.Hq + 2 * p.Hkv;
  const int h0 = (int)blockIdx.y * p.heads_per_thread;
  const int h1 = min(h0 + p.heads_per_thread, heads);
  const uint16_t* src = p.qkv + t * p.stride;
  // (the first head's values travel with the position, not after it)
  Half16 next = load16(src + (int64_t)h0 * D, l, D / 2);
  const int64_t pos = p.positions[t];
  const bool pos_ok = pos >= 0 && pos < p.max_pos;
  const int64_t slot = p.slots ? p.slots[t] : -1;
  const bool slot_ok = slot >= 0 && slot < p.num_slots;
  if (l == 0 && blockIdx.y == 0 && (!pos_ok || slot >= p.num_slots) && p.flags)
    atomicOr(p.flags, 1);
  uint32_t c[4] = {0, 0, 0, 0}, s[4] = {0, 0, 0, 0};
  if (pos_ok && h0 < p.Hq + p.Hkv) {
    const floatx4* ct = reinterpret_cast<const floatx4*>(p.cos_t + pos * (D / 2) + 8 * l);
    const floatx4* st = reinterpret_cast<const floatx4*>(p.sin_t + pos * (D / 2) + 8 * l);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const floatx4 cv = ct[i], sv = st[i];
      c[2 * i] = pack_bf16x2(cv[0], cv[1]);
      c[2 * i + 1] = pack_bf16x2(cv[2], cv[3]);
      s[2 * i] = pack_bf16x2(sv[0], sv[1]);
      s[2 * i + 1] = pack_bf16x2(sv[2], sv[3]);
    }
  }
  for (int hh = h0; hh < h1; ++hh) {
    if (hh >= p.Hq && !slot_ok) break;
    Half16 x = next;
    if (hh + 1 < h1) next = load16(src + (int64_t)(hh + 1) * D, l, D / 2);
    if (hh < p.Hq + p.Hkv) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t a = x.a[i], b = x.b[i];
        rotate(a, b, c[i], s[i]);
        x.a[i] = a;
        x.b[i] = b;
      }
    }
    if (hh < p.Hq) {
      uint16_t* qo = p.q_out + (t * p.Hq + hh) * D;
      *reinterpret_cast<fp8_u32x4*>(qo + 8 * l) = x.a;
      *reinterpret_cast<fp8_u32x4*>(qo + D / 2 + 8 * l) = x.b;
    } else {
      const bool is_v = hh >= p.Hq + p.Hkv;
      const int h = hh - p.Hq - (is_v ? p.Hkv : 0);
      store_row<D>(x, l, is_v, (is_v ? p.vc : p.kc) + (slot * p.Hkv + h) * D,
                   p.scale + scale_at(slot, p.log2P, p.Hkv, h, is_v));
    }
  }
}

struct ReadParams {
  const int64_t* slots;
  int num_tokens, Hkv, log2P;
  int64_t num_slots;
  const uint8_t *kc, *vc, *scale;
  uint16_t *k, *v;
};

// One lane per 16 codes of a (token, K or V, head) row.
template <int D>
__global__ __launch_bounds__(kThreads) void kv_read_fp8_kernel(ReadParams p) {
  constexpr int LPR = D / 16;
  const int64_t gid = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int l = (int)(gid % LPR);
  const int64_t row = gid / LPR;
  const int rows = 2 * p.Hkv;
  const int64_t t = row / rows;
  if (t >= p.num_tokens) return;
  const int r = (int)(row - t * rows);
  const bool is_v = r >= p.Hkv;
  const int h = is_v ? r - p.Hkv : r;
  const int64_t slot = p.slots[t];
  fp8_u32x4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
  if (slot >= 0 && slot < p.num_slots) {
    const fp8_u32x4 w = *reinterpret_cast<const fp8_u32x4*>(
        (is_v ? p.vc : p.kc) + (slot * p.Hkv + h) * D + 16 * l);
    const float s = e8m0_scale(p.scale[scale_at(slot, p.log2P, p.Hkv, h, is_v)]);
    const fp8_u32x2 a = from_fp8x4(w[0], s), b = from_fp8x4(w[1], s), c = from_fp8x4(w[2], s),
                    d = from_fp8x4(w[3], s);
    lo = fp8_u32x4{a[0], a[1], b[0], b[1]};
    hi = fp8_u32x4{c[0], c[1], d[0], d[1]};
  }
  uint16_t* dst = (is_v ? p.v : p.k) + (t * p.Hkv + h) * D + 16 * l;
  *reinterpret_cast<fp8_u32x4*>(dst) = lo;
  *reinterpret_cast<fp8_u32x4*>(dst + 8) = hi;
}

// Checks shared by the three entry points; log2P out.
int32_t check_pool(const void* k_cache, const void* v_cache, const void* kv_scale,
                   int32_t num_kv_heads, int32_t head_dim, int32_t page_size, int64_t num_slots,
                   int* log2P) {
  NSG_CHECK_ARG(k_cache && v_cache && kv_scale, "null pointer argument");
  NSG_CHECK_ARG(num_kv_heads > 0, "num_kv_heads %d", num_kv_heads);
  if (head_dim != 64 && head_dim != 128) {
    set_error("head_dim %d not supported (64 or 128)", head_dim);
    return NSG_ERR_UNSUPPORTED;
  }
  NSG_CHECK_ARG(page_size > 0 && (page_size & (page_size - 1)) == 0,
                "page_size %d must be a power of two", page_size);
  NSG_CHECK_ARG(num_slots >= 0 && num_slots % page_size == 0,
                "num_slots %lld must be whole pages of %d", (long long)num_slots, page_size);
  NSG_CHECK_ARG(((uintptr_t)k_cache | (uintptr_t)v_cache) % 16 == 0,
                "caches must be 16-byte aligned");
  *log2P = __builtin_ctz((unsigned)page_size);
  return NSG_OK;
}

// Workgroups of kThreads lanes for n lanes, or an error past the grid's limit.
int32_t grid_of(int64_t lanes, unsigned* blocks) {
  const int64_t n = (lanes + kThreads - 1) / kThreads;
  NSG_CHECK_ARG(n <= 0x7fffffff / kThreads, "too many rows for one launch");
  *blocks = (unsigned)n;
  return NSG_OK;
}

}  // namespace
}  // namespace nsg

using namespace nsg;

extern "C" int32_t nsg_kv_write_fp8(const void* k, int64_t k_token_stride, const void* v,
                                    int64_t v_token_stride, const int64_t* slots,
                                    int32_t num_tokens, void* k_cache, void* v_cache,
                                    void* kv_scale, int32_t num_kv_heads, int32_t head_dim,
                                    int32_t page_size, int64_t num_slots, nsg_stream_t stream) {
  NSG_CHECK_ARG(num_tokens >= 0, "num_tokens %d < 0", num_tokens);
  if (num_tokens == 0) {
    clear_error();
    return NSG_OK;
  }
  NSG_CHECK_ARG(k && v && slots, "null pointer argument");
  WriteParams p{};
  if (int32_t rc = check_pool(k_cache, v_cache, kv_scale, num_kv_heads, head_dim, page_size,
                              num_slots, &p.log2P))
    return rc;
  const int64_t row = (int64_t)num_kv_heads * head_dim;
  NSG_CHECK_ARG(k_token_stride >= row && k_token_stride % 8 == 0 && v_token_stride >= row &&
                    v_token_stride % 8 == 0,
                "token strides %lld / %lld must be >= %lld and multiples of 8",
                (long long)k_token_stride, (long long)v_token_stride, (long long)row);
  NSG_CHECK_ARG(((uintptr_t)k | (uintptr_t)v) % 16 == 0, "K/V sources must be 16-byte aligned");
  unsigned blocks = 0;
  if (int32_t rc = grid_of((int64_t)num_tokens * 2 * num_kv_heads * (head_dim / 16), &blocks))
    return rc;
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.k_stride = k_token_stride;
  p.v_stride = v_token_stride;
  p.slots = slots;
  p.num_tokens = num_tokens;
  p.Hkv = num_kv_heads;
  p.num_slots = num_slots;
  p.kc = static_cast<uint8_t*>(k_cache);
  p.vc = static_cast<uint8_t*>(v_cache);
  p.scale = static_cast<uint8_t*>(kv_scale);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim == 64)
    hipLaunchKernelGGL(kv_write_fp8_kernel<64>, dim3(blocks), dim3(kThreads), 0, s, p);
  else
    hipLaunchKernelGGL(kv_write_fp8_kernel<128>, dim3(blocks), dim3(kThreads), 0, s, p);
  return launch_status("kv_write_fp8_kernel");
}

extern "C" int32_t nsg_rope_kv_write_fp8(const void* qkv, int64_t qkv_token_stride,
                                         const int64_t* positions, const float* cos_table,
                                         const float* sin_table, int32_t max_position,
                                         const int64_t* slots, int32_t num_tokens,
                                         int32_t num_qo_heads, int32_t num_kv_heads,
                                         int32_t head_dim, int32_t page_size, void* q_out,
                                         void* k_cache, void* v_cache, void* kv_scale,
                                         int64_t num_slots, int32_t* flags,
                                         nsg_stream_t stream) {
  NSG_CHECK_ARG(num_tokens >= 0, "num_tokens %d < 0", num_tokens);
  if (num_tokens == 0) {
    clear_error();
    return NSG_OK;
  }
  NSG_CHECK_ARG(qkv && positions && cos_table && sin_table && q_out, "null pointer argument");
  NSG_CHECK_ARG(num_qo_heads > 0 && max_position > 0, "num_qo_heads %d, max_position %d",
                num_qo_heads, max_position);
  RopeParams p{};
  if (slots) {
    if (int32_t rc = check_pool(k_cache, v_cache, kv_scale, num_kv_heads, head_dim, page_size,
                                num_slots, &p.log2P))
      return rc;
  } else {
    NSG_CHECK_ARG(num_kv_heads > 0, "num_kv_heads %d", num_kv_heads);
    if (head_dim != 64 && head_dim != 128) {
      set_error("head_dim %d not supported (64 or 128)", head_dim);
      return NSG_ERR_UNSUPPORTED;
    }
  }
  const int heads = num_qo_heads + 2 * num_kv_heads;
  NSG_CHECK_ARG(qkv_token_stride >= (int64_t)heads * head_dim && qkv_token_stride % 8 == 0,
                "qkv_token_stride %lld must be >= %lld and a multiple of 8",
                (long long)qkv_token_stride, (long long)heads * head_dim);
  NSG_CHECK_ARG(((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)cos_table | (uintptr_t)sin_table)
                        % 16 == 0,
                "qkv, q_out and the tables must be 16-byte aligned");
  // As many heads per thread, up to 12, as leave every CU its 2048 lanes: the
  // cosines and sines are then loaded that much less often, but few tokens
  // want every lane (16,384 tokens, 32 / 8 heads of 128: 1 / 4 / 12 heads 97 / 87 /
  // 81 us, 4.6 TB/s; 160 tokens, 14 / 2 heads of 64: 1 / 2 heads 3.2 / 3.9).
  const int64_t lanes = (int64_t)num_tokens * (head_dim / 16) * heads;
  p.heads_per_thread = (int)std::min<int64_t>(12, std::max<int64_t>(1, lanes / (256 * 2048)));
  unsigned blocks = 0;
  if (int32_t rc = grid_of((int64_t)num_tokens * (head_dim / 16), &blocks)) return rc;
  const unsigned chunks = (heads + p.heads_per_thread - 1) / p.heads_per_thread;
  NSG_CHECK_ARG(chunks <= 65535, "too many heads (%d)", heads);
  p.qkv = static_cast<const uint16_t*>(qkv);
  p.stride = qkv_token_stride;
  p.positions = positions;
  p.cos_t = cos_table;
  p.sin_t = sin_table;
  p.max_pos = max_position;
  p.slots = slots;
  p.num_tokens = num_tokens;
  p.Hq = num_qo_heads;
  p.Hkv = num_kv_heads;
  p.num_slots = num_slots;
  p.q_out = static_cast<uint16_t*>(q_out);
  p.kc = static_cast<uint8_t*>(k_cache);
  p.vc = static_cast<uint8_t*>(v_cache);
  p.scale = static_cast<uint8_t*>(kv_scale);
  p.flags = flags;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim == 64)
    hipLaunchKernelGGL(rope_kv_write_fp8_kernel<64>, dim3(blocks, chunks), dim3(kThreads), 0, s,
                       p);
  else
    hipLaunchKernelGGL(rope_kv_write_fp8_kernel<128>, dim3(blocks, chunks), dim3(kThreads), 0, s,
                       p);
  return launch_status("rope_kv_write_fp8_kernel");
}

extern "C" int32_t nsg_kv_read_fp8(const int64_t* slots, int32_t num_tokens, const void* k_cache,
                                   const void* v_cache, const void* kv_scale,
                                   int32_t num_kv_heads, int32_t head_dim, int32_t page_size,
                                   int64_t num_slots, void* k, void* v, nsg_stream_t stream) {
  NSG_CHECK_ARG(num_tokens >= 0, "num_tokens %d < 0", num_tokens);
  if (num_tokens == 0) {
    clear_error();
    return NSG_OK;
  }
  NSG_CHECK_ARG(slots && k && v, "null pointer argument");
  ReadParams p{};
  if (int32_t rc = check_pool(k_cache, v_cache, kv_scale, num_kv_heads, head_dim, page_size,
                              num_slots, &p.log2P))
    return rc;
  NSG_CHECK_ARG(((uintptr_t)k | (uintptr_t)v) % 16 == 0, "K/V outputs must be 16-byte aligned");
  unsigned blocks = 0;
  if (int32_t rc = grid_of((int64_t)num_tokens * 2 * num_kv_heads * (head_dim / 16), &blocks))
    return rc;
  p.slots = slots;
  p.num_tokens = num_tokens;
  p.Hkv = num_kv_heads;
  p.num_slots = num_slots;
  p.kc = static_cast<const uint8_t*>(k_cache);
  p.vc = static_cast<const uint8_t*>(v_cache);
  p.scale = static_cast<const uint8_t*>(kv_scale);
  p.k = static_cast<uint16_t*>(k);
  p.v = static_cast<uint16_t*>(v);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim == 64)
    hipLaunchKernelGGL(kv_read_fp8_kernel<64>, dim3(blocks), dim3(kThreads), 0, s, p);
  else
    hipLaunchKernelGGL(kv_read_fp8_kernel<128>, dim3(blocks), dim3(kThreads), 0, s, p);
  return launch_status("kv_read_fp8_kernel");
}
