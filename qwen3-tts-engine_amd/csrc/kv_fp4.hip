// The 4-bit K/V pool's write and read (gfx950).  The row format is fp4_common.h's.
//
// Both are one pass over their bytes, which HBM bounds: a write reads 512 and writes 136 bytes a row pair, a read the reverse.  A wave takes
// 8 tokens of one KV head, 8 lanes a row, and a lane 8 dims of each of the row's halves, so that each load and store of bf16 takes whole
// lines; four lanes share a block's exponent.  The bf16 side passes once and is larger than the caches where time counts: non-temporal.
// 108800 tokens x 8 heads, written and read back: 266 us with 16 dims in a row a lane (a line in two halves by two instructions) and
// cached, 220 so and cached but for the write's loads, 191 so (5.3 TB/s); 35200 tokens read 47.3, 38.2, 28.2 us (6.5 TB/s).
#include "fp4_common.h"
#include "../../include/q3attn.h"

namespace q3a {
namespace {

constexpr int kThreads = 256;

struct WriteArgs {
  const uint16_t *k, *v;
  int64_t k_st, k_sh, v_st, v_sh;
  const int64_t* slots;
  uint8_t *kc, *vc;
  int64_t sp, st, sh;
  uint8_t *ks, *vs;
  int64_t ss_p, ss_h;
  int64_t num_slots;
  int64_t tokens;
  Divisor page_size, hkv;
};

// Where a slot's row and its first exponent byte lie.
struct Where {
  int64_t at, sat;
};
template <class Args>
__device__ __forceinline__ Where where_is(const Args& a, int64_t slot, int h) {
  int64_t page, off;
  if (a.num_slots < (int64_t)1 << 31) {
    const uint32_t i = (uint32_t)slot, q = divide(i, a.page_size);
    page = q;
    off = i - q * a.page_size.d;
  } else {
    page = slot / a.page_size.d;
    off = slot - page * a.page_size.d;
  }
  return {page * a.sp + off * a.st + h * a.sh, page * a.ss_p + h * a.ss_h + off};
}

// a, b: the lane's 8 dims of each half of a row.
__device__ __forceinline__ void write_row(const uint4 a, const uint4 b, bool live, uint8_t* dst, uint8_t* dscale, int sub,
                                          uint32_t page_size) {
  const uint4 x[2] = {a, b};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    const uint32_t s = fp4_scale_byte(dpp_max_u32<kDppXor2>(dpp_max_u32<kDppXor1>(halves_max(bf16_any_amax_pair(w)))));
    const uint32_t c = fp4_codes8(w[0], w[1], w[2], w[3], s);
    if (live) {
      *reinterpret_cast<uint32_t*>(dst + 32 * i + 4 * sub) = c;
      if ((sub & 3) == 0) dscale[(2 * i + (sub >> 2)) * page_size] = (uint8_t)s;
    }
  }
}

__device__ __forceinline__ uint4 ld16_nt(const void* p) {
  return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p)));
}

__global__ __launch_bounds__(kThreads) void fp4_write_kernel(const WriteArgs a) {
  const int lane = threadIdx.x & 63, sub = lane & 7;
  const uint32_t unit = blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t group = divide(unit, a.hkv);
  const int h = (int)(unit - group * a.hkv.d);
  const int64_t first = 8 * (int64_t)group, t = min(first + (lane >> 3), a.tokens - 1);
  if (first >= a.tokens) return;
  const int64_t slot = a.slots[t];
  const uint16_t* kp = a.k + t * a.k_st + h * a.k_sh + 8 * sub;
  const uint16_t* vp = a.v + t * a.v_st + h * a.v_sh + 8 * sub;
  const uint4 k0 = ld16_nt(kp), k1 = ld16_nt(kp + 64), v0 = ld16_nt(vp), v1 = ld16_nt(vp + 64);
  const bool live = first + (lane >> 3) < a.tokens && slot >= 0 && slot < a.num_slots;
  const Where p = where_is(a, live ? slot : 0, h);
  write_row(k0, k1, live, a.kc + p.at, a.ks + p.sat, sub, a.page_size.d);
  write_row(v0, v1, live, a.vc + p.at, a.vs + p.sat, sub, a.page_size.d);
}

struct ReadArgs {
  const uint8_t *kc, *vc;
  int64_t sp, st, sh;
  const uint8_t *ks, *vs;
  int64_t ss_p, ss_h;
  const int64_t* slots;
  int64_t num_slots;
  uint16_t *k, *v;
  int64_t k_st, k_sh, v_st, v_sh;
  Divisor page_size, hkv;
  int64_t tokens;
};

// c, s: the codes and the exponent bytes of the lane's 8 dims of each half.
__device__ __forceinline__ void read_row(const uint32_t (&c)[2], const uint32_t (&s)[2], uint16_t* dst) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float f = fp8_scale(s[i]);
    st16_nt(dst + 64 * i, make_uint4(fp4_pair<0>(c[i], f), fp4_pair<1>(c[i], f), fp4_pair<2>(c[i], f), fp4_pair<3>(c[i], f)));
  }
}

__global__ __launch_bounds__(kThreads) void fp4_read_kernel(const ReadArgs a) {
  const int sub = threadIdx.x & 7;
  const uint32_t unit = blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t group = divide(unit, a.hkv);
  const int h = (int)(unit - group * a.hkv.d);
  const int64_t t = 8 * (int64_t)group + ((threadIdx.x & 63) >> 3);
  if (t >= a.tokens) return;
  const int64_t slot = a.slots[t];
  uint32_t kc[2] = {0u, 0u}, vc[2] = {0u, 0u}, ks[2] = {127u, 127u}, vs[2] = {127u, 127u};
  if (slot >= 0 && slot < a.num_slots) {
    const Where p = where_is(a, slot, h);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t in = p.sat + (2 * i + (sub >> 2)) * (int64_t)a.page_size.d;
      kc[i] = *reinterpret_cast<const uint32_t*>(a.kc + p.at + 32 * i + 4 * sub);
      vc[i] = *reinterpret_cast<const uint32_t*>(a.vc + p.at + 32 * i + 4 * sub);
      ks[i] = a.ks[in];
      vs[i] = a.vs[in];
    }
  }
  read_row(kc, ks, a.k + t * a.k_st + h * a.k_sh + 8 * sub);
  read_row(vc, vs, a.v + t * a.v_st + h * a.v_sh + 8 * sub);
}

}  // namespace

int check_fp4_pool(const char* who, const void* kc, const void* vc, int64_t sp, int64_t st, int64_t sh, const void* ks,
                   const void* vs, int64_t ss_p, int64_t ss_h, int num_pages, int page_size, int hkv) {
  if (kc == nullptr || vc == nullptr || ks == nullptr || vs == nullptr)
    return fail(Q3A_EINVAL, "%s: null pool or scale pointer", who);
  if (num_pages < 0 || page_size < 16 || page_size % 16 != 0 || page_size > (1 << 26))
    return fail(Q3A_EINVAL, "%s: page_size %d must be a multiple of 16 up to 2^26 and num_pages %d >= 0", who, page_size, num_pages);
  if (hkv < 1) return fail(Q3A_EINVAL, "%s: num_kv_heads %d must be positive", who, hkv);
  // the stride of a dimension of one element is not used
  if (hkv == 1) sh = ss_h = 0;
  if (num_pages == 1) sp = ss_p = 0;
  if ((((uintptr_t)kc | (uintptr_t)vc) & 15) != 0 || ((sp | st | sh) & 15) != 0 || sp < 0 || sh < 0 || st < kFp4Row ||
      st > (1 << 26))
    return fail(Q3A_EINVAL, "%s: pool pointers and strides must be 16-byte aligned, strides >= 0, token stride in [64, 2^26] bytes",
                who);
  if ((((uintptr_t)ks | (uintptr_t)vs) & 3) != 0 || ((ss_p | ss_h) & 3) != 0 || ss_p < 0 || ss_h < 0)
    return fail(Q3A_EINVAL, "%s: scale pointers and strides must be multiples of 4 and strides >= 0", who);
  return Q3A_OK;
}

}  // namespace q3a

using namespace q3a;

extern "C" int q3a_paged_write_fp4(const void* k, int64_t k_stride_t, int64_t k_stride_h, const void* v, int64_t v_stride_t,
                                   int64_t v_stride_h, const int64_t* slots, void* k_cache, void* v_cache,
                                   int64_t kv_stride_page, int64_t kv_stride_tok, int64_t kv_stride_head, void* k_scale,
                                   void* v_scale, int64_t scale_stride_page, int64_t scale_stride_head, int num_pages,
                                   int page_size, int64_t num_tokens, int num_kv_heads, int head_dim, void* stream) {
  const char* who = "q3a_paged_write_fp4";
  int rc = check_pool_rows(who, k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h, slots, num_tokens, num_kv_heads, head_dim);
  if (rc != Q3A_OK) return rc;
  rc = check_fp4_pool(who, k_cache, v_cache, kv_stride_page, kv_stride_tok, kv_stride_head, k_scale, v_scale,
                      scale_stride_page, scale_stride_head, num_pages, page_size, num_kv_heads);
  if (rc != Q3A_OK) return rc;
  if (num_tokens == 0) return Q3A_OK;
  WriteArgs a;
  a.k = (const uint16_t*)k;
  a.v = (const uint16_t*)v;
  a.k_st = k_stride_t;
  a.k_sh = k_stride_h;
  a.v_st = v_stride_t;
  a.v_sh = v_stride_h;
  a.slots = slots;
  a.kc = (uint8_t*)k_cache;
  a.vc = (uint8_t*)v_cache;
  a.sp = kv_stride_page;
  a.st = kv_stride_tok;
  a.sh = kv_stride_head;
  a.ks = (uint8_t*)k_scale;
  a.vs = (uint8_t*)v_scale;
  a.ss_p = scale_stride_page;
  a.ss_h = scale_stride_head;
  a.num_slots = (int64_t)num_pages * page_size;
  a.tokens = num_tokens;
  a.page_size = divisor((uint32_t)page_size);
  a.hkv = divisor((uint32_t)num_kv_heads);
  const int64_t waves = (num_tokens + 7) / 8 * num_kv_heads, blocks = (waves + kThreads / 64 - 1) / (kThreads / 64);
  hipLaunchKernelGGL(fp4_write_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, (hipStream_t)stream, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? Q3A_OK : fail(Q3A_ELAUNCH, "%s: %s", who, hipGetErrorString(e));
}

extern "C" int q3a_paged_read_fp4(const void* k_cache, const void* v_cache, int64_t kv_stride_page, int64_t kv_stride_tok,
                                  int64_t kv_stride_head, const void* k_scale, const void* v_scale,
                                  int64_t scale_stride_page, int64_t scale_stride_head, int num_pages, int page_size,
                                  const int64_t* slots, void* k, int64_t k_stride_t, int64_t k_stride_h, void* v,
                                  int64_t v_stride_t, int64_t v_stride_h, int64_t num_tokens, int num_kv_heads,
                                  int head_dim, void* stream) {
  const char* who = "q3a_paged_read_fp4";
  int rc = check_pool_rows(who, k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h, slots, num_tokens, num_kv_heads, head_dim);
  if (rc != Q3A_OK) return rc;
  rc = check_fp4_pool(who, k_cache, v_cache, kv_stride_page, kv_stride_tok, kv_stride_head, k_scale, v_scale,
                      scale_stride_page, scale_stride_head, num_pages, page_size, num_kv_heads);
  if (rc != Q3A_OK) return rc;
  if (num_tokens == 0) return Q3A_OK;
  ReadArgs a;
  a.kc = (const uint8_t*)k_cache;
  a.vc = (const uint8_t*)v_cache;
  a.sp = kv_stride_page;
  a.st = kv_stride_tok;
  a.sh = kv_stride_head;
  a.ks = (const uint8_t*)k_scale;
  a.vs = (const uint8_t*)v_scale;
  a.ss_p = scale_stride_page;
  a.ss_h = scale_stride_head;
  a.slots = slots;
  a.num_slots = (int64_t)num_pages * page_size;
  a.k = (uint16_t*)k;
  a.v = (uint16_t*)v;
  a.k_st = k_stride_t;
  a.k_sh = k_stride_h;
  a.v_st = v_stride_t;
  a.v_sh = v_stride_h;
  a.page_size = divisor((uint32_t)page_size);
  a.hkv = divisor((uint32_t)num_kv_heads);
  a.tokens = num_tokens;
  const int64_t waves = (num_tokens + 7) / 8 * num_kv_heads, blocks = (waves + kThreads / 64 - 1) / (kThreads / 64);
  hipLaunchKernelGGL(fp4_read_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, (hipStream_t)stream, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? Q3A_OK : fail(Q3A_ELAUNCH, "%s: %s", who, hipGetErrorString(e));
}
