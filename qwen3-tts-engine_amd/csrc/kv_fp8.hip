// The 8-bit K/V pool's write and read (gfx950).  The row format is fp8_common.h's.
//
// Both are one pass over their bytes, bound by HBM: a write reads 512 and writes 258 bytes a row pair (64 x 1700 tokens of 8
// heads in 133.7 us, 5.0 TB/s, as fast as a large copy), a read the reverse (32 x 1100 tokens in 47.7 us, 4.6 TB/s).  8 lanes
// share a row: 32 B of bf16 and 16 B of codes a lane, so a row of codes is one 128 B line, a row of bf16 two, and the row's
// maximum is 3 DPP steps.  Non-temporal loads changed nothing, non-temporal stores of what is read took 82 us instead of 47,
// several rows a lane were 2 to 12 % slower.
#include "fp8_common.h"
#include "../../include/q3attn.h"

namespace q3a {
namespace {

constexpr int kThreads = 256;
constexpr int kRowsPerBlock = kThreads / 8;

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

__device__ __forceinline__ void write_row(const uint4 a, const uint4 b, bool live, uint8_t* dst, uint8_t* dscale, int sub) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t top = halves_max(bf16_any_amax_pair(w));
  const bool rare = any_rare(top);
  if (rare) top = halves_max(bf16_amax_pair(w));
  top = dpp_max_u32<kDppXor1>(top);
  top = dpp_max_u32<kDppXor2>(top);
  top = dpp_max_u32<kDppHalfMirror>(top);
  const uint32_t s = fp8_scale_byte(top);
  const float scale = fp8_scale(s);
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = fp8_finite_codes4(w[2 * i], w[2 * i + 1], scale);
  if (rare) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = fp8_codes4(w[2 * i], w[2 * i + 1], s);
  }
  if (live) {
    st16(dst + 16 * sub, make_uint4(c[0], c[1], c[2], c[3]));
    if (sub == 0) *dscale = (uint8_t)s;
  }
}

// A wave takes 8 tokens of one head: where their slots follow each other their scale bytes do too, and go out together.
__global__ __launch_bounds__(kThreads) void fp8_write_kernel(const WriteArgs a) {
  const int lane = threadIdx.x & 63, sub = lane & 7;
  const uint32_t unit = blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t group = divide(unit, a.hkv);
  const int h = (int)(unit - group * a.hkv.d);
  const int64_t first = 8 * (int64_t)group, t = min(first + (lane >> 3), a.tokens - 1);
  if (first >= a.tokens) return;
  const int64_t slot = a.slots[t];
  const uint16_t* kp = a.k + t * a.k_st + h * a.k_sh + 16 * sub;
  const uint16_t* vp = a.v + t * a.v_st + h * a.v_sh + 16 * sub;
  const uint4 k0 = ld16(kp), k1 = ld16(kp + 8), v0 = ld16(vp), v1 = ld16(vp + 8);
  const bool live = first + (lane >> 3) < a.tokens && slot >= 0 && slot < a.num_slots;
  int64_t page, off;
  if (a.num_slots < (int64_t)1 << 31) {
    const uint32_t i = live ? (uint32_t)slot : 0u, q = divide(i, a.page_size);
    page = q;
    off = i - q * a.page_size.d;
  } else {
    const int64_t i = live ? slot : 0;
    page = i / a.page_size.d;
    off = i - page * a.page_size.d;
  }
  const int64_t at = page * a.sp + off * a.st + h * a.sh, sat = page * a.ss_p + h * a.ss_h + off;
  write_row(k0, k1, live, a.kc + at, a.ks + sat, sub);
  write_row(v0, v1, live, a.vc + at, a.vs + sat, sub);
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
  int page_size, hkv;
  int64_t rows;
};

__device__ __forceinline__ void read_row(const uint4 c, uint32_t s, uint16_t* dst) {
  const float f = fp8_scale(s);
  st16(dst, make_uint4(fp8_pair<false>(c.x, f), fp8_pair<true>(c.x, f), fp8_pair<false>(c.y, f), fp8_pair<true>(c.y, f)));
  st16(dst + 8, make_uint4(fp8_pair<false>(c.z, f), fp8_pair<true>(c.z, f), fp8_pair<false>(c.w, f), fp8_pair<true>(c.w, f)));
}

__global__ __launch_bounds__(kThreads) void fp8_read_kernel(const ReadArgs a) {
  const int sub = threadIdx.x & 7;
  const int64_t row = (int64_t)blockIdx.x * kRowsPerBlock + (threadIdx.x >> 3);
  if (row >= a.rows) return;
  const int64_t t = row / a.hkv;
  const int h = (int)(row - t * a.hkv);
  const int64_t slot = a.slots[t];
  uint4 kc = make_uint4(0, 0, 0, 0), vc = kc;
  uint32_t ks = 127, vs = 127;
  if (slot >= 0 && slot < a.num_slots) {
    const int64_t page = slot / a.page_size, off = slot - page * a.page_size;
    const int64_t at = page * a.sp + off * a.st + h * a.sh + 16 * sub, sat = page * a.ss_p + h * a.ss_h + off;
    kc = ld16(a.kc + at);
    vc = ld16(a.vc + at);
    ks = a.ks[sat];
    vs = a.vs[sat];
  }
  read_row(kc, ks, a.k + t * a.k_st + h * a.k_sh + 16 * sub);
  read_row(vc, vs, a.v + t * a.v_st + h * a.v_sh + 16 * sub);
}

}  // namespace

int check_fp8_pool(const char* who, const void* kc, const void* vc, int64_t sp, int64_t st, int64_t sh, const void* ks,
                   const void* vs, int64_t ss_p, int64_t ss_h, int num_pages, int page_size, int hkv) {
  if (kc == nullptr || vc == nullptr || ks == nullptr || vs == nullptr)
    return fail(Q3A_EINVAL, "%s: null pool or scale pointer", who);
  if (num_pages < 0 || page_size < 16 || page_size % 16 != 0)
    return fail(Q3A_EINVAL, "%s: page_size %d must be a multiple of 16 and num_pages %d >= 0", who, page_size, num_pages);
  if (hkv < 1) return fail(Q3A_EINVAL, "%s: num_kv_heads %d must be positive", who, hkv);
  // the stride of a dimension of one element is not used
  if (hkv == 1) sh = ss_h = 0;
  if (num_pages == 1) sp = ss_p = 0;
  if ((((uintptr_t)kc | (uintptr_t)vc) & 15) != 0 || ((sp | st | sh) & 15) != 0 || sp < 0 || sh < 0 || st < kRowDims ||
      st > (1 << 26))
    return fail(Q3A_EINVAL, "%s: pool pointers and strides must be 16-byte aligned, strides >= 0, token stride in [128, 2^26]",
                who);
  if ((((uintptr_t)ks | (uintptr_t)vs) & 3) != 0 || ((ss_p | ss_h) & 3) != 0 || ss_p < 0 || ss_h < 0)
    return fail(Q3A_EINVAL, "%s: scale pointers and strides must be multiples of 4 and strides >= 0", who);
  return Q3A_OK;
}

namespace {
int check_rows(const char* who, const void* k, const void* v, int64_t k_st, int64_t k_sh, int64_t v_st, int64_t v_sh,
               const void* slots, int64_t tokens, int hkv, int head_dim) {
  if (head_dim != kRowDims) return fail(Q3A_EINVAL, "%s: head_dim %d (only 128)", who, head_dim);
  if (tokens < 0 || hkv < 1 || hkv > 65536 || tokens > ((int64_t)1 << 28) / hkv)  // 8 lanes a row, 8 rows a wave: below 2^32
    return fail(Q3A_EINVAL, "%s: bad token count %lld for %d KV heads (at most 65536 heads and 2^28 rows)", who, (long long)tokens, hkv);
  if (tokens == 0) return Q3A_OK;
  if (k == nullptr || v == nullptr || slots == nullptr) return fail(Q3A_EINVAL, "%s: null pointer", who);
  if (hkv == 1) k_sh = v_sh = 0;
  if (tokens == 1) k_st = v_st = 0;
  if ((((uintptr_t)k | (uintptr_t)v) & 15) != 0 || ((k_st | k_sh | v_st | v_sh) & 7) != 0 || ((uintptr_t)slots & 7) != 0)
    return fail(Q3A_EINVAL, "%s: rows must be 16-byte aligned with strides multiples of 8 elements", who);
  return Q3A_OK;
}
}  // namespace
}  // namespace q3a

using namespace q3a;

extern "C" int q3a_paged_write_fp8(const void* k, int64_t k_stride_t, int64_t k_stride_h, const void* v, int64_t v_stride_t,
                                   int64_t v_stride_h, const int64_t* slots, void* k_cache, void* v_cache,
                                   int64_t kv_stride_page, int64_t kv_stride_tok, int64_t kv_stride_head, void* k_scale,
                                   void* v_scale, int64_t scale_stride_page, int64_t scale_stride_head, int num_pages,
                                   int page_size, int64_t num_tokens, int num_kv_heads, int head_dim, void* stream) {
  const char* who = "q3a_paged_write_fp8";
  int rc = check_rows(who, k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h, slots, num_tokens, num_kv_heads, head_dim);
  if (rc != Q3A_OK) return rc;
  rc = check_fp8_pool(who, k_cache, v_cache, kv_stride_page, kv_stride_tok, kv_stride_head, k_scale, v_scale,
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
  hipLaunchKernelGGL(fp8_write_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, (hipStream_t)stream, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? Q3A_OK : fail(Q3A_ELAUNCH, "%s: %s", who, hipGetErrorString(e));
}

extern "C" int q3a_paged_read_fp8(const void* k_cache, const void* v_cache, int64_t kv_stride_page, int64_t kv_stride_tok,
                                  int64_t kv_stride_head, const void* k_scale, const void* v_scale,
                                  int64_t scale_stride_page, int64_t scale_stride_head, int num_pages, int page_size,
                                  const int64_t* slots, void* k, int64_t k_stride_t, int64_t k_stride_h, void* v,
                                  int64_t v_stride_t, int64_t v_stride_h, int64_t num_tokens, int num_kv_heads,
                                  int head_dim, void* stream) {
  const char* who = "q3a_paged_read_fp8";
  int rc = check_rows(who, k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h, slots, num_tokens, num_kv_heads, head_dim);
  if (rc != Q3A_OK) return rc;
  rc = check_fp8_pool(who, k_cache, v_cache, kv_stride_page, kv_stride_tok, kv_stride_head, k_scale, v_scale,
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
  a.page_size = page_size;
  a.hkv = num_kv_heads;
  a.rows = num_tokens * num_kv_heads;
  const int64_t blocks = (a.rows + kRowsPerBlock - 1) / kRowsPerBlock;
  hipLaunchKernelGGL(fp8_read_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, (hipStream_t)stream, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? Q3A_OK : fail(Q3A_ELAUNCH, "%s: %s", who, hipGetErrorString(e));
}
