// Moves of what a paged K/V pool holds (gfx950): whole pages to other pages, and the kept tokens of rows to the front of their
// pages, in every cache of a list (all layers' K and V, and their scales) at once.
//
// Nothing is computed, so HBM bounds both, and at few pages the launch does: a call moves every cache in one launch, where one
// launch a cache would take 56 for 28 layers.  The caches' addresses go in with the kernel's arguments.
// Compaction has one workgroup a (cache, KV head, row), which goes through its row chunk by chunk: with few of them that chain is the time,
// not HBM (rows of 4000 tokens of which 2400 stay, bf16, 8 KV heads: one row in one layer, 16 workgroups, 52.7 us where its bytes take 4.1;
// 16 rows in one layer, 256 workgroups, 64.6 and 65.5 at a large copy's rate; one row in 28 layers 105.8 and 115).
// What is moved passes once: non-temporal stores, and loads in copies (600 pages in 28 layers, 1.1 GB, 212 us or 5.2 TB/s, 224 without
// both; a copy of 4 GiB by the library 4.8 TB/s.  48 rows compacted, 3.1 GB, 656 us or 4.8 TB/s and 672 without; with the loads as well
// 643, but one row 24.9 instead of 21.7).
#include <limits.h>

#include <algorithm>

#include "fp8_common.h"
#include "../../include/q3attn.h"

namespace q3a {
namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------------------------------------------- copies of pages

constexpr int kMaxCopies = 128;    // caches a launch
constexpr int kMaxShapes = 4;      // different shapes of them
constexpr int kCopyUnits = 8;      // units a thread

// A page of a cache as n1 x n0 runs of memory, counted in units of 16 or 4 bytes.
struct PageShape {
  int64_t page;            // strides in bytes
  int64_t s1, s0;
  Divisor per_page, per_run, per_n0;
  int num_pages;
  uint32_t blocks;         // workgroups a cache takes
  int end;                 // caches up to here have this shape, from the last shape's on
};
struct CopyArgs {
  uint8_t* base[kMaxCopies];
  PageShape shape[kMaxShapes];
  const int32_t *src, *dst;
  uint32_t pairs;
};

template <class T, bool kDense>
__global__ __launch_bounds__(kThreads) void copy_pages_kernel(const CopyArgs a) {
  const int e = blockIdx.y;
  int k = 0;
#pragma unroll
  for (int i = 0; i < kMaxShapes - 1; ++i) k += e >= a.shape[i].end ? 1 : 0;
  const PageShape& s = a.shape[k];
  if (blockIdx.x >= s.blocks) return;
  uint8_t* base = a.base[e];
  const uint32_t total = s.per_page.d * a.pairs;  // below 2^31
  const uint32_t first = blockIdx.x * (kThreads * kCopyUnits) + threadIdx.x;
  T x[kCopyUnits];
  int64_t to[kCopyUnits];
#pragma unroll
  for (int i = 0; i < kCopyUnits; ++i) {
    const uint32_t u = first + i * kThreads;
    to[i] = -1;
    if (u < total) {
      const uint32_t pair = divide(u, s.per_page), in = u - pair * s.per_page.d;
      const int p = a.src[pair], q = a.dst[pair];
      if ((unsigned)p < (unsigned)s.num_pages && (unsigned)q < (unsigned)s.num_pages && p != q) {
        int64_t off;
        if constexpr (kDense) {
          off = (int64_t)in * sizeof(T);
        } else {
          const uint32_t run = divide(in, s.per_run), i1 = divide(run, s.per_n0);
          off = (int64_t)(in - run * s.per_run.d) * sizeof(T) + i1 * s.s1 + (run - i1 * s.per_n0.d) * s.s0;
        }
        x[i] = __builtin_nontemporal_load(reinterpret_cast<const T*>(base + p * s.page + off));
        to[i] = q * s.page + off;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kCopyUnits; ++i)
    if (to[i] >= 0) __builtin_nontemporal_store(x[i], reinterpret_cast<T*>(base + to[i]));
}

// ---------------------------------------------------------------------------------------------------- compaction of rows

constexpr int kMaxRows = 128;                 // caches a launch
constexpr int kSpan = 2048;                   // tokens whose mask a workgroup takes at once
constexpr int kSpanPages = kSpan / 16 + 1;    // pages that these may touch

struct CompactArgs {
  uint8_t* code[kMaxRows];
  uint8_t* scale[kMaxRows];
  int64_t sp, st, sh;      // strides in bytes
  int64_t ss_p, ss_h;
  const uint8_t* keep;
  int64_t keep_sb;
  int keep_width;
  const int32_t* seqlens;
  const int32_t* bt;
  int64_t bt_sb;
  int max_pages, num_pages;
  Divisor per_page, hkv;
  int32_t* lengths;        // null in all but a call's first launch
};

// One workgroup a (cache, KV head, row).  Kept tokens go to the front in order, so token j of them comes from a place not before j:
// a chunk's rows are read before any is written (a barrier between), and what a chunk writes lies before all that later ones read.
// kLanes: 16-byte pieces of a row of codes; kBlocks: exponent bytes of it.
template <int kLanes, int kBlocks>
__global__ __launch_bounds__(kThreads) void compact_kernel(const CompactArgs a) {
  constexpr int kAtOnce = kThreads / kLanes;              // tokens of a pass
  constexpr int kPasses = kLanes == 16 ? 8 : 4;           // passes of a chunk
  __shared__ int s_src[kSpan];                            // kept tokens of the span
  __shared__ int s_from[kSpanPages], s_to[kSpanPages];    // page ids of the span's tokens, and of the places they go to
  __shared__ int s_part[kThreads / 64];
  const int thread = threadIdx.x, lane = thread & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6);
  const uint32_t e = divide(blockIdx.x, a.hkv);
  const int h = (int)(blockIdx.x - e * a.hkv.d), b = blockIdx.y;
  const int page_size = (int)a.per_page.d;
  const int L = min(a.seqlens[b], a.max_pages * page_size);
  const bool tells = a.lengths != nullptr && blockIdx.x == 0;
  if (L <= 0) {
    if (tells && thread == 0) a.lengths[b] = L;
    return;
  }
  uint8_t* code = a.code[e] + h * a.sh;
  uint8_t* scale = kBlocks > 0 ? a.scale[e] + h * a.ss_h : nullptr;
  const int32_t* table = a.bt + b * a.bt_sb;
  const uint8_t* keep = a.keep + b * a.keep_sb;
  const int sub = thread & (kLanes - 1);
  int done = 0;  // kept tokens so far
  for (int t0 = 0; t0 < L; t0 += kSpan) {
    // The span's kept tokens, 8 of its tokens a thread.
    constexpr int kEach = kSpan / kThreads;
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int t = t0 + kEach * thread + i;
      if (t < L && (t >= a.keep_width || keep[t] != 0)) bits |= 1u << i;
    }
    int upto = __builtin_popcount(bits);
    const int mine = upto;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int x = __shfl_up(upto, d);
      if (lane >= d) upto += x;
    }
    __syncthreads();  // the last span's readers
    if (lane == 63) s_part[wave] = upto;
    __syncthreads();
    int at = upto - mine, n = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) {
      if (i < wave) at += s_part[i];
      n += s_part[i];
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if ((bits >> i) & 1) s_src[at++] = t0 + kEach * thread + i;
    const int from0 = (int)divide((uint32_t)t0, a.per_page), to0 = (int)divide((uint32_t)done, a.per_page);
    if (thread < kSpanPages) {
      s_from[thread] = from0 + thread < a.max_pages ? table[from0 + thread] : -1;
      s_to[thread] = to0 + thread < a.max_pages ? table[to0 + thread] : -1;
    }
    __syncthreads();
    if (done + n == t0 + min(kSpan, L - t0)) {  // nothing is dropped up to here
      done += n;
      continue;
    }
    for (int c = 0; c < n; c += kAtOnce * kPasses) {
      u32x4 x[kPasses];
      uint8_t y[kPasses];
      int64_t to[kPasses], sto[kPasses];
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        const int j = c + i * kAtOnce + thread / kLanes;
        to[i] = -1;
        if (j < n) {
          const int t = s_src[j], d = done + j;
          const int tp = (int)divide((uint32_t)t, a.per_page), dp = (int)divide((uint32_t)d, a.per_page);
          const int p = s_from[tp - from0], q = s_to[dp - to0];
          if (t != d && (unsigned)p < (unsigned)a.num_pages && (unsigned)q < (unsigned)a.num_pages) {
            const int to_off = t - tp * page_size, d_off = d - dp * page_size;
            x[i] = *reinterpret_cast<const u32x4*>(code + p * a.sp + to_off * a.st + 16 * sub);
            to[i] = q * a.sp + d_off * a.st + 16 * sub;
            if (kBlocks > 0 && sub < kBlocks) {
              y[i] = scale[p * a.ss_p + sub * page_size + to_off];
              sto[i] = q * a.ss_p + sub * page_size + d_off;
            }
          }
        }
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // every lane's reads are done before another's writes
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kPasses; ++i)
        if (to[i] >= 0) {
          __builtin_nontemporal_store(x[i], reinterpret_cast<u32x4*>(code + to[i]));
          if (kBlocks > 0 && sub < kBlocks) scale[sto[i]] = y[i];
        }
    }
    done += n;
  }
  if (tells && thread == 0) a.lengths[b] = done;
}

template <int kLanes, int kBlocks>
int launch_compact(const char* who, const CompactArgs& a, int caches, int hkv, int batch, hipStream_t stream) {
  hipLaunchKernelGGL((compact_kernel<kLanes, kBlocks>), dim3((unsigned)(caches * hkv), (unsigned)batch), dim3(kThreads), 0, stream, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? Q3A_OK : fail(Q3A_ELAUNCH, "%s: %s", who, hipGetErrorString(e));
}

bool same_shape(const q3a_page_cache& a, const q3a_page_cache& b) {
  return a.stride_page == b.stride_page && a.stride_1 == b.stride_1 && a.stride_0 == b.stride_0 && a.n_1 == b.n_1 && a.n_0 == b.n_0 &&
         a.run_bytes == b.run_bytes && a.num_pages == b.num_pages;
}

}  // namespace
}  // namespace q3a

using namespace q3a;

extern "C" int q3a_paged_copy(const q3a_page_cache* caches, int num_caches, const int32_t* src, const int32_t* dst,
                              int64_t num_pairs, void* stream) {
  const char* who = "q3a_paged_copy";
  if (num_caches < 0 || (num_caches > 0 && caches == nullptr)) return fail(Q3A_EINVAL, "%s: bad list of caches", who);
  if (num_pairs < 0 || num_pairs > INT_MAX) return fail(Q3A_EINVAL, "%s: bad number of pairs %lld", who, (long long)num_pairs);
  bool by16 = true, dense = true;
  for (int i = 0; i < num_caches; ++i) {
    const q3a_page_cache& c = caches[i];
    if (c.num_pages < 0 || c.n_0 < 1 || c.n_1 < 1 || c.run_bytes < 1 || c.stride_page < 0 || c.stride_0 < 0 || c.stride_1 < 0)
      return fail(Q3A_EINVAL, "%s: cache %d: sizes must be positive and strides >= 0", who, i);
    const uint64_t all = (uint64_t)(uintptr_t)c.base | c.run_bytes | (c.n_0 > 1 ? c.stride_0 : 0) | (c.n_1 > 1 ? c.stride_1 : 0) |
                         (c.num_pages > 1 ? c.stride_page : 0);
    if ((all & 3) != 0) return fail(Q3A_EINVAL, "%s: cache %d: addresses, runs and strides must be multiples of 4 bytes", who, i);
    by16 = by16 && (all & 15) == 0;
    dense = dense && c.n_0 == 1 && c.n_1 == 1;
    // (in floating point: the products of any sizes)
    if ((double)c.run_bytes * (double)c.n_0 * (double)c.n_1 * (double)std::max<int64_t>(num_pairs, 1) >= 0x1p33)
      return fail(Q3A_EINVAL, "%s: cache %d: 8 GiB or more to copy in one call", who, i);
    if (c.base == nullptr && c.num_pages > 0) return fail(Q3A_EINVAL, "%s: cache %d: null pointer", who, i);
  }
  if (num_caches == 0 || num_pairs == 0) return Q3A_OK;
  if (src == nullptr || dst == nullptr) return fail(Q3A_EINVAL, "%s: null page lists", who);
  const int unit = by16 ? 16 : 4;
  for (int at = 0; at < num_caches;) {
    CopyArgs a = {};
    a.src = src;
    a.dst = dst;
    a.pairs = (uint32_t)num_pairs;
    // The launch's caches in the list's order, which may go from shape to shape (a layer's K, V and their scales, the next layer's).
    uint8_t of[kMaxCopies];                     // each one's shape
    const q3a_page_cache* like[kMaxShapes];     // and a cache of it
    int many[kMaxShapes] = {};
    int n = 0, shapes = 0;
    uint32_t most = 0;
    while (at + n < num_caches && n < kMaxCopies) {
      const q3a_page_cache& c = caches[at + n];
      int k = n > 0 ? of[n - 1] : 0;
      if (n == 0 || !same_shape(c, *like[k])) {
        k = 0;
        while (k < shapes && !same_shape(c, *like[k])) ++k;
      }
      if (k == shapes) {
        if (shapes == kMaxShapes) break;
        PageShape& s = a.shape[shapes];
        like[shapes++] = &c;
        const int64_t run = c.run_bytes / unit;
        s.page = c.stride_page;
        s.s1 = c.stride_1;
        s.s0 = c.stride_0;
        s.num_pages = c.num_pages;
        s.per_run = divisor((uint32_t)run);
        s.per_n0 = divisor((uint32_t)c.n_0);
        s.per_page = divisor((uint32_t)(run * c.n_0 * c.n_1));
        const int64_t units = (int64_t)s.per_page.d * num_pairs;
        s.blocks = (uint32_t)((units + kThreads * kCopyUnits - 1) / (kThreads * kCopyUnits));
        most = std::max(most, s.blocks);
      }
      ++many[k];
      of[n++] = (uint8_t)k;
    }
    int next[kMaxShapes], end = 0;
    for (int k = 0; k < kMaxShapes; ++k) {
      next[k] = end;
      end += many[k];
      a.shape[k].end = end;
    }
    for (int i = 0; i < n; ++i) a.base[next[of[i]]++] = (uint8_t*)caches[at + i].base;
    const dim3 grid(most, (unsigned)n);
    const hipStream_t st = (hipStream_t)stream;
    if (by16 && dense) hipLaunchKernelGGL((copy_pages_kernel<u32x4, true>), grid, dim3(kThreads), 0, st, a);
    else if (by16) hipLaunchKernelGGL((copy_pages_kernel<u32x4, false>), grid, dim3(kThreads), 0, st, a);
    else hipLaunchKernelGGL((copy_pages_kernel<uint32_t, false>), grid, dim3(kThreads), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(Q3A_ELAUNCH, "%s: %s", who, hipGetErrorString(e));
    at += n;
  }
  return Q3A_OK;
}

extern "C" int q3a_paged_compact(void* const* caches, void* const* scales, int num_caches, int row_bytes, int scale_blocks,
                                 int64_t stride_page, int64_t stride_tok, int64_t stride_head, int64_t scale_stride_page,
                                 int64_t scale_stride_head, int num_pages, int page_size, const uint8_t* keep,
                                 int64_t keep_stride_b, int keep_width, const int32_t* cache_seqlens, const int32_t* block_table,
                                 int64_t bt_stride_b, int max_pages_per_seq, int32_t* new_seqlens, int batch, int num_kv_heads,
                                 void* stream) {
  const char* who = "q3a_paged_compact";
  if (num_caches < 1 || caches == nullptr) return fail(Q3A_EINVAL, "%s: at least one cache", who);
  const bool known = (row_bytes == 256 && scale_blocks == 0) || (row_bytes == 128 && (scale_blocks == 0 || scale_blocks == 1)) ||
                     (row_bytes == 64 && (scale_blocks == 0 || scale_blocks == 4));
  if (!known)
    return fail(Q3A_EINVAL, "%s: rows of %d bytes with %d scales (256 with none, 128 with 1, 64 with 4, or codes alone)", who, row_bytes,
                scale_blocks);
  if (scale_blocks > 0 && scales == nullptr) return fail(Q3A_EINVAL, "%s: null scales", who);
  if (batch < 0 || batch > 65535) return fail(Q3A_EINVAL, "%s: batch %d outside [0, 65535]", who, batch);
  if (num_kv_heads < 1 || num_kv_heads > 65536) return fail(Q3A_EINVAL, "%s: %d KV heads, outside [1, 65536]", who, num_kv_heads);
  if (num_pages < 0 || page_size < 16 || page_size % 16 != 0)
    return fail(Q3A_EINVAL, "%s: page_size %d must be a multiple of 16 and num_pages %d >= 0", who, page_size, num_pages);
  if (max_pages_per_seq < 0 || (int64_t)max_pages_per_seq * page_size > (1 << 28))
    return fail(Q3A_EINVAL, "%s: table of %d pages of %d tokens (at most 2^28 tokens a row)", who, max_pages_per_seq, page_size);
  if (keep_width < 0) return fail(Q3A_EINVAL, "%s: bad mask width %d", who, keep_width);
  if (num_kv_heads == 1) stride_head = scale_stride_head = 0;
  if (num_pages == 1) stride_page = scale_stride_page = 0;
  if (((stride_page | stride_tok | stride_head) & 15) != 0 || stride_page < 0 || stride_tok < row_bytes || stride_head < 0 ||
      scale_stride_page < 0 || scale_stride_head < 0)
    return fail(Q3A_EINVAL, "%s: strides must be multiples of 16 bytes (scales': any) and >= 0, the token stride at least a row", who);
  for (int i = 0; i < num_caches; ++i)
    if (caches[i] == nullptr || ((uintptr_t)caches[i] & 15) != 0 || (scale_blocks > 0 && scales[i] == nullptr))
      return fail(Q3A_EINVAL, "%s: cache %d: null, or not 16-byte aligned", who, i);
  if (batch == 0) return Q3A_OK;
  if (cache_seqlens == nullptr || new_seqlens == nullptr || (keep == nullptr && keep_width > 0) ||
      (block_table == nullptr && max_pages_per_seq > 0))
    return fail(Q3A_EINVAL, "%s: null pointer", who);
  CompactArgs a = {};
  a.sp = stride_page;
  a.st = stride_tok;
  a.sh = stride_head;
  a.ss_p = scale_stride_page;
  a.ss_h = scale_stride_head;
  a.keep = keep;
  a.keep_sb = keep_stride_b;
  a.keep_width = keep_width;
  a.seqlens = cache_seqlens;
  a.bt = block_table;
  a.bt_sb = bt_stride_b;
  a.max_pages = max_pages_per_seq;
  a.num_pages = num_pages;
  a.per_page = divisor((uint32_t)page_size);
  a.hkv = divisor((uint32_t)num_kv_heads);
  for (int at = 0; at < num_caches; at += kMaxRows) {
    const int n = std::min(kMaxRows, num_caches - at);
    for (int i = 0; i < n; ++i) {
      a.code[i] = (uint8_t*)caches[at + i];
      a.scale[i] = scale_blocks > 0 ? (uint8_t*)scales[at + i] : nullptr;
    }
    a.lengths = at == 0 ? new_seqlens : nullptr;
    const hipStream_t st = (hipStream_t)stream;
    int rc;
    if (row_bytes == 256) rc = launch_compact<16, 0>(who, a, n, num_kv_heads, batch, st);
    else if (row_bytes == 128) rc = scale_blocks ? launch_compact<8, 1>(who, a, n, num_kv_heads, batch, st) : launch_compact<8, 0>(who, a, n, num_kv_heads, batch, st);
    else rc = scale_blocks ? launch_compact<4, 4>(who, a, n, num_kv_heads, batch, st) : launch_compact<4, 0>(who, a, n, num_kv_heads, batch, st);
    if (rc != Q3A_OK) return rc;
  }
  return Q3A_OK;
}
