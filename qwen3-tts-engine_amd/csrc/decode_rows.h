// What the kernels over rows of a paged pool share (tree_decode.hip, fp4_decode.hip): their arguments, how a wave finds its steps'
// pages, how rows are cut into chunks or put in order, and the records that chunks leave (gfx950).
#pragma once

#include "fp4_common.h"

#include <limits.h>
#include <math.h>

#include <type_traits>

namespace q3a {

// Own keys of a row: none, the tree's nodes, the step's new row behind the cached ones, or that row as one of them (its place in the pool is
// read, whatever it holds, and replaced in registers).
enum { kNoKeys = 0, kTree = 1, kAppend = 2, kAppendKey = 3 };
enum { kBf16Pool = 0, kFp8Pool = 1, kFp4Pool = 2 };

constexpr int kD = kRowDims;
constexpr int kRecord = kD + 2;    // floats per query row of a record: o[128], m, l

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8_t;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float f32x4_t;

struct TreeArgs {
  const uint16_t* q;
  int64_t q_sb, q_sn, q_sh;
  const uint16_t *kn, *vn;  // the nodes' own keys (tree) or the step's new rows (append)
  int64_t kn_sb, kn_sn, kn_sh, vn_sb, vn_sn, vn_sh;
  const uint8_t* mask;      // tree: node n sees own key j if mask[b * m_sb + n * m_sn + j]; nullptr: j <= n
  int64_t m_sb, m_sn;
  uint8_t *kc, *vc;
  int64_t sp, sh;           // pool strides in bytes
  int st;
  uint8_t *ks, *vs;
  int64_t ss_p, ss_h;
  int num_pages, page_size;
  Divisor per_page;
  const int32_t* seqlens;
  const int32_t* bt;
  int64_t bt_sb;
  int max_pages;
  uint16_t* out;
  int64_t o_sb, o_sn, o_sh;
  void* ws;
  float* rec;    // in ws
  int rec_rows;  // query rows of a record, of one head
  int batch, nodes, group, hkv, M;
  Divisor per_hkv;
  uint32_t per_group;  // m / group = m * per_group >> 20 for m < 4096
  int mblocks;
  int units, target;  // rows, or chunks at most and as many as there should be
  float per_target, per_target_one;  // 1 / target, a little more; the same of half as many workgroups
  int xcd_units;
  int order;  // whole rows start in the order of their lengths
  float scale_log2, ahead;  // positive; kAhead / scale_log2, as far as a score may be added to it
  uint32_t q_sign;    // turns the signs of a pair of bf16, or nothing
};

// Query row m's node.
__device__ __forceinline__ int node_of(const TreeArgs& a, int m) { return (int)(((uint32_t)m * a.per_group) >> 20); }

// The lane's number, worked out where it is asked for.  What derives from it only where rows start and end would else be
// computed once and hold registers through the loops between.
__device__ __forceinline__ int lane_now() {
  int zero = 0;
  asm volatile("" : "+v"(zero));
  return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, (uint32_t)zero));
}

__device__ __forceinline__ int readlane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// The kernel's arguments read again from where they are passed.  The compiler loads every argument at a kernel's start and
// holds it in scalar registers, which run out (and spill); what only the end of a row needs goes through here instead.
__device__ __forceinline__ const TreeArgs& args_again() {
  typedef __attribute__((address_space(4))) const TreeArgs karg;
  auto p = (karg*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const TreeArgs*)p;
}

// The pool places of a wave's next kWindow steps, one subtile a lane: worked out by the lanes at once, so that a step reads
// its two with a few lane reads (on the scalar unit it took 120 instructions a step, more than the step's arithmetic).
struct Window {
  uint32_t at, sat;  // offset of the first key in 16 bytes, and of its scale byte
  int valid;         // keys that are seen: 0 past the row's end, and where the table has no page
};

// A step is kSub subtiles of 16 keys; lane l's is l % kSub of step `step` of row b: its first token, that token's place in its page,
// the table's entry (-1 past the table); and, once that has come, where it lies, given the row's L cached tokens.  `on`: there is
// such a step.
struct Entry {
  int tok, off, page;
};
template <int kSub>
__device__ __forceinline__ Entry entry_of(int b, int step, int lane) {
  const TreeArgs& a = args_again();
  Entry e = {16 * kSub * step + 16 * (lane & (kSub - 1)), 0, -1};
  const int pi = (int)divide((uint32_t)e.tok, a.per_page);
  e.off = e.tok - pi * a.page_size;
  if (a.max_pages == 0) return e;
  const int page = a.bt[(int64_t)b * a.bt_sb + min(pi, a.max_pages - 1)];
  e.page = pi < a.max_pages ? page : -1;
  return e;
}
template <int kPool>
__device__ __forceinline__ Window window_of(const Entry& e, int L, bool on) {
  const TreeArgs& a = args_again();
  Window w = {0u, 0u, 0};
  if (on && (unsigned)e.page < (unsigned)a.num_pages) {
    w.at = (uint32_t)(((int64_t)e.page * a.sp + (int64_t)e.off * a.st) >> 4);
    if constexpr (kPool != kBf16Pool) w.sat = (uint32_t)(e.page * a.ss_p + e.off);
    w.valid = max(0, min(16, L - e.tok));
  }
  return w;
}

// One row (b), KV head and block of 16 kMT query rows.
struct Work {
  int b, h, mb;
  int L;   // cached tokens that are attended
  int Tc;  // steps of cached keys; the own keys' come behind them
};

__device__ __forceinline__ int row_tokens(int b, int mode) {
  const TreeArgs& a = args_again();
  const int n = a.seqlens[b];
  const int cap = a.max_pages * a.page_size;
  if (mode == kAppend) return n < cap ? n : -1;  // no room for the new row: skipped
  return min(n, cap);
}

// Steps of kKeys keys, the own ones among them.
template <int kKeys>
__device__ __forceinline__ int steps_of(int L, int mode) {
  if (L < 0) return 0;
  const TreeArgs& a = args_again();
  return (L + kKeys - 1) / kKeys + (mode == kTree ? (a.nodes + kKeys - 1) / kKeys : mode == kAppend ? 1 : 0);
}

// Cache policy of the pool's loads.  Non-temporal where a load instruction takes whole 128-byte lines that no other workgroup
// reads.
constexpr int kNt = 2;

// The larger of two scores, NaN if one is (its row will be NaN either way).  fmaxf would quiet each operand first.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

__device__ __forceinline__ uint16_t* out_row(int b, int h, int m) {
  const TreeArgs& a = args_again();
  const int n = node_of(a, m);
  return a.out + (int64_t)b * a.o_sb + (int64_t)n * a.o_sn + (int64_t)(h * a.group + m - n * a.group) * a.o_sh;
}

__device__ __forceinline__ void store_out(uint16_t* op, const float (&acc)[8], float sum) {
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  st16(op, make_uint4(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv),
                      pack_bf16x2(acc[4] * inv, acc[5] * inv), pack_bf16x2(acc[6] * inv, acc[7] * inv)));
}

__device__ __forceinline__ void zero_rows(int b, int h, int mb, int rows) {
  const int row = threadIdx.x >> 4, d0 = 8 * (threadIdx.x & 15);
  for (int i = row; i < rows; i += blockDim.x >> 4) {
    const int m = mb * rows + i;
    if (m < args_again().M) st16(out_row(b, h, m) + d0, make_uint4(0u, 0u, 0u, 0u));
  }
}

// The arguments with the pools at KV head h.
__device__ __forceinline__ TreeArgs at_head(const TreeArgs& a, int h) {
  TreeArgs b = a;
  b.kc += (int64_t)h * a.sh;
  b.vc += (int64_t)h * a.sh;
  b.ks += (int64_t)h * a.ss_h;
  b.vs += (int64_t)h * a.ss_h;
  return b;
}

// A workgroup's KV head, block of query rows and unit (a row, or a chunk of one).  Workgroups go to the 8 XCDs in
// turn.  With many units, unit i goes to XCD i % 8 with all its heads, which follow each other there: their exponent bytes
// share lines, and their rows of a token-major pool share DRAM pages.  With few units the heads go to different XCDs.
__device__ __forceinline__ void unit_of(const TreeArgs& a, int& h, int& mb, int& unit) {
  const uint32_t y = a.xcd_units ? blockIdx.x >> 3 : blockIdx.x;
  mb = (int)divide(y, a.per_hkv);
  h = (int)y - mb * a.hkv;
  unit = a.xcd_units ? 8 * blockIdx.y + (blockIdx.x & 7) : blockIdx.y;
}

// Inclusive sum over the wave's lanes.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  auto add = [&](auto ctrl, auto rows) __attribute__((always_inline)) {
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
  };
  using std::integral_constant;
  add(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});  // lanes 1, 2, 4, 8 below in the row of 16
  add(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
  add(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
  add(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
  add(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});  // row 0's last lane to row 1, row 2's to row 3
  add(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});  // row 1's last to rows 2 and 3
  return x;
}

// What the chunked form's workgroup finds for its chunk.
struct Chunk {
  int row, L;           // row < 0: there is no such chunk
  int index, count;     // which of the row's chunks
};

struct Joined {
  int first, count;  // a row's chunks
};

// Rounds of kKeys keys, a step of each wave, that a row's work makes.  (Counting the own ones threefold, as long as they take, made the
// chunks longer and lost 5 %.)
template <int kKeys>
__device__ __forceinline__ uint32_t rounds_of(const TreeArgs& a, int L, int mode) {
  if (L < 0) return 0;
  const uint32_t cached = (uint32_t)(L + kKeys - 1) / kKeys;
  return cached + (mode == kTree ? (a.nodes + kKeys - 1) / kKeys : mode == kAppend ? 1 : 0);
}

// Chunk `at` of all rows' chunks laid end to end.  64 rows at a time, one a lane; every wave does it.  A chunk has up to `size`
// rounds: total / target, rounded up, so that a row's 1 + floor(rounds / size) come to target + batch at most.  The target is two
// workgroups a compute unit.  One alone has its rounds in 0.6 of the time, and spares the other's start and records, about a round
// and a half: so it is one where its size is not longer by more than that (8 rows x 4000 tokens 19.0 -> 17.7 us, 1 x 4000 x 64
// nodes 20.4 -> 16.9; ragged batches mostly need two: 6 long rows x 63 nodes take 86 us with two and 135 with one).
template <int kKeys>
__device__ __forceinline__ Chunk chunk_at(const TreeArgs& a, uint32_t at, int mode) {
  const int lane = lane_now(), batch = a.batch, cap = a.max_pages * a.page_size;
  auto tokens = [&](int b) {  // row_tokens
    const int n = b < batch ? a.seqlens[b] : -1;
    return mode == kAppend ? (n < cap ? n : -1) : mode == kAppendKey ? (n >= 0 && n < cap ? n + 1 : -1) : min(n, cap);
  };
  uint32_t total = 0;  // below 2^32: 1024 rows of 2^21
  int L = -1;
  for (int b = 0; b < batch; b += 64) {
    L = tokens(b + lane);
    total += (uint32_t)readlane((int)wave_scan(rounds_of<kKeys>(a, L, mode)), 63);
  }
  // (The reciprocals are a little large and a little small: neither count may come out too high.)
  const float two = fmaxf(1.f, floorf((float)total * a.per_target + 0.999f)), one = floorf((float)total * a.per_target_one + 0.999f);
  const float size = one <= 1.7f * two + 1.5f ? fmaxf(one, two) : two;
  const float per_size = __builtin_amdgcn_rcpf(size) * 0.999999f;
  uint32_t before = 0;
  for (int b = 0; b < batch; b += 64) {
    if (batch > 64) L = tokens(b + lane);
    const uint32_t n = b + lane < batch ? 1 + (uint32_t)((float)rounds_of<kKeys>(a, L, mode) * per_size) : 0u;
    const uint32_t upto = before + wave_scan(n);
    const uint64_t has = __builtin_amdgcn_ballot_w64(at < upto);
    if (has != 0) {
      const int j = (int)__builtin_ctzll(has), count = readlane((int)n, j);
      return {b + j, readlane(L, j), (int)at - (readlane((int)upto, j) - count), count};
    }
    before = (uint32_t)readlane((int)upto, 63);
  }
  return {-1, 0, 0, 0};
}

// The k-th of the batch's last rows, from row0 on (up to 64 kW), by their lengths, longest first.  Workgroups start in the order
// of their numbers, and the last to start should be short: 250 rows of 200 to 1200 tokens took 57.3 us as they came, 48.5 so,
// 256 rows of 8 nodes 121.3 and 110.7 (equal ones 106.3 and 107.8, over the 8-bit pool 61.8 and 64.4), 576 rows of 100 to 1700
// tokens 119.4 and 110.0 (all 576 in order, with four times the rows a wave, gained 2 % more, but equal rows lost 5 %).  Rows are
// told apart by eighths of octaves below the table's length, 64 of them, and stand in their own order within one: each wave counts
// a part of them in LDS, and the wave whose count the k-th falls into finds it.
template <int kW>
__device__ __forceinline__ int kth_longest(const TreeArgs& a, int row0, int k, int wave) {
  __shared__ int s_count[kW][64];
  __shared__ int s_row;
  const int lane = lane_now(), b = row0 + 64 * wave + lane;
  const int cap = a.max_pages * a.page_size;
  const int L = a.seqlens[min(b, a.batch - 1)];
  s_count[wave][lane] = 0;
  auto eighths = [](int n) { return __float_as_int((float)n) >> 20; };
  const int bin = min(63, eighths(cap + 32) - eighths(max(0, min(L, cap)) + 32));
  const bool is = b < a.batch;
  if (is) atomicAdd(&s_count[wave][bin], 1);
  __syncthreads();
  int n[kW], all = 0;
#pragma unroll
  for (int i = 0; i < kW; ++i) {
    n[i] = s_count[i][lane];
    all += n[i];
  }
  const int upto = (int)wave_scan((uint32_t)all);
  const int in = (int)__builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > k));  // the k-th's bin
  k -= readlane(upto - all, in);
#pragma unroll
  for (int i = 0; i < kW - 1; ++i)
    if (i < wave) k -= readlane(n[i], in);
  const uint64_t alike = __builtin_amdgcn_ballot_w64(is && bin == in);
  if (is && bin == in && k == (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(alike >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)alike, 0u)))
    s_row = b;
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(s_row);
}

// Decode over the 4-bit pool with up to 8 query heads to a KV head (fp4_decode.hip): rows whole, or in chunks where a.target > 0.
hipError_t launch_fp4_decode(const TreeArgs& a, int mode, dim3 grid, hipStream_t stream);

}  // namespace q3a
