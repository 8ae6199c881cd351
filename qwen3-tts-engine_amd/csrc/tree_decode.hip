// Attention of a few query tokens per row over the paged K/V pool, on MFMA (gfx950): decode over the 8-bit pool (plain, and
// with the step's quantising write) and attention for trees of drafted tokens over the 8-bit or the bf16 pool.
//
// Row b has N query tokens (nodes) and ctx cached tokens, all visible to every node, and N keys of its own of which node n
// sees those that its mask row allows (decode: N = 1 and no own key, or its own one as the pool will hold it).  With
// G = Hq / Hkv the M = N G query rows m = (n, g) of a KV head share every key:
//   s_mj = scale q_m . k_j,   o_m = sum_j exp(s_mj - max_j s_mj) v_j / sum_j exp(s_mj - max_j s_mj);   zeros if nothing is seen.
// K and V are read once for each block of 16 kMT query rows, so with few query rows HBM bounds it: 768 rows of 512 tokens over
// the 8-bit pool run at 6.4 TB/s (with 5 % more than the keys for the exponent bytes' lines), 256 rows of 600 tokens and 8 nodes
// over bf16 at 6.1.  63 nodes are bound by vector instructions (430 TFLOP/s), calls of a few rows by latency: 5 us from start to
// end of the shortest row, of which the keys' way is 2.5.
//
// A step is 32 keys (two 16-token subtiles, each inside one page) by 16 kMT query rows, on one wave, from registers alone (kMT is
// 1 up to 16 query rows, else 2: more do not fit the registers):
//   S^T = K Q^T   A = 16 keys, B = Q^T.  bf16: v_mfma_f32_16x16x32_bf16; lane l holds key l % 16 and, of each 32 dims, the 8
//                 that its quarter g = l / 16 takes: any split of the 128 dims over (step, quarter) is right as long as Q has
//                 the same.  8-bit codes are converted on the way, their exponent byte with them.
//   O^T = V^T P^T A = V^T: lane l holds for dim index l % 16 the 8 keys 4 g .. 4 g + 3 of both subtiles, which are the keys
//                 whose P its S^T registers hold, so P needs no lane moves.  Row i of MFMA j stands for dim 8 i + j: the
//                 lane loads 8 dims in a row of its 8 keys, and the transpose is byte permutes within the lane.
// Lane l of O^T then holds 32 dims in a row of query row l % 16.  V's scale goes onto P.  Scores, statistics and O are fp32; P
// goes into the product as two bf16 numbers, which leave 2^-15 of each term at worst.
#include <float.h>
#include <limits.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "fp8_common.h"
#include "../../include/q3attn.h"

namespace q3a {
namespace {

constexpr int kD = kRowDims;
constexpr int kStep = 32;       // keys per step
constexpr int kWindow = 32;     // steps whose page ids a wave holds at once (one id a lane)
constexpr int kMergeRow = kD + 4;  // floats per row of the merge buffer (16-byte rows off the bank period)
constexpr int kRecord = kD + 2;    // floats per query row of a record: o[128], m, l
enum { kNoKeys = 0, kTree = 1, kAppend = 2 };

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8_t;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float f32x4_t;
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));

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
  float* rec;  // in ws
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

// The first of the 8 dims that MFMA step c's operand holds in quarter g, and the 16 B piece of the row it lies in.
template <bool kFp8>
__device__ __forceinline__ int dim_of(int c, int g) {
  return kFp8 ? (c >> 1) * 64 + g * 16 + (c & 1) * 8 : c * 32 + g * 8;
}

// A step's K and V in registers: the 8-bit pool's codes, or bf16.
template <bool kFp8>
struct KeyTile;
template <>
struct KeyTile<true> {
  i32x8_t k[2];
  uint32_t ks[2];  // scale byte of key l % 16
};
template <>
struct KeyTile<false> {
  uint4 k[2][4];
};
template <bool kFp8>
struct ValueTile;
template <>
struct ValueTile<true> {
  uint2 v[2][4];
  uint32_t vs[2];  // scale bytes of keys 4 g .. 4 g + 3
};
template <>
struct ValueTile<false> {
  uint4 v[2][4];
};

// Where a step's two subtiles lie in the pool, the same on every lane.
struct Place {
  int64_t at[2];    // byte offset of the first key,
  uint32_t sat[2];  // and of its scale byte
  int valid[2];     // keys that are seen
};

// The pool places of a wave's next kWindow steps, one subtile a lane: worked out by the lanes at once, so that a step reads
// its two with a few lane reads (on the scalar unit it took 120 instructions a step, more than the step's arithmetic).
struct Window {
  uint32_t at, sat;  // offset of the first key in 16 bytes, and of its scale byte
  int valid;         // keys that are seen: 0 past the row's end, and where the table has no page
};

// Lane l's subtile is half l & 1 of step `step` of row b: its first token, that token's place in its page, the table's entry (-1
// past the table); and, once that has come, where it lies, given the row's L cached tokens.  `on`: there is such a step.
struct Entry {
  int tok, off, page;
};
__device__ __forceinline__ Entry entry_of(int b, int step, int lane) {
  const TreeArgs& a = args_again();
  Entry e = {kStep * step + 16 * (lane & 1), 0, -1};
  const int pi = (int)divide((uint32_t)e.tok, a.per_page);
  e.off = e.tok - pi * a.page_size;
  if (a.max_pages == 0) return e;
  const int page = a.bt[(int64_t)b * a.bt_sb + min(pi, a.max_pages - 1)];
  e.page = pi < a.max_pages ? page : -1;
  return e;
}
template <bool kFp8>
__device__ __forceinline__ Window window_of(const Entry& e, int L, bool on) {
  const TreeArgs& a = args_again();
  Window w = {0u, 0u, 0};
  if (on && (unsigned)e.page < (unsigned)a.num_pages) {
    w.at = (uint32_t)(((int64_t)e.page * a.sp + (int64_t)e.off * a.st) >> 4);
    if constexpr (kFp8) w.sat = (uint32_t)(e.page * a.ss_p + e.off);
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

template <int kMT>
struct State {
  f32x4_t o[kMT][8];
  float m[kMT], l[kMT];  // of query row l % 16: the exponents' base, unscaled; sum, of this quarter's keys until the merge
};

__device__ __forceinline__ int row_tokens(int b, int mode) {
  const TreeArgs& a = args_again();
  const int n = a.seqlens[b];
  const int cap = a.max_pages * a.page_size;
  if (mode == kAppend) return n < cap ? n : -1;  // no room for the new row: skipped
  return min(n, cap);
}

__device__ __forceinline__ int steps_of(int L, int mode) {
  if (L < 0) return 0;
  const TreeArgs& a = args_again();
  return (L + kStep - 1) / kStep + (mode == kTree ? (a.nodes + kStep - 1) / kStep : mode == kAppend ? 1 : 0);
}

// Cache policy of the pool's loads.  Non-temporal where a load instruction takes whole 128-byte lines that no other workgroup
// reads.
constexpr int kNt = 2;

// A step's keys are loaded from the pool by three functions.
//
// A line is 8 lanes' 16 bytes, but an A operand has a row on 4 lanes only, so loading operand rows as they are takes each line
// in two halves by two instructions, which the non-temporal policy does not suit (a twentieth of the decode's time).  So two
// lanes that hold neighbouring rows load from one key at a time:
//   8-bit codes   load i: half r & 1 of key (r & ~1) + i.  The two lanes then exchange what is the other's (a DPP move and a
//                 select a register, before the product).
//   bf16, kPaired operand row r of a load holds half (r & 1) of a line of key (r & ~3) + 2 i + ((r >> 1) & 1),
//                 i the load's pair.  Even rows have to meet Q's dims of the lines' first half, odd rows the second's: two
//                 products of which each uses half, and the score of a key is the sum of two neighbouring rows, which one lane
//                 holds.  The lane's four keys stay 4 g .. 4 g + 3.
// With 32 query rows, which vector instructions bound, the keys are loaded in rows: the exchange and the second product would cost
// more than they give.
//
// No branches and always the same loads, also for a step that is not there (its page ids are -1): only so does the compiler
// know how many newer loads may be in flight when older ones are waited for, and not wait for all.
// `live`: there is such a step; its places are not used else.  tokens: what the row has from the step on.
template <bool kFp8>
__device__ __forceinline__ Place place_of(const Window& w, int slot, bool live, int tokens) {
  Place p;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    p.at[u] = (int64_t)(uint32_t)readlane((int)w.at, 2 * slot + u) << 4;
    if constexpr (kFp8) p.sat[u] = (uint32_t)readlane((int)w.sat, 2 * slot + u);
    const int n = readlane(w.valid, 2 * slot + u), left = tokens - 16 * u;
    p.valid[u] = live ? (n < left ? n : left < 0 ? 0 : left) : 0;  // (min as a chain of scalar selects)
  }
  return p;
}

// Descriptors end with the last seen key: what lies past it is not read and comes as zeros.
template <bool kFp8>
__device__ __forceinline__ uint32_t extent(const TreeArgs& a, int valid) {
  return valid > 0 ? (uint32_t)(valid - 1) * (uint32_t)a.st + (kFp8 ? kD : 2 * kD) : 0u;
}

template <bool kOnce>
__device__ __forceinline__ void load_k(const TreeArgs& a, const Place& p, int lane, KeyTile<true>& x) {
  const int r = lane & 15, g = lane >> 4;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const auto rk = make_rsrc(a.kc + p.at[u], extent<true>(a, p.valid[u]));
    const uint32_t row = kOnce ? (uint32_t)(r & ~1) * (uint32_t)a.st + 64 * (r & 1) + 16 * g : (uint32_t)r * (uint32_t)a.st + 16 * g;
    auto ld = [&](uint32_t o) {
      return __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rk, (int)o, 0, kOnce ? kNt : 0));
    };
    x.k[u] = __builtin_shufflevector(ld(row), ld(row + (kOnce ? (uint32_t)a.st : 64u)), 0, 1, 2, 3, 4, 5, 6, 7);
    const auto rs = make_rsrc(a.ks + p.sat[u], p.valid[u] > 0 ? 16 : 0);
    x.ks[u] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(rs, r, 0, 0);
  }
}
template <bool kPaired>
__device__ __forceinline__ void load_k(const TreeArgs& a, const Place& p, int lane, KeyTile<false>& x) {
  const int r = lane & 15, g = lane >> 4;
  const uint32_t st = (uint32_t)a.st;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const auto rk = make_rsrc(a.kc + p.at[u], extent<false>(a, p.valid[u]));
    if constexpr (kPaired) {
      const uint32_t row = (uint32_t)((r & ~3) + ((r >> 1) & 1)) * st + 64 * (r & 1) + 16 * g;
#pragma unroll
      for (int i = 0; i < 4; ++i)  // pair i >> 1, line i & 1
        x.k[u][i] = buffer_load16_stream(rk, row + 2 * (i >> 1) * st + 128 * (i & 1));
    } else {
      const uint32_t row = (uint32_t)r * st + 16 * g;
#pragma unroll
      for (int i = 0; i < 4; ++i) x.k[u][i] = buffer_load16(rk, row + 64 * i);
    }
  }
}

template <bool kFp8, bool kOnce>
__device__ __forceinline__ void load_v(const TreeArgs& a, const Place& p, int lane, ValueTile<kFp8>& x) {
  const int r = lane & 15, g = lane >> 4;
  const uint32_t st = (uint32_t)a.st;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const auto rv = make_rsrc(a.vc + p.at[u], extent<kFp8>(a, p.valid[u]));
    const uint32_t row = (uint32_t)(4 * g) * st + (kFp8 ? 8 : 16) * r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kFp8) {
        x.v[u][i] = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rv, (int)(row + i * st), 0, kOnce ? kNt : 0));
      } else {
        x.v[u][i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rv, (int)(row + i * st), 0, kOnce ? kNt : 0));
      }
    }
    if constexpr (kFp8) {
      const auto rt = make_rsrc(a.vs + p.sat[u], p.valid[u] > 0 ? 16 : 0);
      x.vs[u] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rt, 4 * g, 0, 0);
    }
  }
}

// The A operands of O^T for dims 8 i + j, j = jj and jj + 1 (jj even): the pairs of keys (0, 1), (2, 3) of both subtiles.
__device__ __forceinline__ void v_operands(const ValueTile<true>& x, int jj, bf16x8_t& a0, bf16x8_t& a1) {
  uint32_t p0[4], p1[4];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const uint2 c0 = x.v[u][2 * p], c1 = x.v[u][2 * p + 1];
      const uint32_t w0 = jj < 4 ? c0.x : c0.y, w1 = jj < 4 ? c1.x : c1.y;
      // bytes (key 0 dim d, key 1 dim d, key 0 dim d + 1, key 1 dim d + 1)
      const uint32_t t = perm_b32(w1, w0, (jj & 2) ? 0x07030602u : 0x05010400u);
      p0[2 * u + p] = fp8_pair<false>(t, 1.f);
      p1[2 * u + p] = fp8_pair<true>(t, 1.f);
    }
  a0 = __builtin_bit_cast(bf16x8_t, make_uint4(p0[0], p0[1], p0[2], p0[3]));
  a1 = __builtin_bit_cast(bf16x8_t, make_uint4(p1[0], p1[1], p1[2], p1[3]));
}
__device__ __forceinline__ uint32_t word_of(const uint4& w, int i) { return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w; }
__device__ __forceinline__ void v_operands(const ValueTile<false>& x, int jj, bf16x8_t& a0, bf16x8_t& a1) {
  uint32_t p0[4], p1[4];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const uint32_t w0 = word_of(x.v[u][2 * p], jj >> 1), w1 = word_of(x.v[u][2 * p + 1], jj >> 1);
      p0[2 * u + p] = perm_b32(w1, w0, kPermLoLo);
      p1[2 * u + p] = perm_b32(w1, w0, kPermHiHi);
    }
  a0 = __builtin_bit_cast(bf16x8_t, make_uint4(p0[0], p0[1], p0[2], p0[3]));
  a1 = __builtin_bit_cast(bf16x8_t, make_uint4(p1[0], p1[1], p1[2], p1[3]));
}

// Q^T as B operands, in bf16.
template <int kMT>
struct Query {
  bf16x8_t v[kMT][4];
};

// A step's scores S^T, unscaled.  kSwapped: the keys are as load_k left them.
//
// 8-bit keys are converted to bf16, exactly: 16 instructions a subtile, which take the exponent byte along.  So the scores are those of
// the bf16 row.  (The scaled 8-bit matrix instruction takes the codes as they are, but wants Q in 8 bits too.  Two such numbers an
// element do not hold what is below 2^-14 of its row's largest element, and scores over keys that are small where that one is were
// wrong; two products where they do hold a wave's queries, and this where not, took longer than this alone: 83.2 us for 82.0, 6 long
// rows x 63 nodes, 19.9 for 19.0, 32 rows x 13 nodes, 8.8 for 8.3, one row x 1000.)
template <bool kSwapped, int kMT>
__device__ __forceinline__ void scores(const KeyTile<true>& x, const Query<kMT>& q, f32x4_t (&s)[kMT][2]) {
  const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    i32x8_t k = x.k[u];
    if constexpr (kSwapped) {
      const bool odd = (threadIdx.x & 1) != 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int even_gets = __builtin_amdgcn_update_dpp(0, k[i], kDppXor1, 0xF, 0xF, false);
        const int odd_gets = __builtin_amdgcn_update_dpp(0, k[i + 4], kDppXor1, 0xF, 0xF, false);
        k[i + 4] = odd ? k[i + 4] : even_gets;
        k[i] = odd ? odd_gets : k[i];
      }
    }
    const float f = fp8_scale(x.ks[u]);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t a = (uint32_t)k[2 * c], b = (uint32_t)k[2 * c + 1];
      const bf16x8_t kf = __builtin_bit_cast(
          bf16x8_t, make_uint4(fp8_pair<false>(a, f), fp8_pair<true>(a, f), fp8_pair<false>(b, f), fp8_pair<true>(b, f)));
#pragma unroll
      for (int t = 0; t < kMT; ++t)
        s[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, q.v[t][c], c == 0 ? zero : s[t][u], 0, 0, 0);
    }
  }
}
template <bool kPaired, int kMT>
__device__ __forceinline__ void scores(const KeyTile<false>& x, const Query<kMT>& q, f32x4_t (&s)[kMT][2]) {
  const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    if constexpr (kPaired) {
      static_assert(kMT == 1, "paired rows cost a second product");
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f32x4_t even = zero, odd = zero;
#pragma unroll
        for (int e = 0; e < 2; ++e) {  // line e
          const bf16x8_t kf = __builtin_bit_cast(bf16x8_t, x.k[u][2 * i + e]);
          even = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, q.v[0][2 * e], even, 0, 0, 0);
          odd = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, q.v[0][2 * e + 1], odd, 0, 0, 0);
        }
        s[0][u][2 * i] = even[0] + odd[1];
        s[0][u][2 * i + 1] = even[2] + odd[3];
      }
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int t = 0; t < kMT; ++t)
          s[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, x.k[u][c]), q.v[t][c],
                                                            c == 0 ? zero : s[t][u], 0, 0, 0);
    }
  }
}

// The larger of two scores, NaN if one is (its row will be NaN either way).  fmaxf would quiet each operand first.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// The scores to probabilities: scaled, masked, exp2 of them minus a base, which with the sum is updated and O rescaled to.
// kMasked: seen[t] tells which of the lane's 8 keys (bit 4 u + i) its query row sees; else the subtiles' valid ones.
//
// The base need not be the maximum, only near it and not below: where some query row's scores have outgrown it, it is set to
// their maximum and 2^kAhead more (a.ahead, in unscaled scores), which after a row's first steps hardly happens again, while with
// 16 or 32 query rows some row's maximum grows in almost every step, and rescaling is a sixth to a quarter of a step's vector
// instructions (6 rows x 63 nodes: 89.1 us with kAhead = 0, 85.5 with 4, 84.3 with 6).  No probability passes 1 for it, so that a
// product with the largest V stays finite.
constexpr float kAhead = 4.f;

template <bool kMasked, int kMT>
__device__ __forceinline__ void softmax(const int (&valid)[2], const uint32_t (&seen)[kMT], float scale, float ahead,
                                        f32x4_t (&s)[kMT][2], State<kMT>& st) {
  const bool full = valid[0] == 16 && valid[1] == 16;
  if (kMasked || !full) {
    const int g = lane_now() >> 4;
#pragma unroll
    for (int t = 0; t < kMT; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool ok = kMasked ? ((seen[t] >> (4 * u + i)) & 1) != 0 : 4 * g + i < valid[u];
          s[t][u][i] = ok ? s[t][u][i] : -INFINITY;
        }
  }
  float top[kMT];
  bool grown = false;
#pragma unroll
  for (int t = 0; t < kMT; ++t) {
    top[t] = larger(larger(larger(s[t][0][0], s[t][0][1]), larger(s[t][0][2], s[t][0][3])),
                    larger(larger(s[t][1][0], s[t][1][1]), larger(s[t][1][2], s[t][1][3])));
    top[t] = max_xor32(max_xor16(top[t]));
    grown = grown | (top[t] > st.m[t]);
  }
  if (__builtin_amdgcn_ballot_w64(grown) != 0) {
#pragma unroll
    for (int t = 0; t < kMT; ++t) {
      const float m = top[t] > st.m[t] ? top[t] + ahead : st.m[t];
      const float alpha = fast_exp2((st.m[t] - (m == -INFINITY ? 0.f : m)) * scale);
      st.m[t] = m;
      st.l[t] *= alpha;
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) st.o[t][j][i] *= alpha;
    }
  }
#pragma unroll
  for (int t = 0; t < kMT; ++t) {
    const float base = st.m[t] == -INFINITY ? 0.f : st.m[t] * scale;  // nothing seen so far: every exp2 below is of -inf
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[t][u][i] = fast_exp2(__builtin_fmaf(s[t][u][i], scale, -base));
    st.l[t] += ((s[t][0][0] + s[t][0][1]) + (s[t][0][2] + s[t][0][3])) + ((s[t][1][0] + s[t][1][1]) + (s[t][1][2] + s[t][1][3]));
  }
}

// O^T += V^T P^T, with each probability as the sum of two bf16 numbers.
//
// One bf16 number holds 8 of its significant bits, and only a row's largest one is a power of two: over eight calls the results were
// off by 0.0018 to 0.0023 of their norm instead of the 0.0017 that their own rounding to bf16 takes.  Two hold 16 bits (2^-15 of
// each probability is left) and reach the 0.0017.  The second product takes nothing where HBM is the bound (576 rows 96.8 and
// 97.0 us), a little of 32 rows x 13 nodes (18.2 -> 18.9) and more of 6 long rows x 63 nodes (76.1 -> 85.5), which vector
// instructions bound.
// Over the 8-bit pool the first part is rounded to nearest.  Over bf16, whose V may hold infinities, both parts of a probability
// over 0 have to be over 0, that no product of 0 and an infinity makes a NaN: the first is cut off from the next smaller number.
template <bool kFp8, int kMT>
__device__ __forceinline__ void values(const ValueTile<kFp8>& x, const int (&valid)[2], int lane, const f32x4_t (&p)[kMT][2],
                                       State<kMT>& st) {
  const int g = lane >> 4;
  float f[2][4];  // V's scales
  if constexpr (kFp8) {
    uint32_t bytes[2] = {x.vs[0], x.vs[1]};
    if (valid[0] != 16 || valid[1] != 16) {  // the scale byte of a key that is not seen may be anything
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int left = max(0, min(4, valid[u] - 4 * g));
        bytes[u] &= (uint32_t)((1ull << (8 * left)) - 1);
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) f[u][i] = fp8_scale((bytes[u] >> (8 * i)) & 0xffu);
  }
  bf16x8_t hi[kMT], lo[kMT];
#pragma unroll
  for (int t = 0; t < kMT; ++t) {
    uint32_t h[4], r[4];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const float a = kFp8 ? p[t][u][i] * f[u][i] : p[t][u][i], b = kFp8 ? p[t][u][i + 1] * f[u][i + 1] : p[t][u][i + 1];
        const int w = 2 * u + (i >> 1);
        if constexpr (kFp8) {
          h[w] = pack_bf16x2(a, b);
          r[w] = pack_bf16x2(a - bf16_lo(h[w]), b - bf16_hi(h[w]));
        } else {
          const uint32_t ah = __builtin_elementwise_sub_sat(__float_as_uint(a), 1u);
          const uint32_t bh = __builtin_elementwise_sub_sat(__float_as_uint(b), 1u);
          h[w] = perm_b32(bh, ah, kPermHiHi);
          r[w] = pack_bf16x2(a - bf16_hi(ah), b - bf16_hi(bh));
        }
      }
    hi[t] = __builtin_bit_cast(bf16x8_t, make_uint4(h[0], h[1], h[2], h[3]));
    lo[t] = __builtin_bit_cast(bf16x8_t, make_uint4(r[0], r[1], r[2], r[3]));
  }
#pragma unroll
  for (int jj = 0; jj < 8; jj += 2) {
    bf16x8_t a0, a1;
    v_operands(x, jj, a0, a1);
#pragma unroll
    for (int t = 0; t < kMT; ++t) {
      st.o[t][jj] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, lo[t], st.o[t][jj], 0, 0, 0);
      st.o[t][jj + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1, lo[t], st.o[t][jj + 1], 0, 0, 0);
      st.o[t][jj] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, hi[t], st.o[t][jj], 0, 0, 0);
      st.o[t][jj + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1, hi[t], st.o[t][jj + 1], 0, 0, 0);
    }
  }
}

// The pair with its halves that are not finite set to zero.
__device__ __forceinline__ uint32_t finite_halves(uint32_t w) {
  if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
  if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
  return w;
}
// 1.0 in the halves that are of kind 0 (+inf), 1 (-inf) or 2 (NaN), 0 in the others.
__device__ __forceinline__ uint32_t halves_of_kind(uint32_t w, int kind) {
  auto is = [&](uint32_t h) { return kind == 0 ? h == 0x7f80u : kind == 1 ? h == 0xff80u : (h & 0x7fffu) > 0x7f80u; };
  return (is(w & 0xffffu) ? 0x3f80u : 0u) | (is(w >> 16) ? 0x3f800000u : 0u);
}

// Adds to O what the own V elements that are not finite give the rows that see their keys: for each kind, a product of
// zeros and ones counts them.  (The elements are read again: holding them would cost every call 32 registers.)
template <int kMT>
__device__ __forceinline__ void add_not_finite(const uint16_t* vb, int ts, const uint32_t (&seen)[kMT], State<kMT>& st) {
  const TreeArgs& a = args_again();
  bf16x8_t sees[kMT];
#pragma unroll
  for (int t = 0; t < kMT; ++t) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = ((seen[t] >> (2 * i)) & 1 ? 0x3f80u : 0u) | ((seen[t] >> (2 * i + 1)) & 1 ? 0x3f800000u : 0u);
    sees[t] = __builtin_bit_cast(bf16x8_t, make_uint4(w[0], w[1], w[2], w[3]));
  }
#pragma unroll 1
  for (int kind = 0; kind < 3; ++kind) {
    const int lane = lane_now();  // (nothing of the elements is computed ahead of the loop)
    const float what = kind == 0 ? INFINITY : kind == 1 ? -INFINITY : __builtin_nanf("");
    ValueTile<false> x;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = kStep * ts + 16 * u + 4 * (lane >> 4) + i;
        const uint4 e = ld16(vb + (int64_t)min(j, a.nodes - 1) * a.vn_sn + 8 * (lane & 15));  // a key of none is not seen
        x.v[u][i] = make_uint4(halves_of_kind(e.x, kind), halves_of_kind(e.y, kind), halves_of_kind(e.z, kind),
                               halves_of_kind(e.w, kind));
      }
#pragma unroll
    for (int jj = 0; jj < 8; jj += 2) {
      bf16x8_t a[2];
      v_operands(x, jj, a[0], a[1]);
#pragma unroll
      for (int t = 0; t < kMT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const f32x4_t n = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[e], sees[t], f32x4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (n[i] > 0.f) st.o[t][jj + e][i] += what;
        }
    }
  }
}

// The nodes' own keys 32 ts .. + 31, in bf16, with each lane's query rows' view of its 8 keys.  An own V element that is
// not finite must not reach the rows that do not see its key (0 * inf in the product): such elements are zeroed in the
// product and added afterwards for the rows that see them.
template <bool kFp8, int kMT>
__device__ __forceinline__ void tree_step(const Work& w, int ts, const Query<kMT>& q, State<kMT>& st) {
  const int lane = lane_now();
  const int r = lane & 15, g = lane >> 4;
  const TreeArgs& a = args_again();
  const uint16_t* kb = a.kn + (int64_t)w.b * a.kn_sb + (int64_t)w.h * a.kn_sh;
  const uint16_t* vb = a.vn + (int64_t)w.b * a.vn_sb + (int64_t)w.h * a.vn_sh;
  KeyTile<false> x;
  ValueTile<false> y;
  // Rows past the last node read the last one's, without a branch: no query row sees them, and their V is zeroed.
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int j = min(kStep * ts + 16 * u + r, a.nodes - 1);
#pragma unroll
    for (int c = 0; c < 4; ++c) x.k[u][c] = ld16(kb + (int64_t)j * a.kn_sn + dim_of<kFp8>(c, g));
  }
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = kStep * ts + 16 * u + 4 * g + i;
      const uint4 e = ld16(vb + (int64_t)min(j, a.nodes - 1) * a.vn_sn + 8 * r);
      const uint32_t keep = j < a.nodes ? ~0u : 0u;
      y.v[u][i] = make_uint4(e.x & keep, e.y & keep, e.z & keep, e.w & keep);
    }
  uint32_t seen[kMT];
#pragma unroll
  for (int t = 0; t < kMT; ++t) {
    const int n = node_of(a, (w.mb * kMT + t) * 16 + r);
    seen[t] = 0;
    if (a.mask != nullptr) {
      const uint8_t* row = a.mask + (int64_t)w.b * a.m_sb + (int64_t)min(n, a.nodes - 1) * a.m_sn;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          seen[t] |= (row[min(kStep * ts + 16 * u + 4 * g + i, a.nodes - 1)] != 0 ? 1u : 0u) << (4 * u + i);
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) seen[t] |= (kStep * ts + 16 * u + 4 * g + i <= n ? 1u : 0u) << (4 * u + i);
    }
    // keys past the last node, and query rows of none
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int left = n < a.nodes ? max(0, min(4, a.nodes - (kStep * ts + 16 * u + 4 * g))) : 0;
      seen[t] &= ~(((0xfu << left) & 0xfu) << (4 * u));
    }
  }
  const int any[2] = {16, 16};
  f32x4_t sc[kMT][2];
  scores<false, kMT>(x, q, sc);
  softmax<true, kMT>(any, seen, a.scale_log2, a.ahead, sc, st);
  uint32_t top = 0;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w4[4] = {y.v[u][i].x, y.v[u][i].y, y.v[u][i].z, y.v[u][i].w};
      top = pk_max_u16(top, bf16_any_amax_pair(w4));
    }
  const bool any_odd = __builtin_amdgcn_ballot_w64(halves_max(top) >= 0x7f80u) != 0;
  if (any_odd) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 e = y.v[u][i];
        y.v[u][i] = make_uint4(finite_halves(e.x), finite_halves(e.y), finite_halves(e.z), finite_halves(e.w));
      }
  }
  values<false, kMT>(y, any, lane, sc, st);
  if (any_odd) add_not_finite<kMT>(vb, ts, seen, st);
}

// The largest over the four lanes that hold a row (small integers order as floats do).
__device__ __forceinline__ uint32_t row_max(uint32_t x) {
  return (uint32_t)__float_as_int(max_xor32(max_xor16(__int_as_float((int)x))));
}

// The append form's new row, quantised as the write kernel does and stored, then attended as a cached subtile of one key.
__device__ __forceinline__ void append_keys(const TreeArgs& a, const Work& w, bool store, KeyTile<true>& x, ValueTile<true>& y, int& valid) {
  const int lane = lane_now();
  const int r = lane & 15, g = lane >> 4;
  const TreeArgs& more = args_again();
  const uint16_t* kb = more.kn + (int64_t)w.b * more.kn_sb + (int64_t)w.h * more.kn_sh;
  const uint16_t* vb = more.vn + (int64_t)w.b * more.vn_sb + (int64_t)w.h * more.vn_sh;
  const int pi = (int)divide((uint32_t)w.L, more.per_page), off = w.L - pi * more.page_size;
  const int page = more.bt[(int64_t)w.b * more.bt_sb + pi];
  const bool ok = (unsigned)page < (unsigned)a.num_pages;
  uint32_t kw[16], vw[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint4 e = ld16(kb + dim_of<true>(i, g));
    kw[4 * i] = e.x;
    kw[4 * i + 1] = e.y;
    kw[4 * i + 2] = e.z;
    kw[4 * i + 3] = e.w;
  }
  const uint4 e = ld16(vb + 8 * r);
  vw[0] = e.x;
  vw[1] = e.y;
  vw[2] = e.z;
  vw[3] = e.w;
  uint32_t km = halves_max(bf16_any_amax_pair(kw)), vm = halves_max(bf16_any_amax_pair(vw));
  const bool rare = any_rare(max(km, vm));
  if (rare) {
    km = halves_max(bf16_amax_pair(kw));
    vm = halves_max(bf16_amax_pair(vw));
  }
  km = row_max(km);
  vm = dpp_max_u32<kDppXor1>(vm);
  vm = dpp_max_u32<kDppXor2>(vm);
  vm = dpp_max_u32<kDppHalfMirror>(vm);
  vm = dpp_max_u32<kDppMirror>(vm);
  const uint32_t ks = fp8_scale_byte(km), vs = fp8_scale_byte(vm);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    x.ks[u] = ks;
    y.vs[u] = vs;
    x.k[u] = i32x8_t{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) y.v[u][i] = make_uint2(0u, 0u);
  }
  uint32_t kc[8], vc[2];
#pragma unroll
  for (int i = 0; i < 8; ++i) kc[i] = fp8_finite_codes4(kw[2 * i], kw[2 * i + 1], fp8_scale(ks));
#pragma unroll
  for (int i = 0; i < 2; ++i) vc[i] = fp8_finite_codes4(vw[2 * i], vw[2 * i + 1], fp8_scale(vs));
  if (rare) {
#pragma unroll
    for (int i = 0; i < 8; ++i) kc[i] = fp8_codes4(kw[2 * i], kw[2 * i + 1], ks);
#pragma unroll
    for (int i = 0; i < 2; ++i) vc[i] = fp8_codes4(vw[2 * i], vw[2 * i + 1], vs);
  }
  valid = ok ? 1 : 0;
  if (r == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x.k[0][i] = (int)kc[i];
  }
  if (g == 0) y.v[0][0] = make_uint2(vc[0], vc[1]);
  if (store && ok) {
    const int64_t at = (int64_t)page * a.sp + (int64_t)off * a.st;
    const int64_t sat = (int64_t)page * a.ss_p + off;
    if (r == 0) {
      st16(a.kc + at + dim_of<true>(0, g), make_uint4(kc[0], kc[1], kc[2], kc[3]));
      st16(a.kc + at + dim_of<true>(2, g), make_uint4(kc[4], kc[5], kc[6], kc[7]));
    }
    if (g == 0) *reinterpret_cast<u32x2*>(a.vc + at + 8 * r) = u32x2{vc[0], vc[1]};
    if (lane == 0) {
      a.ks[sat] = (uint8_t)ks;
      a.vs[sat] = (uint8_t)vs;
    }
  }
}

template <int kMT>
__device__ __forceinline__ void clear(State<kMT>& st) {
#pragma unroll
  for (int t = 0; t < kMT; ++t) {
    st.m[t] = -INFINITY;
    st.l[t] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) st.o[t][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
}

// Q^T of the row's block of query rows as B operands; columns past the last query row have the last one's again.
template <bool kFp8, int kMT>
__device__ __forceinline__ void load_q(const Work& w, bf16x8_t (&q)[kMT][4]) {
  const int lane = lane_now();
  const TreeArgs& a = args_again();
  const int r = lane & 15, g = lane >> 4;
#pragma unroll
  for (int t = 0; t < kMT; ++t) {
    const int m = min((w.mb * kMT + t) * 16 + r, a.M - 1);
    const int n = node_of(a, m);
    const uint16_t* qp = a.q + (int64_t)w.b * a.q_sb + (int64_t)n * a.q_sn + (int64_t)(w.h * a.group + m - n * a.group) * a.q_sh;
#pragma unroll
    for (int c = 0; c < 4; ++c) q[t][c] = __builtin_bit_cast(bf16x8_t, ld16(qp + dim_of<kFp8>(c, g)));
  }
}

// A wave's cached steps in registers: as soon as a step's K has been multiplied, the next step's K is loaded in its place, and
// its V behind the V product.  (Two steps in registers ahead of the one computed were no faster, where they fitted.)
template <bool kFp8, int kMT>
struct Stream {
  static constexpr bool kOnce = kMT == 1;    // else other blocks of query rows may read the keys too
  static constexpr bool kLayout = kMT == 1;  // swapped, or paired
  KeyTile<kFp8> k;
  ValueTile<kFp8> v;
  int valid[2];

  __device__ __forceinline__ void load(const TreeArgs& a, const Place& p, int lane) {
    load_k<kOnce>(a, p, lane, k);
    load_v<kFp8, kOnce>(a, p, lane, v);
    valid[0] = p.valid[0];
    valid[1] = p.valid[1];
  }
  // Computes the step and loads the next one.
  __device__ __forceinline__ void turn(const TreeArgs& a, const Place& next, const Query<kMT>& q, int lane, State<kMT>& st) {
    const uint32_t all[kMT] = {};
    f32x4_t s[kMT][2];
    scores<kLayout, kMT>(k, q, s);
    __builtin_amdgcn_sched_barrier(0);
    load_k<kOnce>(a, next, lane, k);
    __builtin_amdgcn_sched_barrier(0);
    softmax<false, kMT>(valid, all, a.scale_log2, a.ahead, s, st);
    values<kFp8, kMT>(v, valid, lane, s, st);
    __builtin_amdgcn_sched_barrier(0);
    load_v<kFp8, kOnce>(a, next, lane, v);
    __builtin_amdgcn_sched_barrier(0);
    valid[0] = next.valid[0];
    valid[1] = next.valid[1];
  }
};

// The append form's step: the new row.
template <int kMT>
__device__ __forceinline__ void append_step(const TreeArgs& a, const Work& w, const Query<kMT>& q, int lane, State<kMT>& st) {
  const uint32_t all[kMT] = {};
  f32x4_t s[kMT][2];
  KeyTile<true> x;
  ValueTile<true> y;
  int one[2] = {0, 0};
  append_keys(a, w, w.mb == 0, x, y, one[0]);
  scores<false, kMT>(x, q, s);
  softmax<false, kMT>(one, all, a.scale_log2, a.ahead, s, st);
  values<true, kMT>(y, one, lane, s, st);
}

// Q, as it was loaded, with the sign that the scale asks for; an element that is not finite becomes NaN, as its row's result then is
// (scores of -inf alone would else give zeros).
template <int kMT>
__device__ __forceinline__ void turn_signs(Query<kMT>& q) {
  const uint32_t sign = args_again().q_sign;
  uint32_t top = 0;
#pragma unroll
  for (int t = 0; t < kMT; ++t)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint4 v = __builtin_bit_cast(uint4, q.v[t][c]);
      const uint32_t w[4] = {v.x ^ sign, v.y ^ sign, v.z ^ sign, v.w ^ sign};
      top = pk_max_u16(top, bf16_any_amax_pair(w));
      q.v[t][c] = __builtin_bit_cast(bf16x8_t, make_uint4(w[0], w[1], w[2], w[3]));
    }
  if (__builtin_amdgcn_ballot_w64(halves_max(top) >= 0x7f80u) != 0) {
#pragma unroll
    for (int t = 0; t < kMT; ++t)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint4 v = __builtin_bit_cast(uint4, q.v[t][c]);
        q.v[t][c] = __builtin_bit_cast(bf16x8_t, make_uint4(nan_if_not_finite(v.x), nan_if_not_finite(v.y), nan_if_not_finite(v.z),
                                                            nan_if_not_finite(v.w)));
      }
  }
}

// Query rows that the waves merge at once, 34 KB of them.
template <int kW>
struct MergeLds {
  static constexpr int kRows = 64 / kW;
  float o[kW][kRows][kMergeRow];
  float m[kW][kRows], l[kW][kRows];
};

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

// Merges the waves' states through LDS into the output (rec == nullptr) or a record of (o[128], m, l) floats a query row.
template <int kMT, int kW>
__device__ __forceinline__ void merge_waves(const Work& w, const State<kMT>& st, float* rec, int wave, MergeLds<kW>& s) {
  const int lane = lane_now(), thread = 64 * wave + lane;
  constexpr int kRows = MergeLds<kW>::kRows;
  const int r = lane & 15, g = lane >> 4;
  const int M = args_again().M;
  const float scale = args_again().scale_log2;
#pragma unroll
  for (int t = 0; t < kMT; ++t) {
    const float l = sum_xor32(sum_xor16(st.l[t]));
#pragma unroll
    for (int i0 = 0; i0 < 16; i0 += kRows) {
      const int m0 = (w.mb * kMT + t) * 16 + i0;
      if (m0 >= M) break;
      __syncthreads();  // the buffer's last readers
      if ((unsigned)(r - i0) < (unsigned)kRows) {
        if (g == 0) {
          s.m[wave][r - i0] = st.m[t] * scale;
          s.l[wave][r - i0] = l;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float* o = &s.o[wave][r - i0][32 * g + 8 * i];
          *reinterpret_cast<f32x4_t*>(o) = f32x4_t{st.o[t][0][i], st.o[t][1][i], st.o[t][2][i], st.o[t][3][i]};
          *reinterpret_cast<f32x4_t*>(o + 4) = f32x4_t{st.o[t][4][i], st.o[t][5][i], st.o[t][6][i], st.o[t][7][i]};
        }
      }
      __syncthreads();
      const int row = thread >> 4, d0 = 8 * (thread & 15), m = m0 + row;
      if (row < kRows && m < M) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < kW; ++i) top = fmaxf(top, s.m[i][row]);
        const float base = top == -INFINITY ? 0.f : top;
        float acc[8] = {}, sum = 0.f;
#pragma unroll
        for (int i = 0; i < kW; ++i) {
          const float f = fast_exp2(s.m[i][row] - base);
          sum += f * s.l[i][row];
#pragma unroll
          for (int d = 0; d < 8; ++d) acc[d] += f * s.o[i][row][d0 + d];
        }
        if (rec == nullptr) {
          store_out(out_row(w.b, w.h, m) + d0, acc, sum);
        } else {
          float* o = rec + (16 * t + i0 + row) * kRecord;
          if (d0 == 0) *reinterpret_cast<float2*>(o + kD) = make_float2(top, sum);
#pragma unroll
          for (int d = 0; d < 8; d += 2) *reinterpret_cast<float2*>(o + d0 + d) = make_float2(acc[d], acc[d + 1]);
        }
      }
    }
  }
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

// Rounds of kW steps that a row's work makes.  (Counting the own ones threefold, as long as they take, made the chunks longer and
// lost 5 %.)
template <int kW>
__device__ __forceinline__ uint32_t rounds_of(const TreeArgs& a, int L, int mode) {
  if (L < 0) return 0;
  const uint32_t cached = (uint32_t)(L + kStep * kW - 1) / (kStep * kW);
  return cached + (mode == kTree ? (a.nodes + kStep * kW - 1) / (kStep * kW) : mode == kAppend ? 1 : 0);
}

// Chunk `at` of all rows' chunks laid end to end.  64 rows at a time, one a lane; every wave does it.  A chunk has up to `size`
// rounds: total / target, rounded up, so that a row's 1 + floor(rounds / size) come to target + batch at most.  The target is two
// workgroups a compute unit.  One alone has its rounds in 0.6 of the time, and spares the other's start and records, about a round
// and a half: so it is one where its size is not longer by more than that (8 rows x 4000 tokens 19.0 -> 17.7 us, 1 x 4000 x 64
// nodes 20.4 -> 16.9; ragged batches mostly need two: 6 long rows x 63 nodes take 86 us with two and 135 with one).
template <int kW>
__device__ __forceinline__ Chunk chunk_at(const TreeArgs& a, uint32_t at, int mode) {
  const int lane = lane_now(), batch = a.batch, cap = a.max_pages * a.page_size;
  auto tokens = [&](int b) {  // row_tokens
    const int n = b < batch ? a.seqlens[b] : -1;
    return mode == kAppend ? (n < cap ? n : -1) : min(n, cap);
  };
  uint32_t total = 0;  // below 2^32: 1024 rows of 2^21
  int L = -1;
  for (int b = 0; b < batch; b += 64) {
    L = tokens(b + lane);
    total += (uint32_t)readlane((int)wave_scan(rounds_of<kW>(a, L, mode)), 63);
  }
  // (The reciprocals are a little large and a little small: neither count may come out too high.)
  const float two = fmaxf(1.f, floorf((float)total * a.per_target + 0.999f)), one = floorf((float)total * a.per_target_one + 0.999f);
  const float size = one <= 1.7f * two + 1.5f ? fmaxf(one, two) : two;
  const float per_size = __builtin_amdgcn_rcpf(size) * 0.999999f;
  uint32_t before = 0;
  for (int b = 0; b < batch; b += 64) {
    if (batch > 64) L = tokens(b + lane);
    const uint32_t n = b + lane < batch ? 1 + (uint32_t)((float)rounds_of<kW>(a, L, mode) * per_size) : 0u;
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
  const int bin = min(63, eighths(cap + kStep) - eighths(max(0, min(L, cap)) + kStep));
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

// One workgroup a (row, KV head, block of 16 kMT query rows), its kW waves taking the row's steps in turn; or (kChunked) one of
// a chunk of a row's steps, which leaves a record for the join kernel unless it is the row's only one.
template <bool kFp8, int kMode, int kMT, int kW, bool kChunked>
__global__ __launch_bounds__(64 * kW, kMT == 2 || (kMode == kTree && kChunked) ? 2 : 3) void tree_kernel(const TreeArgs args) {
  __shared__ __align__(16) MergeLds<kW> lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Work w;
  int unit;
  unit_of(args, w.h, w.mb, unit);
  if (unit >= args.units) return;
  Window win;
  Query<kMT> q;
  int s0 = 0, s1;  // the chunk's steps
  float* rec = nullptr;
  if constexpr (kChunked) {
    const Chunk c = chunk_at<kW>(args, (uint32_t)unit, kMode);
    if (c.row < 0) return;
    w.b = c.row;
    w.L = c.L;
    const int T = steps_of(w.L, kMode);
    w.Tc = w.L > 0 ? (w.L + kStep - 1) / kStep : 0;
    const int steps = (int)((rounds_of<kW>(args, w.L, kMode) + c.count - 1) / c.count) * kW;
    s0 = min(w.Tc, c.index * steps);
    s1 = c.index == c.count - 1 ? T : min(w.Tc, s0 + steps);  // the last one has the own steps
    if (c.count > 1)
      rec = args_again().rec + (((int64_t)unit * args_again().mblocks + w.mb) * args_again().hkv + w.h) * (int64_t)(16 * kMT * kRecord);
    if (c.index == 0 && w.h == 0 && w.mb == 0 && threadIdx.x == 0)
      reinterpret_cast<Joined*>(args_again().ws)[w.b] = Joined{unit - c.index, c.count};
    const int s = s0 + wave + kW * (lane >> 1);
    const Entry e = entry_of(w.b, s, lane);
    load_q<kFp8, kMT>(w, q.v);
    win = window_of<kFp8>(e, w.L, s < min(s1, w.Tc));
  } else {
    w.b = unit;
    const int row0 = max(0, args.batch - 64 * kW);
    if (args.order && unit >= row0) w.b = kth_longest<kW>(args, row0, unit - row0, wave);
    // The first window's page ids do not wait for the row's length.
    const Entry e = entry_of(w.b, wave + kW * (lane >> 1), lane);
    load_q<kFp8, kMT>(w, q.v);
    win = window_of<kFp8>(e, INT_MAX, true);
    w.L = __builtin_amdgcn_readfirstlane(row_tokens(w.b, kMode));
    w.Tc = w.L > 0 ? (w.L + kStep - 1) / kStep : 0;
    s1 = steps_of(w.L, kMode);
  }
  const TreeArgs a = at_head(args, w.h);
  if (s1 == 0 && rec == nullptr) {
    zero_rows(w.b, w.h, w.mb, 16 * kMT);
    return;
  }
  State<kMT> st;
  if (s0 + wave >= s1) {
    clear(st);
  } else {
    const int first = s0 + wave;
    const int n = max(0, (min(s1, w.Tc) - first + kW - 1) / kW);  // this wave's cached steps: first, first + kW, ...
    const int own = first + n * kW;  // and its first own step, taken ahead of them, while they are on their way
    auto place = [&](int j) __attribute__((always_inline)) {
      if ((j & (kWindow - 1)) == 0 && j > 0 && j < n) {
        const int l = lane_now();
        win = window_of<kFp8>(entry_of(w.b, first + kW * (j + (l >> 1)), l), w.L, j + (l >> 1) < n);
      }
      return place_of<kFp8>(win, j & (kWindow - 1), j < n, w.L - kStep * (first + kW * j));
    };
    Stream<kFp8, kMT> x;
    if constexpr (kMode == kTree) {
      // A wave that has own steps takes them first.  Chunks, which are few, ask for their keys ahead of them; where the chip is
      // full the registers that this takes would cost every compute unit its third workgroup (256 rows x 600 tokens x 8 nodes
      // over the 8-bit pool: 64.4 us with three, 67.6 with two; one row of four nodes: 0.5 us the other way).
      constexpr bool kEarly = kChunked && (kFp8 || kMT == 1);
      auto own_steps = [&]() __attribute__((always_inline)) {
        turn_signs(q);
        clear(st);
        for (int s = own; s < s1; s += kW) tree_step<kFp8, kMT>(w, s - w.Tc, q, st);
      };
      if constexpr (kEarly) {
        x.load(a, place(0), lane);
        own_steps();
      } else if (own < s1) {
        own_steps();
        x.load(a, place(0), lane);
      } else {
        x.load(a, place(0), lane);
        turn_signs(q);
        clear(st);
      }
    } else {
      x.load(a, place(0), lane);
      turn_signs(q);
      clear(st);
      if constexpr (kMode == kAppend) {
        if (own < s1) append_step<kMT>(a, w, q, lane, st);
      }
    }
    const TreeArgs again = at_head(args_again(), w.h);  // (not held in registers, and spilled, since the kernel's start)
    for (int i = 0; i < n; ++i) x.turn(again, place(i + 1), q, lane, st);
  }
  merge_waves<kMT, kW>(w, st, rec, wave, lds);
}

// Merges a row's records, for 16 query rows of a head.  16 lanes a query row, 8 dims a lane; the thread groups that the query
// rows leave share the records.  A chain of two round trips (where the records are, and they), so what can be is worked out ahead
// of them, without divisions.
template <int kMT>
__global__ __launch_bounds__(256) void tree_join_kernel(const TreeArgs a) {
  __shared__ float s_o[16][kD + 4];
  __shared__ float s_m[16], s_l[16];
  const int h = blockIdx.x, b = blockIdx.y, mb = blockIdx.z / kMT, tile = 16 * (blockIdx.z % kMT);
  const Joined d = reinterpret_cast<const Joined*>(a.ws)[b];
  const int n = d.count, rows = min(16, a.M - mb * 16 * kMT - tile);
  if (n == 1 || rows <= 0) return;
  const int group = threadIdx.x >> 4, d0 = 8 * (threadIdx.x & 15);
  const int bits = rows > 8 ? 4 : rows > 4 ? 3 : rows > 2 ? 2 : rows - 1;  // 2^bits query rows at once
  const int share = 16 >> bits, mine = group >> bits, i = group & ((1 << bits) - 1);
  const int64_t step = (int64_t)a.mblocks * a.hkv * (16 * kMT * kRecord);  // from a chunk's records to the next one's
  const float* rec = a.rec + d.first * step + ((int64_t)mb * a.hkv + h) * (16 * kMT * kRecord) + (tile + i) * kRecord;
  const int m = mb * 16 * kMT + tile + i, node = node_of(a, m);
  uint16_t* out = a.out + b * a.o_sb + node * a.o_sn + (int64_t)(h * a.group + m - node * a.group) * a.o_sh + d0;
  float acc[8] = {}, sum = 0.f, top = -INFINITY;
  if (i < rows) {
#pragma unroll 4
    for (int c = mine; c < n; c += share) {
      const float* o = rec + c * step;
      const float2 ml = *reinterpret_cast<const float2*>(o + kD);
      float e[8];
#pragma unroll
      for (int k = 0; k < 8; k += 2) {
        const float2 v = *reinterpret_cast<const float2*>(o + d0 + k);
        e[k] = v.x;
        e[k + 1] = v.y;
      }
      const float next = fmaxf(top, ml.x), base = next == -INFINITY ? 0.f : next;
      const float f0 = fast_exp2(top - base), f1 = fast_exp2(ml.x - base);
      top = next;
      sum = sum * f0 + ml.y * f1;
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[k] = acc[k] * f0 + e[k] * f1;
    }
  }
  if (share > 1) {  // the same for every thread
    if (d0 == 0) {
      s_m[group] = top;
      s_l[group] = sum;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) s_o[group][d0 + k] = acc[k];
    __syncthreads();
    if (mine == 0) {
      float all = -INFINITY;
      for (int c = 0; c < share; ++c) all = fmaxf(all, s_m[(c << bits) + i]);
      const float base = all == -INFINITY ? 0.f : all;
      sum = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[k] = 0.f;
      for (int c = 0; c < share; ++c) {
        const float f = fast_exp2(s_m[(c << bits) + i] - base);
        sum += f * s_l[(c << bits) + i];
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] += f * s_o[(c << bits) + i][d0 + k];
      }
    }
  }
  if (mine == 0 && i < rows) store_out(out, acc, sum);
}

// ---------------------------------------------------------------------------------------------------- host side

constexpr int kWaves = 4;

int tiles_per_wave(int M) { return M <= 16 ? 1 : 2; }


struct Plan {
  int mblocks, units, target, target_one;  // target == 0: whole rows
  size_t rows, bytes;
};

// From the shape alone: the lengths are on the device.
Plan plan_of(int batch, int nodes, int hq, int hkv, int64_t capacity) {
  Plan p = {};
  const int M = nodes * (hq / hkv), tiles = tiles_per_wave(M);
  p.mblocks = (M + 16 * tiles - 1) / (16 * tiles);
  p.units = batch;
  // Whole rows take one launch, but the longest row's steps follow each other on one compute unit; chunks cost the join (3.7 us)
  // and records.  Rows of one length, us whole and in chunks: 8 workgroups of 512 tokens 7.5 and 8.2, of 1000 11.1 and 8.4; 64 of
  // 1000 11.5 and 11.0; 128 of 1000 12.1 and 12.7, of 2000 20.5 and 18.2; 256 of 1000 13.7 and 18.1.  Ragged rows leave whole ones
  // waiting for the longest: 192 workgroups of up to 1373 tokens 15.0 and 12.8, 256 of up to 1725 (13 nodes) 23.4 and 19.1, but 512
  // of up to 1500 18.9 and 23.2.  Rows that are more than the chip holds at once balance by themselves.
  const int64_t groups = (int64_t)batch * hkv * p.mblocks;
  if (batch > 1024 || capacity * num_cus() <= 700 * (num_cus() + groups)) return p;
  // (Three workgroups a compute unit: decode 3 % slower, trees of 32 query rows 6 to 25 %.)
  auto target = [&](int each) {
    const int slots = each * num_cus() / (hkv * p.mblocks);
    return std::max({1, slots - batch / 2, slots / 2});
  };
  if (target(2) < 2) return p;  // a single row's heads and nodes fill the chip, or nearly
  p.target = target(2);
  p.target_one = target(1);
  p.units = p.target + batch;
  p.rows = ((size_t)batch * sizeof(Joined) + 15) & ~(size_t)15;
  p.bytes = p.rows + (size_t)p.units * p.mblocks * hkv * 16 * tiles * kRecord * sizeof(float);
  return p;
}

template <bool kFp8, int kMode, int kMT>
int launch(const TreeArgs& a, const char* who, hipStream_t stream) {
  hipError_t e;
  const unsigned heads = (unsigned)(a.hkv * a.mblocks), units = (unsigned)a.units;
  const dim3 grid = a.xcd_units ? dim3(8 * heads, (units + 7) / 8) : dim3(heads, units);
  if (a.target == 0) {
    hipLaunchKernelGGL((tree_kernel<kFp8, kMode, kMT, kWaves, false>), grid, dim3(64 * kWaves), 0, stream, a);
    e = hipGetLastError();
  } else {
    hipLaunchKernelGGL((tree_kernel<kFp8, kMode, kMT, kWaves, true>), grid, dim3(64 * kWaves), 0, stream, a);
    e = hipGetLastError();
    if (e == hipSuccess) {
      hipLaunchKernelGGL((tree_join_kernel<kMT>), dim3(a.hkv, (unsigned)a.batch, a.mblocks * kMT), dim3(256), 0, stream, a);
      e = hipGetLastError();
    }
  }
  return e == hipSuccess ? Q3A_OK : fail(Q3A_ELAUNCH, "%s: %s", who, hipGetErrorString(e));
}

int check_shape(const char* who, int batch, int nodes, int hq, int hkv, int head_dim, int max_pages, int page_size) {
  if (head_dim != kD) return fail(Q3A_EINVAL, "%s: head_dim %d (only 128)", who, head_dim);
  if (batch < 0 || batch > 65535) return fail(Q3A_EINVAL, "%s: batch %d outside [0, 65535]", who, batch);
  if (nodes < 1 || nodes > 256) return fail(Q3A_EINVAL, "%s: %d query tokens a row, outside [1, 256]", who, nodes);
  if (hkv < 1 || hkv > 64 || hq < hkv || hq % hkv != 0 || hq / hkv > 16)
    return fail(Q3A_EINVAL, "%s: %d query heads over %d KV heads (a multiple, at most 16 to one; at most 64 KV heads)", who, hq,
                hkv);
  if (page_size < 16 || page_size % 16 != 0) return fail(Q3A_EINVAL, "%s: page_size %d must be a multiple of 16", who, page_size);
  if (max_pages < 0 || (int64_t)max_pages * page_size > (1 << 28))
    return fail(Q3A_EINVAL, "%s: table of %d pages of %d tokens (at most 2^28 tokens a row)", who, max_pages, page_size);
  return Q3A_OK;
}

bool misaligned(const void* p, int64_t a, int64_t b, int64_t c) { return ((uintptr_t)p & 15) != 0 || ((a | b | c) & 7) != 0; }

// Fills what every form shares and launches; `mode` as the enum.
int run(const char* who, TreeArgs a, int mode, bool fp8, int batch, int hq, size_t workspace_bytes, int64_t kv_page, int64_t kv_tok,
        int64_t kv_head, float softmax_scale, void* stream) {
  const int elem = fp8 ? 1 : 2;
  // the stride of a dimension of one element may be anything
  if (batch == 1) a.q_sb = a.o_sb = a.kn_sb = a.vn_sb = 0;
  if (a.nodes == 1) a.q_sn = a.o_sn = a.kn_sn = a.vn_sn = 0;
  if (a.hkv == 1) a.kn_sh = a.vn_sh = 0;
  if (hq == 1) a.q_sh = a.o_sh = 0;
  if (a.num_pages == 1) kv_page = a.ss_p = 0;
  if (a.q == nullptr || a.out == nullptr || a.seqlens == nullptr || (a.bt == nullptr && a.max_pages > 0))
    return fail(Q3A_EINVAL, "%s: null pointer", who);
  if (misaligned(a.q, a.q_sb, a.q_sn, a.q_sh) || misaligned(a.out, a.o_sb, a.o_sn, a.o_sh))
    return fail(Q3A_EINVAL, "%s: q and out rows must be 16-byte aligned with strides multiples of 8 elements", who);
  if (mode != kNoKeys) {
    if (a.kn == nullptr || a.vn == nullptr) return fail(Q3A_EINVAL, "%s: null new rows", who);
    if (misaligned(a.kn, a.kn_sb, a.kn_sn, a.kn_sh) || misaligned(a.vn, a.vn_sb, a.vn_sn, a.vn_sh))
      return fail(Q3A_EINVAL, "%s: new k and v rows must be 16-byte aligned with strides multiples of 8 elements", who);
  }
  a.group = hq / a.hkv;
  a.M = a.nodes * a.group;
  // (in floating point: the products of any strides)
  if (((double)a.num_pages * (double)kv_page + (double)a.page_size * (double)kv_tok) * elem >= 0x1p36 ||
      (fp8 && (double)a.num_pages * (double)a.ss_p + a.page_size >= 0x1p32))
    return fail(Q3A_EINVAL, "%s: a cache of 64 GiB or more, or scales of 4 GiB", who);
  const Plan p = plan_of(batch, a.nodes, hq, a.hkv, (int64_t)a.max_pages * a.page_size);
  if (p.bytes > 0 && (a.ws == nullptr || workspace_bytes < p.bytes || ((uintptr_t)a.ws & 15) != 0))
    return fail(Q3A_ESPACE, "%s: workspace of %zu bytes, %zu needed (16-byte aligned)", who, workspace_bytes, p.bytes);
  a.batch = batch;
  a.per_group = ((1u << 20) + a.group - 1) / a.group;
  a.per_page = divisor((uint32_t)a.page_size);
  a.per_hkv = divisor((uint32_t)a.hkv);
  a.mblocks = p.mblocks;
  a.units = p.units;
  a.target = p.target;
  if (p.target > 0) {
    a.per_target = 1.000001f / (float)p.target;
    a.per_target_one = 1.000001f / (float)p.target_one;
  }
  a.xcd_units = p.units >= 32;
  a.order = p.target == 0 && batch > 1 && (int64_t)batch * a.hkv * p.mblocks > num_cus();
  a.rec = p.target > 0 ? reinterpret_cast<float*>(static_cast<char*>(a.ws) + p.rows) : nullptr;
  a.sp = kv_page * elem;
  a.st = (int)(kv_tok * elem);
  a.sh = kv_head * elem;
  // The kernels take a positive scale (maxima are of the unscaled scores): Q's sign is turned for a negative one, and 0, with
  // which masked scores of -inf would be NaN, becomes the smallest there is.
  a.q_sign = softmax_scale < 0.f ? 0x80008000u : 0u;
  a.scale_log2 = softmax_scale == 0.f ? FLT_MIN : fabsf(softmax_scale) * kLog2e;
  a.ahead = std::min(kAhead / a.scale_log2, 1e30f);
  const hipStream_t s = (hipStream_t)stream;
  if (mode == kNoKeys) return launch<true, kNoKeys, 1>(a, who, s);
  if (mode == kAppend) return launch<true, kAppend, 1>(a, who, s);
  switch (tiles_per_wave(a.M)) {
    case 1: return fp8 ? launch<true, kTree, 1>(a, who, s) : launch<false, kTree, 1>(a, who, s);
    default: return fp8 ? launch<true, kTree, 2>(a, who, s) : launch<false, kTree, 2>(a, who, s);
  }
}

}  // namespace
}  // namespace q3a

using namespace q3a;

extern "C" size_t q3a_paged_decode_tree_workspace_bytes(int batch, int num_nodes, int num_q_heads, int num_kv_heads, int head_dim,
                                                        int max_pages_per_seq, int page_size) {
  if (check_shape("q3a_paged_decode_tree_workspace_bytes", batch, num_nodes, num_q_heads, num_kv_heads, head_dim,
                  max_pages_per_seq, page_size) != Q3A_OK || batch == 0)
    return 0;
  return plan_of(batch, num_nodes, num_q_heads, num_kv_heads, (int64_t)max_pages_per_seq * page_size).bytes;
}

extern "C" int q3a_paged_decode_fp8(const void* q, int64_t q_stride_b, int64_t q_stride_h, const void* k_cache,
                                    const void* v_cache, int64_t kv_stride_page, int64_t kv_stride_tok, int64_t kv_stride_head,
                                    const void* k_scale, const void* v_scale, int64_t scale_stride_page,
                                    int64_t scale_stride_head, int num_pages, int page_size, const int32_t* cache_seqlens,
                                    const int32_t* block_table, int64_t bt_stride_b, int max_pages_per_seq, void* out,
                                    int64_t o_stride_b, int64_t o_stride_h, void* workspace, size_t workspace_bytes, int batch,
                                    int num_q_heads, int num_kv_heads, int head_dim, float softmax_scale, void* stream) {
  const char* who = "q3a_paged_decode_fp8";
  int rc = check_shape(who, batch, 1, num_q_heads, num_kv_heads, head_dim, max_pages_per_seq, page_size);
  if (rc != Q3A_OK) return rc;
  rc = check_fp8_pool(who, k_cache, v_cache, kv_stride_page, kv_stride_tok, kv_stride_head, k_scale, v_scale,
                      scale_stride_page, scale_stride_head, num_pages, page_size, num_kv_heads);
  if (rc != Q3A_OK || batch == 0) return rc;
  TreeArgs a = {};
  a.q = (const uint16_t*)q;
  a.q_sb = q_stride_b;
  a.q_sh = q_stride_h;
  a.kc = (uint8_t*)const_cast<void*>(k_cache);
  a.vc = (uint8_t*)const_cast<void*>(v_cache);
  a.ks = (uint8_t*)const_cast<void*>(k_scale);
  a.vs = (uint8_t*)const_cast<void*>(v_scale);
  a.ss_p = scale_stride_page;
  a.ss_h = scale_stride_head;
  a.num_pages = num_pages;
  a.page_size = page_size;
  a.seqlens = cache_seqlens;
  a.bt = block_table;
  a.bt_sb = bt_stride_b;
  a.max_pages = max_pages_per_seq;
  a.out = (uint16_t*)out;
  a.o_sb = o_stride_b;
  a.o_sh = o_stride_h;
  a.ws = workspace;
  a.nodes = 1;
  a.hkv = num_kv_heads;
  return run(who, a, kNoKeys, true, batch, num_q_heads, workspace_bytes, kv_stride_page, kv_stride_tok, kv_stride_head,
             softmax_scale, stream);
}

extern "C" int q3a_paged_decode_fp8_append(
    const void* q, int64_t q_stride_b, int64_t q_stride_h, const void* k_new, int64_t kn_stride_b, int64_t kn_stride_h,
    const void* v_new, int64_t vn_stride_b, int64_t vn_stride_h, void* k_cache, void* v_cache, int64_t kv_stride_page,
    int64_t kv_stride_tok, int64_t kv_stride_head, void* k_scale, void* v_scale, int64_t scale_stride_page,
    int64_t scale_stride_head, int num_pages, int page_size, const int32_t* cache_seqlens, const int32_t* block_table,
    int64_t bt_stride_b, int max_pages_per_seq, void* out, int64_t o_stride_b, int64_t o_stride_h, void* workspace,
    size_t workspace_bytes, int batch, int num_q_heads, int num_kv_heads, int head_dim, float softmax_scale, void* stream) {
  const char* who = "q3a_paged_decode_fp8_append";
  int rc = check_shape(who, batch, 1, num_q_heads, num_kv_heads, head_dim, max_pages_per_seq, page_size);
  if (rc != Q3A_OK) return rc;
  rc = check_fp8_pool(who, k_cache, v_cache, kv_stride_page, kv_stride_tok, kv_stride_head, k_scale, v_scale,
                      scale_stride_page, scale_stride_head, num_pages, page_size, num_kv_heads);
  if (rc != Q3A_OK || batch == 0) return rc;
  TreeArgs a = {};
  a.q = (const uint16_t*)q;
  a.q_sb = q_stride_b;
  a.q_sh = q_stride_h;
  a.kn = (const uint16_t*)k_new;
  a.kn_sb = kn_stride_b;
  a.kn_sh = kn_stride_h;
  a.vn = (const uint16_t*)v_new;
  a.vn_sb = vn_stride_b;
  a.vn_sh = vn_stride_h;
  a.kc = (uint8_t*)k_cache;
  a.vc = (uint8_t*)v_cache;
  a.ks = (uint8_t*)k_scale;
  a.vs = (uint8_t*)v_scale;
  a.ss_p = scale_stride_page;
  a.ss_h = scale_stride_head;
  a.num_pages = num_pages;
  a.page_size = page_size;
  a.seqlens = cache_seqlens;
  a.bt = block_table;
  a.bt_sb = bt_stride_b;
  a.max_pages = max_pages_per_seq;
  a.out = (uint16_t*)out;
  a.o_sb = o_stride_b;
  a.o_sh = o_stride_h;
  a.ws = workspace;
  a.nodes = 1;
  a.hkv = num_kv_heads;
  return run(who, a, kAppend, true, batch, num_q_heads, workspace_bytes, kv_stride_page, kv_stride_tok, kv_stride_head,
             softmax_scale, stream);
}

extern "C" int q3a_paged_decode_tree(
    const void* q, int64_t q_stride_b, int64_t q_stride_n, int64_t q_stride_h, const void* k_new, int64_t kn_stride_b,
    int64_t kn_stride_n, int64_t kn_stride_h, const void* v_new, int64_t vn_stride_b, int64_t vn_stride_n, int64_t vn_stride_h,
    const uint8_t* tree_mask, int64_t mask_stride_b, int64_t mask_stride_n, const void* k_cache, const void* v_cache,
    int64_t kv_stride_page, int64_t kv_stride_tok, int64_t kv_stride_head, const void* k_scale, const void* v_scale,
    int64_t scale_stride_page, int64_t scale_stride_head, int num_pages, int page_size, const int32_t* cache_seqlens,
    const int32_t* block_table, int64_t bt_stride_b, int max_pages_per_seq, void* out, int64_t o_stride_b, int64_t o_stride_n,
    int64_t o_stride_h, void* workspace, size_t workspace_bytes, int batch, int num_nodes, int num_q_heads, int num_kv_heads,
    int head_dim, float softmax_scale, void* stream) {
  const char* who = "q3a_paged_decode_tree";
  int rc = check_shape(who, batch, num_nodes, num_q_heads, num_kv_heads, head_dim, max_pages_per_seq, page_size);
  if (rc != Q3A_OK) return rc;
  const bool fp8 = k_scale != nullptr || v_scale != nullptr;
  if (fp8) {
    rc = check_fp8_pool(who, k_cache, v_cache, kv_stride_page, kv_stride_tok, kv_stride_head, k_scale, v_scale,
                        scale_stride_page, scale_stride_head, num_pages, page_size, num_kv_heads);
    if (rc != Q3A_OK) return rc;
  } else if (k_cache == nullptr || v_cache == nullptr || num_pages < 0 || (((uintptr_t)k_cache | (uintptr_t)v_cache) & 15) != 0 ||
             (num_pages > 1 && ((kv_stride_page & 7) != 0 || kv_stride_page < 0)) ||
             (num_kv_heads > 1 && ((kv_stride_head & 7) != 0 || kv_stride_head < 0)) || (kv_stride_tok & 7) != 0 ||
             kv_stride_tok < kD || kv_stride_tok > (1 << 26)) {
    return fail(Q3A_EINVAL, "%s: pool pointers must be 16-byte aligned, strides >= 0 and multiples of 8, token stride in "
                            "[128, 2^26]", who);
  }
  if (batch == 0) return Q3A_OK;
  TreeArgs a = {};
  a.q = (const uint16_t*)q;
  a.q_sb = q_stride_b;
  a.q_sn = q_stride_n;
  a.q_sh = q_stride_h;
  a.kn = (const uint16_t*)k_new;
  a.kn_sb = kn_stride_b;
  a.kn_sn = kn_stride_n;
  a.kn_sh = kn_stride_h;
  a.vn = (const uint16_t*)v_new;
  a.vn_sb = vn_stride_b;
  a.vn_sn = vn_stride_n;
  a.vn_sh = vn_stride_h;
  a.mask = tree_mask;
  a.m_sb = mask_stride_b;
  a.m_sn = mask_stride_n;
  a.kc = (uint8_t*)const_cast<void*>(k_cache);
  a.vc = (uint8_t*)const_cast<void*>(v_cache);
  a.ks = (uint8_t*)const_cast<void*>(k_scale);
  a.vs = (uint8_t*)const_cast<void*>(v_scale);
  a.ss_p = scale_stride_page;
  a.ss_h = scale_stride_head;
  a.num_pages = num_pages;
  a.page_size = page_size;
  a.seqlens = cache_seqlens;
  a.bt = block_table;
  a.bt_sb = bt_stride_b;
  a.max_pages = max_pages_per_seq;
  a.out = (uint16_t*)out;
  a.o_sb = o_stride_b;
  a.o_sn = o_stride_n;
  a.o_sh = o_stride_h;
  a.ws = workspace;
  a.nodes = num_nodes;
  a.hkv = num_kv_heads;
  return run(who, a, kTree, fp8, batch, num_q_heads, workspace_bytes, kv_stride_page, kv_stride_tok, kv_stride_head,
             softmax_scale, stream);
}
