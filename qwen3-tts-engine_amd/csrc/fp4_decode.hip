// Decode attention over the 4-bit K/V pool with up to 8 query heads to a KV head (gfx950).  (More than 8 take tree_decode.hip's
// kernel, which converts 4-bit keys to bf16.)
//
// At 136 bytes a token and KV head the pool's keys pass at four times the rate of bf16 ones, and what bounds the general kernel over
// them is vector instructions: 16 query rows' worth of softmax for 2, and a conversion for every pair of codes.  Here a wave's step is
// 64 keys (four 16-token subtiles u, each inside one page), 160 vector instructions for up to 4 heads.  HBM bounds long rows (128 x 4000
// tokens 6.4 TB/s, 576 of 64 to 1800 5.6), few rows the chain of a row's start, its longest wave's steps (0.7 us each) and the merge: 5.6 us
// for one of 64 tokens, 7.2 for one of 900.  With:
//   S = Q K^T     the scaled matrix instruction takes K's codes and exponent bytes as they are stored: v_mfma_scale_f32_16x16x128,
//                 B = 16 keys: lane l holds block g = l / 16 (32 dims) of key l % 16.  It wants 8 bits or fewer of Q too, so Q is
//                 split, exactly, into four e4m3 parts with exponents of their own for each block (prepare_q), and the 16 rows of A
//                 are 4 query heads x 4 parts.  Quarter g of the result holds the parts of head g, one a register: their sum is the
//                 score of head g and key l % 16.
//   O = P V       v_mfma_f32_16x16x32_bf16, without a transpose of V.  A byte of codes is two dims of one key, and so is the pair of
//                 bf16 that it converts to: an operand register's two k places are those two dims (d, d + 1) of one key, where P is
//                 (p, 0) in one row of A and (0, p) in another.  Their results are the two dims.  With P as two bf16 numbers (2^-15 of a
//                 probability is left) the 16 rows are 4 heads x 2 numbers x 2 dims, and quarter g of O is head g's, as of S: the
//                 softmax's statistics, O's rescaling and its last sums stay in the lane.  P goes to the operand's layout through 1 or
//                 2 KB of the wave's own LDS, without a barrier.  B = V: lane l holds dims 8 (l % 16) .. + 7 of the keys 8 (g / 2) +
//                 2 i + g % 2, i = 0 .. 3 of each subtile; column l % 16 of MFMA j stands for dims 8 (l % 16) + 2 j, + 1.
#include <algorithm>

#include "decode_rows.h"
#include "../../include/q3attn.h"

namespace q3a {
namespace {

constexpr int kSub = 4;
constexpr int kStep = 16 * kSub;      // keys per step
constexpr int kWindow = 64 / kSub;    // steps whose pages a wave holds at once
constexpr int kQRow = kD + 16;        // bytes of a row of Q's parts in LDS, off the bank period
constexpr int kPRow = 2 * kStep + 16; // the same of a row of P: one of the two numbers of 64 probabilities

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int key_of(int g, int i) { return 8 * (g >> 1) + 2 * i + (g & 1); }

// Global loads of a scalar base and a lane's offset.  (The offset is made new for each: widened to 64 bits once, ahead of the loop, it would
// take two registers and two additions a load.)
typedef const __attribute__((address_space(1))) uint8_t* gptr;
template <class T>
__device__ __forceinline__ T load_at(gptr base, uint32_t off) {
  asm volatile("" : "+v"(off));
  return *(const __attribute__((address_space(1))) T*)(base + off);
}
// Codes.  kOnce: a head's tokens are neighbours in memory, so that a load takes whole lines which no other workgroup reads: non-temporal
// (128 rows x 4000 tokens 86.5 us, 98.8 without).  Else two heads share a line, and one's load leaves it for the other's (125.2 us, 141.0
// with).
template <bool kOnce, class T>
__device__ __forceinline__ T load_codes(gptr base, uint32_t off) {
  asm volatile("" : "+v"(off));
  const auto p = (const __attribute__((address_space(1))) T*)(base + off);
  return kOnce ? __builtin_nontemporal_load(p) : *p;
}

// The pool at one KV head.
struct Pool {
  gptr kc, vc, ks, vs;
  int st, page_size;
};
__device__ __forceinline__ Pool pool_of(const TreeArgs& a, int h) {
  return {(gptr)a.kc + (int64_t)h * a.sh, (gptr)a.vc + (int64_t)h * a.sh, (gptr)a.ks + (int64_t)h * a.ss_h, (gptr)a.vs + (int64_t)h * a.ss_h,
          a.st, a.page_size};
}

// Where a step lies, the same on every lane.
struct Place {
  int64_t at[kSub];      // byte offset of a subtile's first key,
  uint32_t sat[kSub];    // and of its first exponent byte
  int full;              // all keys are seen, else
  int valid[kSub];       // so many of each subtile
};

// The lane's offsets in a subtile: of its key's block and of its four keys' dims, and of their exponent bytes.  All 16 keys of a subtile
// are loaded whatever part of them is seen (a page is a multiple of 16), and the pool's first ones where the table has no page: any codes
// are finite, and meet probabilities of 0.
struct Offsets {
  uint32_t k, ks, v[4], vs;
};
__device__ __forceinline__ Offsets offsets_of(const Pool& a, int lane) {
  const int r = lane & 15, g = lane >> 4;
  Offsets o;
  o.k = (uint32_t)(r * a.st + 16 * g);
  o.ks = (uint32_t)(g * a.page_size + (r & ~3));
#pragma unroll
  for (int i = 0; i < 4; ++i) o.v[i] = (uint32_t)(key_of(g, i) * a.st + 4 * r);
  o.vs = (uint32_t)((r >> 2) * a.page_size + 8 * (g >> 1));
  return o;
}

struct Tile {
  uint4 k[kSub];            // block g of key l % 16
  uint32_t ks[kSub];        // its exponent byte, with its neighbours' of the aligned four
  uint32_t v[kSub][4];      // dims 8 (l % 16) .. + 7 of keys key_of(g, 0 .. 3)
  uint2 vs[kSub];           // their block's exponent bytes of keys 8 (g / 2) .. + 7

  template <bool kOnce>
  __device__ __forceinline__ void load_k(const Pool& a, const Place& p, int u, const Offsets& o) {
    k[u] = __builtin_bit_cast(uint4, load_codes<kOnce, u32x4>(a.kc + p.at[u], o.k));
    ks[u] = load_at<uint32_t>(a.ks + p.sat[u], o.ks);
  }
  template <bool kOnce>
  __device__ __forceinline__ void load_v(const Pool& a, const Place& p, int u, const Offsets& o) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[u][i] = load_codes<kOnce, uint32_t>(a.vc + p.at[u], o.v[i]);
    vs[u] = __builtin_bit_cast(uint2, load_at<u32x2>(a.vs + p.sat[u], o.vs));
  }
};

// Q's parts as A operands, kT groups of 4 query heads: lane l holds, of row l % 16 = 4 head + part, dims 16 g .. + 15 and 64 + 16 g ..
// + 15, and the exponent byte of block g.  plain: some block's elements differ too much for the parts, or are not finite.
template <int kT>
struct Query {
  i32x8_t v[kT];
  uint32_t s[kT];
  bool plain;
};

template <int kT, int kW>
struct Lds {
  static constexpr int kRows = 4 * kT;                         // query heads
  alignas(16) uint8_t q[16 * kT][kQRow];
  uint8_t qs[16 * kT][4];
  alignas(16) uint8_t p[kW][2 * kRows][kPRow];
  float m[kW][kRows], l[kW][kRows];
  alignas(16) uint8_t own[2][kFp4Row];                         // the append form's new row, of one wave: codes of K and V,
  uint8_t own_s[2][kFp4Blocks];                                // and their exponent bytes
  int plain;
};

// Splits Q.  A bf16 number has 8 significant bits, e4m3 4 of them between 2^-6 and 2^8 (and multiples of 2^-9 below).  In a block whose
// largest element lies in [2^7, 2^8) after its scaling, elements of at least 2^-6 are the sum of their upper 4 bits (part 0) and the
// lower 4, which times 2^4 are e4m3 numbers too (part 1); those 2^14 times smaller are in parts 2 and 3 likewise.  Elements that are
// smaller still by 2^28 and more than the largest one have no part (`plain`: one in 10^8 of normal ones).  So the parts hold Q exactly.
// Each of the workgroup's first four waves makes one part of all rows.
template <int kT, int kW>
__device__ __forceinline__ void prepare_q(uint32_t sign, const uint4 (&x)[kT], int wave, Lds<kT, kW>& lds, Query<kT>& q) {
  const int lane = lane_now(), part = wave & 3;
  uint32_t bad = 0;
  if (wave < 4) {
#pragma unroll
    for (int t = 0; t < kT; ++t) {
      const uint32_t e[4] = {x[t].x ^ sign, x[t].y ^ sign, x[t].z ^ sign, x[t].w ^ sign};
      uint32_t top = dpp_max_u32<kDppXor2>(dpp_max_u32<kDppXor1>(halves_max(bf16_any_amax_pair(e))));  // of the block's four lanes
      const int x7 = (int)(top >> 7);
      const uint32_t least = (uint32_t)max(0, x7 - 27) << 7, large = (uint32_t)max(0, x7 - 13) << 7;
      bad |= (top >= 0x7f80u || (top != 0 && x7 < 28)) ? 1u : 0u;
      const uint32_t field = top == 0 ? 127u : (uint32_t)(x7 - 7 - (part == 0 ? 0 : part == 1 ? 4 : part == 2 ? 14 : 18));
      const float scale = __uint_as_float((field & 0xffu) << 23);
      s16x2 c[2] = {{0, 0}, {0, 0}};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float f[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t b = k == 0 ? e[i] & 0xffffu : e[i] >> 16, mag = b & 0x7fffu;
          bad |= (mag != 0 && mag < least) ? 1u : 0u;
          const bool here = (mag >= large) == (part < 2);
          const float whole = __uint_as_float(b << 16), upper = __uint_as_float((b & 0xfff0u) << 16);
          f[k] = here ? ((part & 1) != 0 ? whole - upper : upper) : 0.f;
        }
        if (i & 1) c[i >> 1] = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c[i >> 1], f[0], f[1], scale, true);
        else c[i >> 1] = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c[i >> 1], f[0], f[1], scale, false);
      }
      const int row = 16 * t + 4 * (lane >> 4) + part, seg = lane & 15;
      *reinterpret_cast<u32x2*>(&lds.q[row][8 * seg]) = u32x2{__builtin_bit_cast(uint32_t, c[0]), __builtin_bit_cast(uint32_t, c[1])};
      if ((seg & 3) == 0) lds.qs[row][seg >> 2] = (uint8_t)field;
    }
    const bool any = __builtin_amdgcn_ballot_w64(bad != 0) != 0;
    if (wave == 0 && lane == 0) lds.plain = any ? 1 : 0;
  }
  __syncthreads();
  q.plain = __builtin_amdgcn_readfirstlane(lds.plain) != 0;
  const int r = lane & 15, g = lane >> 4;
#pragma unroll
  for (int t = 0; t < kT; ++t) {
    const i32x4_t lo = *reinterpret_cast<const i32x4_t*>(&lds.q[16 * t + r][16 * g]);
    const i32x4_t hi = *reinterpret_cast<const i32x4_t*>(&lds.q[16 * t + r][64 + 16 * g]);
    q.v[t] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    q.s[t] = lds.qs[16 * t + r][g];
  }
}

// The row of Q that a lane's head is: the last one again past it.
__device__ __forceinline__ const uint16_t* q_row(const TreeArgs& a, int b, int h, int head) {
  return a.q + (int64_t)b * a.q_sb + (int64_t)(h * a.group + min(head, a.group - 1)) * a.q_sh;
}

// The parts' sum.
__device__ __forceinline__ float sum_parts(const f32x4_t d) { return (d[0] + d[1]) + (d[2] + d[3]); }

// A subtile's scores where Q has no parts: codes converted to bf16, Q read again, in the rows of part 0.  (Piece by piece, to hold few
// registers: what the loop has in flight stays in its own.)
template <int kT>
__device__ __forceinline__ void plain_scores(const Work& w, const uint4& k, uint32_t ks, f32x4_t (&d)[kT]) {
  const uint32_t k4[4] = {k.x, k.y, k.z, k.w};
  const float f = fp8_scale(ks);
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int t = 0; t < kT; ++t) {
      const int lane = lane_now(), r = lane & 15, g = lane >> 4;
      const uint32_t sign = args_again().q_sign;
      uint4 x = ld16(q_row(args_again(), w.b, w.h, 4 * t + (r >> 2)) + 32 * g + 8 * c);
      x = make_uint4(nan_if_not_finite(x.x ^ sign), nan_if_not_finite(x.y ^ sign), nan_if_not_finite(x.z ^ sign),
                     nan_if_not_finite(x.w ^ sign));
      if ((r & 3) != 0) x = make_uint4(0u, 0u, 0u, 0u);
      const bf16x8_t kf = __builtin_bit_cast(
          bf16x8_t, make_uint4(fp4_pair<0>(k4[c], f), fp4_pair<1>(k4[c], f), fp4_pair<2>(k4[c], f), fp4_pair<3>(k4[c], f)));
      const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
      d[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, x), kf, c == 0 ? zero : d[t], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
}

template <int kT>
struct State {
  f32x4_t o[kT][4];        // MFMA j, of head 4 t + g: dims 8 (l % 16) + 2 j, + 1 by the probabilities' first numbers, then by the second
  float m[kT], l[kT];      // of head 4 t + g: the exponents' base, unscaled; sum, of this lane's keys until the merge
};

// Two products of Q's parts and 16 keys' codes (u0, u1: exponent bytes), and the wait for them.
//
// The compiler counts the passes of the scaled instruction as if both operands had 4 bits: 8 wait states ahead of the result's first use
// instead of the 12 that an 8-bit operand takes, and the register that was read first then held something else.  So the wait is ours, 16
// states behind the second product, in one statement with them: nothing that the compiler adds, a copy or a move to another register, can
// come between.  (The 2 states ahead are what operands want that a vector instruction wrote last.)
__device__ __forceinline__ void two_products(const i32x8_t& q0, uint32_t s0, const i32x8_t& q1, uint32_t s1, const uint4& k0, uint32_t u0,
                                             const uint4& k1, uint32_t u1, f32x4_t& d0, f32x4_t& d1) {
  asm volatile(
      "s_nop 1\n\t"
      "v_mfma_scale_f32_16x16x128_f8f6f4 %0, %2, %4, 0, %6, %8 op_sel_hi:[0,0,0] blgp:4\n\t"
      "v_mfma_scale_f32_16x16x128_f8f6f4 %1, %3, %5, 0, %7, %9 op_sel_hi:[0,0,0] blgp:4\n\t"
      "s_nop 15"
      : "=&v"(d0), "=&v"(d1)
      : "v"(q0), "v"(q1), "v"(__builtin_bit_cast(i32x4_t, k0)), "v"(__builtin_bit_cast(i32x4_t, k1)), "v"(s0), "v"(s1), "v"(u0), "v"(u1));
}

// A step's scores.
template <int kT>
__device__ __forceinline__ void scores(const Work& w, const uint4 (&codes)[kSub], const uint32_t (&four)[kSub], const Query<kT>& q, int lane,
                                       float (&s)[kT][kSub]) {
  uint32_t ks[kSub];  // the exponent byte lowest: only that counts
#pragma unroll
  for (int u = 0; u < kSub; ++u) ks[u] = four[u] >> (8 * (lane & 3));
  if (__builtin_expect(q.plain, 0)) {
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      f32x4_t d[kT];
      plain_scores<kT>(w, codes[u], ks[u] & 0xffu, d);
#pragma unroll
      for (int t = 0; t < kT; ++t) s[t][u] = sum_parts(d[t]);
    }
    return;
  }
  constexpr int kAtOnce = kT == 1 ? 2 : 1;  // (as registers allow)
#pragma unroll
  for (int u0 = 0; u0 < kSub; u0 += kAtOnce) {
    f32x4_t d[2];
    constexpr int t1 = kT - 1;
    const int u1 = u0 + kAtOnce - 1;
    two_products(q.v[0], q.s[0], q.v[t1], q.s[t1], codes[u0], ks[u0], codes[u1], ks[u1], d[0], d[1]);
#pragma unroll
    for (int e = 0; e < 2; ++e) s[kT == 1 ? 0 : e][kT == 1 ? u0 + e : u0] = sum_parts(d[e]);
  }
}

template <int kCtrl>
__device__ __forceinline__ float dpp_max(float x) { return fmaxf(x, dpp_f32<kCtrl>(x)); }

// The scores to probabilities, in s; the base (as tree_decode.hip's softmax has it) and the sum are updated and O rescaled.
template <int kT>
__device__ __forceinline__ void softmax(const Place& at, float scale, float ahead, float (&s)[kT][kSub], State<kT>& st) {
  if (__builtin_expect(at.full == 0, 0)) {
    const int r = lane_now() & 15;
#pragma unroll
    for (int t = 0; t < kT; ++t)
#pragma unroll
      for (int u = 0; u < kSub; ++u) s[t][u] = r < at.valid[u] ? s[t][u] : -INFINITY;
  }
  float top[kT];
  bool grown = false;
#pragma unroll
  for (int t = 0; t < kT; ++t) {
    top[t] = larger(larger(s[t][0], s[t][1]), larger(s[t][2], s[t][3]));
    grown = grown | (top[t] > st.m[t]);
  }
  if (__builtin_amdgcn_ballot_w64(grown) != 0) {
#pragma unroll
    for (int t = 0; t < kT; ++t) {
      const float all = dpp_max<kDppMirror>(dpp_max<kDppHalfMirror>(dpp_max<kDppXor2>(dpp_max<kDppXor1>(top[t]))));
      const float m = all > st.m[t] ? all + ahead : st.m[t];
      const float alpha = fast_exp2((st.m[t] - (m == -INFINITY ? 0.f : m)) * scale);
      st.m[t] = m;
      st.l[t] *= alpha;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) st.o[t][j][i] *= alpha;
    }
  }
#pragma unroll
  for (int t = 0; t < kT; ++t) {
    const float base = st.m[t] == -INFINITY ? 0.f : st.m[t] * scale;
#pragma unroll
    for (int u = 0; u < kSub; ++u) s[t][u] = fast_exp2(__builtin_fmaf(s[t][u], scale, -base));
    st.l[t] += (s[t][0] + s[t][1]) + (s[t][2] + s[t][3]);
  }
}

__device__ __forceinline__ uint32_t pair_at(uint32_t w, int byte, float f) {
  return byte == 0 ? fp4_pair<0>(w, f) : byte == 1 ? fp4_pair<1>(w, f) : byte == 2 ? fp4_pair<2>(w, f) : fp4_pair<3>(w, f);
}

// Between a wave's writes to its LDS and its reads of them by other lanes.  A wave's LDS operations run in order: only the compiler has to
// keep them so.
__device__ __forceinline__ void in_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// The probabilities as two bf16 numbers into the wave's LDS, a row each.  A row has its 64 keys as the operands want them: of a quarter's
// 16 keys (32 bytes) each i's first two subtiles, then each i's other two.
template <int kT>
__device__ __forceinline__ void store_p(const float (&p)[kT][kSub], int lane, uint8_t (*lds)[kPRow]) {
  const int r = lane & 15, g = lane >> 4;
  const int i = (r >> 1) & 3, quarter = 2 * (r >> 3) + (r & 1), pos = 32 * quarter + 4 * i;
#pragma unroll
  for (int t = 0; t < kT; ++t) {
#pragma unroll
    for (int u = 0; u < kSub; u += 2) {
      const uint32_t hi = pack_bf16x2(p[t][u], p[t][u + 1]);
      *reinterpret_cast<uint32_t*>(&lds[8 * t + 2 * g][pos + 8 * u]) = hi;
      *reinterpret_cast<uint32_t*>(&lds[8 * t + 2 * g + 1][pos + 8 * u]) = pack_bf16x2(p[t][u] - bf16_lo(hi), p[t][u + 1] - bf16_hi(hi));
    }
  }
  in_order();
}

// Operands of P: lane l has row l % 16 = 4 head + 2 number + dim, whose pairs are (p, 0) or (0, p).
struct Pairs {
  uint32_t of[2];  // byte selectors: of a dword's lower half, of its upper one
};
__device__ __forceinline__ Pairs pairs_of(int lane) {
  return (lane & 1) != 0 ? Pairs{{0x01000c0cu, 0x03020c0cu}} : Pairs{{0x0c0c0100u, 0x0c0c0302u}};
}

// O += P V, `then` behind each subtile's.
template <int kT, class Then>
__device__ __forceinline__ void values(const Tile& x, const Place& at, const float (&p)[kT][kSub], int lane, uint8_t (*lds)[kPRow],
                                       State<kT>& st, Then&& then) {
  const int r = lane & 15, g = lane >> 4;
  store_p<kT>(p, lane, lds);
  uint2 vs[kSub];
#pragma unroll
  for (int u = 0; u < kSub; ++u) vs[u] = x.vs[u];
  if (__builtin_expect(at.full == 0, 0)) {  // the exponent byte of a key that is not seen may be anything
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      // (on the scalar unit, for the tokens 0 .. 7 and 8 .. 15)
      const uint64_t lo = at.valid[u] >= 8 ? ~0ull : (1ull << (8 * at.valid[u])) - 1;
      const uint64_t hi = at.valid[u] >= 16 ? ~0ull : (1ull << (8 * max(0, at.valid[u] - 8))) - 1;
      vs[u].x &= (g & 2) != 0 ? (uint32_t)hi : (uint32_t)lo;
      vs[u].y &= (g & 2) != 0 ? (uint32_t)(hi >> 32) : (uint32_t)(lo >> 32);
    }
  }
  // The lane's keys are every second one of 8: bytes 0 and 2, or 1 and 3, of both dwords.  Only the exponent's bits of a scale count (all
  // 256 of them were compared with other bits and signs around them), so a byte is brought there by one shift.
  const int left = (g & 1) != 0 ? 15 : 23, around = (g & 1) != 0 ? 1 : 25;
  const Pairs pairs = pairs_of(lane);
  uint4 two[kT];  // P of two subtiles
#pragma unroll
  for (int u = 0; u < kSub; ++u) {
    if ((u & 1) == 0) {
#pragma unroll
      for (int t = 0; t < kT; ++t) two[t] = ld16(lds[8 * t + (r >> 1)] + 32 * g + 8 * u);
    }
    const float f[4] = {__uint_as_float(vs[u].x << left), __uint_as_float(__builtin_amdgcn_alignbit(vs[u].x, vs[u].x, around)),
                        __uint_as_float(vs[u].y << left), __uint_as_float(__builtin_amdgcn_alignbit(vs[u].y, vs[u].y, around))};
    bf16x8_t a[kT];
#pragma unroll
    for (int t = 0; t < kT; ++t) {
      const uint32_t by = pairs.of[u & 1];
      a[t] = __builtin_bit_cast(bf16x8_t, make_uint4(perm_b32(0u, two[t].x, by), perm_b32(0u, two[t].y, by), perm_b32(0u, two[t].z, by),
                                                     perm_b32(0u, two[t].w, by)));
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bf16x8_t b = __builtin_bit_cast(bf16x8_t, make_uint4(pair_at(x.v[u][0], j, f[0]), pair_at(x.v[u][1], j, f[1]),
                                                                 pair_at(x.v[u][2], j, f[2]), pair_at(x.v[u][3], j, f[3])));
#pragma unroll
      for (int t = 0; t < kT; ++t) st.o[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[t], b, st.o[t][j], 0, 0, 0);
    }
    then(u);
  }
}

// The append form's new row, quantised as the write kernel does, into LDS: lane l has 8 dims from 8 (l % 16) of K (l & 16: of V).
template <int kT, int kW>
__device__ __forceinline__ void quantise_own(const uint4& x, Lds<kT, kW>& lds) {
  const int lane = lane_now() & 31, r = lane & 15;  // (lanes from 32 on write the same again)
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  const uint32_t s = fp4_scale_byte(dpp_max_u32<kDppXor2>(dpp_max_u32<kDppXor1>(halves_max(bf16_any_amax_pair(w)))));
  *reinterpret_cast<uint32_t*>(&lds.own[lane >> 4][4 * r]) = fp4_codes8(w[0], w[1], w[2], w[3], s);
  lds.own_s[lane >> 4][r >> 2] = (uint8_t)s;
  in_order();
}
// And into the pool, if `page` is one of it.
template <int kT, int kW>
__device__ __forceinline__ void store_own(int h, int page, int off, const Lds<kT, kW>& lds) {
  const TreeArgs& a = args_again();
  const int lane = lane_now(), r = lane & 15, v = (lane >> 4) & 1;
  if (lane < 32 && (unsigned)page < (unsigned)a.num_pages) {
    const int64_t at = (int64_t)page * a.sp + (int64_t)h * a.sh + (int64_t)off * a.st + 4 * r;
    const int64_t sat = (int64_t)page * a.ss_p + (int64_t)h * a.ss_h + off + (r >> 2) * a.page_size;
    *reinterpret_cast<uint32_t*>((v ? a.vc : a.kc) + at) = *reinterpret_cast<const uint32_t*>(&lds.own[v][4 * r]);
    if ((r & 3) == 0) (v ? a.vs : a.ks)[sat] = lds.own_s[v][r >> 2];
  }
}

// The new row in a step's registers: key `at` of it, the same on every lane.  (The empty statements keep the branches on it apart: else they
// become an index into registers.)
template <int kT, int kW>
__device__ __forceinline__ void own_key(Tile& x, int at, const Lds<kT, kW>& lds) {
  const int lane = lane_now(), r = lane & 15, g = lane >> 4;
  const uint4 c = ld16(&lds.own[0][16 * g]);
  const uint32_t s = (uint32_t)lds.own_s[0][g] << (8 * (lane & 3));
  const bool here = r == (at & 15);
#pragma unroll
  for (int u = 0; u < kSub; ++u)
    if (u == at >> 4) {
      asm volatile("" : "+v"(x.ks[u]));
      x.k[u] = make_uint4(here ? c.x : x.k[u].x, here ? c.y : x.k[u].y, here ? c.z : x.k[u].z, here ? c.w : x.k[u].w);
      x.ks[u] = here ? s : x.ks[u];
    }
}
template <int kT, int kW>
__device__ __forceinline__ void own_value(Tile& x, int at, const Lds<kT, kW>& lds) {
  const int lane = lane_now(), r = lane & 15, g = lane >> 4;
  const uint32_t c = *reinterpret_cast<const uint32_t*>(&lds.own[1][4 * r]), shift = 8 * (at & 3);
  const uint32_t s = (uint32_t)lds.own_s[1][r >> 2] << shift, others = ~(0xffu << shift);
  const int key = at & 15;
  const bool here = g == 2 * (key >> 3) + (key & 1), half = (g >> 1) == key >> 3;
#pragma unroll
  for (int u = 0; u < kSub; ++u)
    if (u == at >> 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i == ((key >> 1) & 3)) {
          asm volatile("" : "+v"(x.v[u][i]));
          x.v[u][i] = here ? c : x.v[u][i];
        }
      if ((key & 4) == 0) x.vs[u].x = half ? (x.vs[u].x & others) | s : x.vs[u].x;
      else x.vs[u].y = half ? (x.vs[u].y & others) | s : x.vs[u].y;
    }
}

// Merges the waves' states into the output (rec == nullptr) or a record of (o[128], m, l) floats a query head.
template <int kT, int kW>
__device__ __forceinline__ void merge_waves(const Work& w, const State<kT>& st, float* rec, int wave, float (*so)[4 * kT][kD + 4],
                                            Lds<kT, kW>& lds) {
  const int lane = lane_now(), thread = 64 * wave + lane, r = lane & 15, g = lane >> 4;
  const float scale = args_again().scale_log2;
#pragma unroll
  for (int t = 0; t < kT; ++t) {
    const float l = row16_sum(st.l[t]);
    if (r == 0) {
      lds.m[wave][4 * t + g] = st.m[t] * scale;
      lds.l[wave][4 * t + g] = l;
    }
  }
#pragma unroll
  for (int t = 0; t < kT; ++t) {
    float* to = &so[wave][4 * t + g][8 * r];
#pragma unroll
    for (int j = 0; j < 4; j += 2)
      *reinterpret_cast<f32x4_t*>(to + 2 * j) = f32x4_t{st.o[t][j][0] + st.o[t][j][2], st.o[t][j][1] + st.o[t][j][3],
                                                        st.o[t][j + 1][0] + st.o[t][j + 1][2], st.o[t][j + 1][1] + st.o[t][j + 1][3]};
  }
  __syncthreads();
  constexpr int kDims = kT == 2 && kW == 4 ? 4 : 2;  // a thread
  const int row = thread / (kD / kDims), d0 = kDims * (thread % (kD / kDims));
  if (row >= args_again().M) return;  // at most 4 kT rows
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kW; ++i) top = fmaxf(top, lds.m[i][row]);
  const float base = top == -INFINITY ? 0.f : top;
  float acc[kDims] = {}, sum = 0.f;
#pragma unroll
  for (int i = 0; i < kW; ++i) {
    const float f = fast_exp2(lds.m[i][row] - base);
    sum += f * lds.l[i][row];
#pragma unroll
    for (int d = 0; d < kDims; ++d) acc[d] += f * so[i][row][d0 + d];
  }
  if (rec == nullptr) {
    uint16_t* op = out_row(w.b, w.h, row) + d0;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int d = 0; d < kDims; d += 2) *reinterpret_cast<uint32_t*>(op + d) = pack_bf16x2(acc[d] * inv, acc[d + 1] * inv);
  } else {
    float* o = rec + row * kRecord;
    if (d0 == 0) *reinterpret_cast<float2*>(o + kD) = make_float2(top, sum);
#pragma unroll
    for (int d = 0; d < kDims; d += 2) *reinterpret_cast<float2*>(o + d0 + d) = make_float2(acc[d], acc[d + 1]);
  }
}

// The pool places of a wave's next kWindow steps, one subtile a lane (4 slot + u), worked out by the lanes at once.
struct Window4 {
  uint32_t at, sat;   // offset of the first key in 16 bytes, and of its exponent byte
  int tok, valid;     // its token; the keys that are seen
  bool page;          // the table has a page for it
  uint64_t whole;     // lanes with all 16 keys
};

// One workgroup a (row, KV head), its kW waves taking the row's steps in turn; or (kChunked) one of a chunk of a row's steps, which
// leaves a record for the join unless it is the row's only one.
template <int kMode, int kT, int kW, bool kChunked, bool kOnce>
__global__ __launch_bounds__(64 * kW, kT == 1 ? 4 : 3) void fp4_decode_kernel(const TreeArgs args) {
  __shared__ Lds<kT, kW> lds;
  __shared__ __align__(16) float s_o[kW][4 * kT][kD + 4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Work w;
  int unit;
  unit_of(args, w.h, w.mb, unit);
  if (unit >= args.units) return;
  uint4 raw[kT], own;
  auto load_q = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < kT; ++t) raw[t] = ld16(q_row(args, w.b, w.h, 4 * t + (lane >> 4)) + 8 * (lane & 15));
  };
  Window4 win;
  int id, off;   // on the way: the lane's table entry, and its token's place in the page
  auto look_up = [&](const TreeArgs& a, int step) __attribute__((always_inline)) {
    win.tok = kStep * step + 16 * (lane_now() & (kSub - 1));
    const int pi = (int)divide((uint32_t)win.tok, a.per_page);
    off = win.tok - pi * a.page_size;
    id = -1;
    if (pi < a.max_pages) id = a.bt[(int64_t)w.b * a.bt_sb + pi];
  };
  auto find = [&](const TreeArgs& a) __attribute__((always_inline)) {
    win.page = (unsigned)id < (unsigned)a.num_pages;
    const int page = win.page ? id : 0, in = win.page ? off : 0;
    win.at = (uint32_t)(((int64_t)page * a.sp + (int64_t)in * a.st) >> 4);
    win.sat = (uint32_t)(page * a.ss_p + in);
  };
  auto see = [&](int limit) __attribute__((always_inline)) {
    win.valid = win.page ? max(0, min(16, limit - win.tok)) : 0;
    win.whole = __builtin_amdgcn_ballot_w64(win.valid == 16);
  };
  int s0 = 0, s1;  // the chunk's steps: of whole rows all Tc
  float* rec = nullptr;
  if constexpr (kChunked) {
    const Chunk c = chunk_at<kStep * kW>(args, (uint32_t)unit, kMode);
    if (c.row < 0) return;
    w.b = c.row;
    w.L = c.L;
    w.Tc = w.L > 0 ? (w.L + kStep - 1) / kStep : 0;
    const int steps = (int)((rounds_of<kStep * kW>(args, w.L, kMode) + c.count - 1) / c.count) * kW;
    s0 = min(w.Tc, c.index * steps);
    s1 = min(w.Tc, s0 + steps);
    look_up(args, s0 + wave + kW * (lane >> 2));
    load_q();
    if (c.count > 1) rec = args.rec + ((int64_t)unit * args.hkv + w.h) * (int64_t)(args.rec_rows * kRecord);
    if (c.index == 0 && w.h == 0 && threadIdx.x == 0) reinterpret_cast<Joined*>(args.ws)[w.b] = Joined{unit - c.index, c.count};
    find(args);
  } else {
    w.b = unit;
    if constexpr (kW == 4) {
      const int row0 = max(0, args.batch - 64 * kW);
      if (args.order && unit >= row0) w.b = kth_longest<kW>(args, row0, unit - row0, wave);
    }
    const int tokens = args.seqlens[w.b], cap = args.max_pages * args.page_size;
    // The first window's page ids do not wait for the row's length.
    look_up(args, wave + kW * (lane >> 2));
    load_q();
    find(args);
    w.L = __builtin_amdgcn_readfirstlane(kMode == kAppendKey ? (tokens >= 0 && tokens < cap ? tokens + 1 : -1) : min(tokens, cap));
    w.Tc = w.L > 0 ? (w.L + kStep - 1) / kStep : 0;
    s1 = w.Tc;
  }
  if (s1 == 0 && rec == nullptr) {
    zero_rows(w.b, w.h, w.mb, 16);
    return;
  }
  const int first = s0 + wave, limit = min(w.L, kStep * s1);
  const int n = max(0, (s1 - first + kW - 1) / kW);  // this wave's steps: first, first + kW, ...
  see(limit);
  // The append form's new row is key w.L - 1, in the last of all steps: the wave that has that one quantises it.
  const bool has_own = kMode == kAppendKey && n > 0 && first + kW * (n - 1) == w.Tc - 1;
  const int own_at = has_own ? w.L - 1 - kStep * (w.Tc - 1) : -1;
  int own_page = -1, own_off = 0;
  if (has_own) {
    const int pi = (int)divide((uint32_t)(w.L - 1), args.per_page);
    own_off = w.L - 1 - pi * args.page_size;
    own = ld16((lane & 16) != 0 ? args.vn + (int64_t)w.b * args.vn_sb + (int64_t)w.h * args.vn_sh + 8 * (lane & 15)
                                : args.kn + (int64_t)w.b * args.kn_sb + (int64_t)w.h * args.kn_sh + 8 * (lane & 15));
    own_page = args.bt[(int64_t)w.b * args.bt_sb + pi];
  }
  auto place = [&](int j) __attribute__((always_inline)) {
    if ((j & (kWindow - 1)) == 0 && j > 0) {
      const TreeArgs& a = args_again();
      look_up(a, first + kW * (j + (lane_now() >> 2)));
      find(a);
      see(limit);
    }
    const int slot = kSub * (j & (kWindow - 1));
    Place p;
    p.full = ((win.whole >> slot) & 15) == 15 ? 1 : 0;
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      p.at[u] = (int64_t)(uint32_t)readlane((int)win.at, slot + u) << 4;
      p.sat[u] = (uint32_t)readlane((int)win.sat, slot + u);
      p.valid[u] = 16;
    }
    if (__builtin_expect(p.full == 0, 0)) {
#pragma unroll
      for (int u = 0; u < kSub; ++u) p.valid[u] = readlane(win.valid, slot + u);
    }
    return p;
  };
  const Pool pool = pool_of(args, w.h);
  const Offsets offsets = offsets_of(pool, lane);
  Tile x;  // (loaded without a branch, also by a wave without steps: only so can what was asked for before be waited for alone)
  Place at = place(0);
#pragma unroll
  for (int u = 0; u < kSub; ++u) x.load_k<kOnce>(pool, at, u, offsets);
#pragma unroll
  for (int u = 0; u < kSub; ++u) x.load_v<kOnce>(pool, at, u, offsets);
  Query<kT> q;
  prepare_q<kT, kW>(args.q_sign, raw, wave, lds, q);
  if (has_own) {
    quantise_own<kT, kW>(own, lds);
    store_own<kT, kW>(w.h, own_page, own_off, lds);  // (early: a workgroup lasts until its stores are done)
  }
  State<kT> st;
#pragma unroll
  for (int t = 0; t < kT; ++t) {
    st.m[t] = -INFINITY;
    st.l[t] = 0.f;
  }
#pragma unroll
  for (int t = 0; t < kT; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) st.o[t][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const float scale = args.scale_log2, ahead = args.ahead;
  auto step = [&](int i, auto more) __attribute__((always_inline)) {
    Place next = at;
    if constexpr (decltype(more)::value) next = place(i + 1);
    float s[kT][kSub];
    if (kMode == kAppendKey && !decltype(more)::value && has_own) own_key<kT, kW>(x, own_at, lds);
    scores<kT>(w, x.k, x.ks, q, lane, s);
    if constexpr (decltype(more)::value) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < kSub; ++u) x.load_k<kOnce>(pool, next, u, offsets);
      __builtin_amdgcn_sched_barrier(0);
    }
    softmax<kT>(at, scale, ahead, s, st);
    if (kMode == kAppendKey && !decltype(more)::value && has_own) own_value<kT, kW>(x, own_at, lds);
    values<kT>(x, at, s, lane, lds.p[wave], st, [&](int u) __attribute__((always_inline)) {
      if constexpr (decltype(more)::value) {
        __builtin_amdgcn_sched_barrier(0);
        x.load_v<kOnce>(pool, next, u, offsets);
        __builtin_amdgcn_sched_barrier(0);
      }
    });
    at = next;
  };
  // The last step by itself: with branches around the loads the compiler would not know how many of them are newer than those that it
  // waits for, and wait for all.
  for (int i = 0; i < n - 1; ++i) step(i, std::true_type{});
  if (n > 0) step(n - 1, std::false_type{});
  merge_waves<kT, kW>(w, st, rec, wave, s_o, lds);
}

template <int kMode, int kT, int kW, bool kChunked>
void launch(const TreeArgs& a, dim3 grid, hipStream_t stream) {
  if (a.st == kFp4Row) hipLaunchKernelGGL((fp4_decode_kernel<kMode, kT, kW, kChunked, true>), grid, dim3(64 * kW), 0, stream, a);
  else hipLaunchKernelGGL((fp4_decode_kernel<kMode, kT, kW, kChunked, false>), grid, dim3(64 * kW), 0, stream, a);
}
// Four waves a workgroup.  Eight for chunks of 5 to 8 query heads, whose registers leave room for 12 waves on a compute unit: one workgroup
// of eight does as much as three of four with a third of the records (5 rows of 20000 to 65000 tokens 23.0 us in the kernel; two of four
// 26.4, three 24.0).
// Eight also for whole rows that leave each compute unit one workgroup at most.  More rows lose by it where they are ragged or have 5 to 8
// query heads to a KV head, for what a wave does once for its row is as long as two steps.  A call's us with the step's write, 8 KV heads,
// with eight waves and with four:
//   2 query heads each   1 x 1500 tokens 8.9 and 10.5, 16 x 1000 8.4 and 8.9, 24 x 1500 10.1 and 10.9, 24 x 188 to 1500 9.6 and 10.7,
//                        32 x 2000 12.9 and 13.1; past the limit 33 x 1000 11.2 and 11.4, 33 x 2000 17.8 and 18.7, 33 x 100 to 1500
//                        11.9 and 11.1, 64 x 1000 13.6 and 13.5, 64 x 2000 23.4 and 23.9, 100 x 100 to 1500 21.3 and 18.2
//   8 query heads each   1 x 1500 11.1 and 12.9, 32 x 2000 14.5 and 15.9; past the limit 33 x 1000 17.1 and 13.7, 64 x 2000 29.2 and 26.9
template <int kMode, int kT>
void launch(const TreeArgs& a, dim3 grid, hipStream_t stream) {
  const int groups = a.batch * a.hkv;
  if (a.target > 0) launch<kMode, kT, kT == 1 ? 4 : 8, true>(a, grid, stream);
  else if (groups <= num_cus()) launch<kMode, kT, 8, false>(a, grid, stream);
  else launch<kMode, kT, 4, false>(a, grid, stream);
}

}  // namespace

hipError_t launch_fp4_decode(const TreeArgs& args, int mode, dim3 grid, hipStream_t stream) {
  TreeArgs a = args;
  if (a.num_pages == 0) a.max_pages = 0;  // no row has a token: the kernel loads some page's codes for every step
  if (a.group <= 4) {
    if (mode == kAppend) launch<kAppendKey, 1>(a, grid, stream);
    else launch<kNoKeys, 1>(a, grid, stream);
  } else {
    if (mode == kAppend) launch<kAppendKey, 2>(a, grid, stream);
    else launch<kNoKeys, 2>(a, grid, stream);
  }
  return hipGetLastError();
}

}  // namespace q3a
