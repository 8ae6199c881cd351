// Decode attention over the 4-bit K/V pool with up to 8 query heads to a KV head (gfx950).  (More than 8 take tree_decode.hip's
// kernel, which converts 4-bit keys to bf16.)
//
// At 136 bytes a token and KV head the pool's keys pass at four times the rate of bf16 ones, and what bounds the general kernel over
// them is vector instructions: 16 query rows' worth of softmax for 2, and a conversion for every pair of codes.  Here a wave's step is
// 64 keys (four 16-token subtiles u, each inside one page), and:
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

struct Tile {
  uint4 k[kSub];            // block g of key l % 16
  uint32_t ks[kSub];        // its exponent byte
  uint32_t v[kSub][4];      // dims 8 (l % 16) .. + 7 of keys key_of(g, 0 .. 3)
  uint2 vs[kSub];           // their block's exponent bytes of keys 8 (g / 2) .. + 7
  int valid[kSub];          // keys that are seen

  __device__ __forceinline__ static __amdgpu_buffer_rsrc_t codes(const TreeArgs& a, const uint8_t* base, int valid) {
    // Descriptors end with the last seen key: what lies past it is not read and comes as zeros.
    return make_rsrc(base, valid > 0 ? (uint32_t)(valid - 1) * (uint32_t)a.st + kFp4Row : 0u);
  }
  __device__ __forceinline__ static __amdgpu_buffer_rsrc_t exps(const TreeArgs& a, const uint8_t* base, int valid) {
    return make_rsrc(base, valid > 0 ? (kFp4Blocks - 1) * a.page_size + 16 : 0);
  }
  __device__ __forceinline__ void load_k(const TreeArgs& a, const int64_t (&at)[kSub], const uint32_t (&sat)[kSub],
                                         const int (&seen)[kSub], int lane) {
    const int r = lane & 15, g = lane >> 4;
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      k[u] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(codes(a, a.kc + at[u], seen[u]), r * a.st + 16 * g, 0, kNt));
      ks[u] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(exps(a, a.ks + sat[u], seen[u]), g * a.page_size + r, 0, 0);
    }
  }
  __device__ __forceinline__ void load_v(const TreeArgs& a, const int64_t (&at)[kSub], const uint32_t (&sat)[kSub],
                                         const int (&seen)[kSub], int lane) {
    const int r = lane & 15, g = lane >> 4;
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      const auto rv = codes(a, a.vc + at[u], seen[u]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[u][i] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rv, key_of(g, i) * a.st + 4 * r, 0, kNt);
      vs[u] = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(exps(a, a.vs + sat[u], seen[u]),
                                                                             (r >> 2) * a.page_size + 8 * (g >> 1), 0, 0));
      valid[u] = seen[u];
    }
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
};

// Splits Q.  A bf16 number has 8 significant bits, e4m3 4 of them between 2^-6 and 2^8 (and multiples of 2^-9 below).  In a block whose
// largest element lies in [2^7, 2^8) after its scaling, elements of at least 2^-6 are the sum of their upper 4 bits (part 0) and the
// lower 4, which times 2^4 are e4m3 numbers too (part 1); those 2^14 times smaller are in parts 2 and 3 likewise.  Elements that are
// smaller still by 2^28 and more than the largest one have no part (`plain`: one in 10^8 of normal ones).  So the parts hold Q exactly.
// Each of the workgroup's first four waves makes one part of all rows; every wave looks at all elements.
template <int kT, int kW>
__device__ __forceinline__ void prepare_q(const Work& w, const uint4 (&x)[kT], int wave, Lds<kT, kW>& lds, Query<kT>& q) {
  const int lane = lane_now(), part = wave & 3;
  const uint32_t sign = args_again().q_sign;
  uint32_t bad = 0;
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
    if (wave < 4) {
      const int row = 16 * t + 4 * (lane >> 4) + part, seg = lane & 15;
      *reinterpret_cast<u32x2*>(&lds.q[row][8 * seg]) = u32x2{__builtin_bit_cast(uint32_t, c[0]), __builtin_bit_cast(uint32_t, c[1])};
      if ((seg & 3) == 0) lds.qs[row][seg >> 2] = (uint8_t)field;
    }
  }
  q.plain = __builtin_amdgcn_ballot_w64(bad != 0) != 0;
  __syncthreads();
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
__device__ __forceinline__ const uint16_t* q_row(const Work& w, int head) {
  const TreeArgs& a = args_again();
  return a.q + (int64_t)w.b * a.q_sb + (int64_t)(w.h * a.group + min(head, a.group - 1)) * a.q_sh;
}

__device__ __forceinline__ float sum_parts(const f32x4_t d) { return (d[0] + d[1]) + (d[2] + d[3]); }

// A subtile's scores where Q has no parts: codes converted to bf16, Q read again, in the rows of part 0.  (A loop, to be short.)
template <int kT>
__device__ __forceinline__ void plain_scores(const Work& w, uint4 k, uint32_t ks, f32x4_t (&d)[kT]) {
  const int lane = lane_now(), r = lane & 15, g = lane >> 4;
  const uint32_t sign = args_again().q_sign;
  const float f = fp8_scale(ks);
#pragma unroll
  for (int t = 0; t < kT; ++t) d[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    const bf16x8_t kf =
        __builtin_bit_cast(bf16x8_t, make_uint4(fp4_pair<0>(k.x, f), fp4_pair<1>(k.x, f), fp4_pair<2>(k.x, f), fp4_pair<3>(k.x, f)));
    k = make_uint4(k.y, k.z, k.w, 0u);
#pragma unroll
    for (int t = 0; t < kT; ++t) {
      uint4 x = ld16(q_row(w, 4 * t + (r >> 2)) + 32 * g + 8 * c);
      x = make_uint4(nan_if_not_finite(x.x ^ sign), nan_if_not_finite(x.y ^ sign), nan_if_not_finite(x.z ^ sign),
                     nan_if_not_finite(x.w ^ sign));
      if ((r & 3) != 0) x = make_uint4(0u, 0u, 0u, 0u);
      d[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, x), kf, d[t], 0, 0, 0);
    }
  }
}

template <int kT>
struct State {
  f32x4_t o[kT][4];        // MFMA j, of head 4 t + g: dims 8 (l % 16) + 2 j, + 1 by the probabilities' first numbers, then by the second
  float m[kT], l[kT];      // of head 4 t + g: the exponents' base, unscaled; sum, of this lane's keys until the merge
};

// A subtile's scores.
//
// The compiler counts the passes of the scaled instruction as if both operands had 4 bits: 8 wait states ahead of the result's first use
// instead of the 12 that an 8-bit operand takes, and the register that was read first then held something else.  So the wait is ours: 16
// states behind the last product, ahead of any use.
template <int kT>
__device__ __forceinline__ void scores(const Work& w, const uint4& codes, uint32_t ks, const Query<kT>& q, float (&s)[kT]) {
  f32x4_t d[kT];
  if (q.plain) {
    plain_scores<kT>(w, codes, ks, d);
  } else {
    const i32x8_t k = {(int)codes.x, (int)codes.y, (int)codes.z, (int)codes.w, 0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < kT; ++t)
      d[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(q.v[t], k, f32x4_t{0.f, 0.f, 0.f, 0.f}, 0, 4, 0, (int)q.s[t], 0, (int)ks);
    if constexpr (kT == 1) asm volatile("s_nop 15" : "+v"(d[0]));
    else asm volatile("s_nop 15" : "+v"(d[0]), "+v"(d[1]));
  }
#pragma unroll
  for (int t = 0; t < kT; ++t) s[t] = sum_parts(d[t]);
}

template <int kCtrl>
__device__ __forceinline__ float dpp_max(float x) { return fmaxf(x, dpp_f32<kCtrl>(x)); }

// The scores to probabilities, in s; the base (as tree_decode.hip's softmax has it) and the sum are updated and O rescaled.
template <int kT>
__device__ __forceinline__ void softmax(const int (&valid)[kSub], float scale, float ahead, float (&s)[kT][kSub], State<kT>& st) {
  if (((valid[0] & valid[1] & valid[2] & valid[3]) & 16) == 0) {
    const int r = lane_now() & 15;
#pragma unroll
    for (int t = 0; t < kT; ++t)
#pragma unroll
      for (int u = 0; u < kSub; ++u) s[t][u] = r < valid[u] ? s[t][u] : -INFINITY;
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

// The probabilities as two bf16 numbers into the wave's LDS, a row each.  A row has its 64 keys as the operands want them: of a quarter's
// 16 keys (32 bytes) each i's four subtiles, so that a lane's four probabilities are neighbours.
template <int kT>
__device__ __forceinline__ void store_p(const float (&p)[kT][kSub], int lane, uint8_t (*lds)[kPRow]) {
  const int r = lane & 15, g = lane >> 4;
  const int i = (r >> 1) & 3, quarter = 2 * (r >> 3) + (r & 1), pos = 32 * quarter + 8 * i;
#pragma unroll
  for (int t = 0; t < kT; ++t) {
    const u32x2 hi = {pack_bf16x2(p[t][0], p[t][1]), pack_bf16x2(p[t][2], p[t][3])};
    const u32x2 lo = {pack_bf16x2(p[t][0] - bf16_lo(hi.x), p[t][1] - bf16_hi(hi.x)),
                      pack_bf16x2(p[t][2] - bf16_lo(hi.y), p[t][3] - bf16_hi(hi.y))};
    *reinterpret_cast<u32x2*>(&lds[8 * t + 2 * g][pos]) = hi;
    *reinterpret_cast<u32x2*>(&lds[8 * t + 2 * g + 1][pos]) = lo;
  }
}

// Operands of P: lane l has row l % 16 = 4 head + 2 number + dim, whose pairs are (p, 0) or (0, p).
struct Pairs {
  uint32_t of[2];  // byte selectors: of a dword's lower half, of its upper one
};
__device__ __forceinline__ Pairs pairs_of(int lane) {
  return (lane & 1) != 0 ? Pairs{{0x01000c0cu, 0x03020c0cu}} : Pairs{{0x0c0c0100u, 0x0c0c0302u}};
}

// O += P V.
template <int kT>
__device__ __forceinline__ void values(const Tile& x, const float (&p)[kT][kSub], int lane, uint8_t (*lds)[kPRow], State<kT>& st) {
  const int r = lane & 15, g = lane >> 4;
  store_p<kT>(p, lane, lds);
  uint2 vs[kSub];
#pragma unroll
  for (int u = 0; u < kSub; ++u) vs[u] = x.vs[u];
  if (((x.valid[0] & x.valid[1] & x.valid[2] & x.valid[3]) & 16) == 0) {  // the exponent byte of a key that is not seen may be anything
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      const int left = max(0, min(8, x.valid[u] - 8 * (g >> 1)));
      vs[u].x &= (uint32_t)((1ull << (8 * min(left, 4))) - 1);
      vs[u].y &= (uint32_t)((1ull << (8 * max(left - 4, 0))) - 1);
    }
  }
  // The lane's keys are every second one of 8: bytes 0 and 2, or 1 and 3, of both dwords.  Only the exponent's bits of a scale count (all
  // 256 of them were compared with other bits and signs around them), so a byte is brought there by one shift.
  const int left = (g & 1) != 0 ? 15 : 23, around = (g & 1) != 0 ? 1 : 25;
  const Pairs pairs = pairs_of(lane);
  uint32_t w[kT][8];
#pragma unroll
  for (int t = 0; t < kT; ++t) {
    const uint8_t* row = lds[8 * t + (r >> 1)] + 32 * g;
    const uint4 a = ld16(row), b = ld16(row + 16);
    w[t][0] = a.x, w[t][1] = a.y, w[t][2] = a.z, w[t][3] = a.w, w[t][4] = b.x, w[t][5] = b.y, w[t][6] = b.z, w[t][7] = b.w;
  }
#pragma unroll
  for (int u = 0; u < kSub; ++u) {
    const float f[4] = {__uint_as_float(vs[u].x << left), __uint_as_float(__builtin_amdgcn_alignbit(vs[u].x, vs[u].x, around)),
                        __uint_as_float(vs[u].y << left), __uint_as_float(__builtin_amdgcn_alignbit(vs[u].y, vs[u].y, around))};
    bf16x8_t a[kT];
#pragma unroll
    for (int t = 0; t < kT; ++t) {
      uint32_t e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i] = perm_b32(0u, w[t][2 * i + (u >> 1)], pairs.of[u & 1]);
      a[t] = __builtin_bit_cast(bf16x8_t, make_uint4(e[0], e[1], e[2], e[3]));
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bf16x8_t b = __builtin_bit_cast(bf16x8_t, make_uint4(pair_at(x.v[u][0], j, f[0]), pair_at(x.v[u][1], j, f[1]),
                                                                 pair_at(x.v[u][2], j, f[2]), pair_at(x.v[u][3], j, f[3])));
#pragma unroll
      for (int t = 0; t < kT; ++t) st.o[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[t], b, st.o[t][j], 0, 0, 0);
    }
  }
}

// The append form's new row, quantised as the write kernel does and stored, and attended: key 0 of a step, whose other keys take no
// registers.
template <int kT>
__device__ __forceinline__ void append_step(const TreeArgs& a, const Work& w, const Query<kT>& q, uint8_t (*lds)[kPRow], State<kT>& st) {
  const int lane = lane_now(), r = lane & 15, g = lane >> 4;
  const TreeArgs& more = args_again();
  const uint16_t* kb = more.kn + (int64_t)w.b * more.kn_sb + (int64_t)w.h * more.kn_sh;
  const uint16_t* vb = more.vn + (int64_t)w.b * more.vn_sb + (int64_t)w.h * more.vn_sh;
  const int pi = (int)divide((uint32_t)w.L, more.per_page), off = w.L - pi * more.page_size;
  const int page = more.bt[(int64_t)w.b * more.bt_sb + pi];
  if ((unsigned)page >= (unsigned)a.num_pages) return;
  uint32_t kw[16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint4 e = ld16(kb + 32 * g + 8 * i);
    kw[4 * i] = e.x;
    kw[4 * i + 1] = e.y;
    kw[4 * i + 2] = e.z;
    kw[4 * i + 3] = e.w;
  }
  const uint4 e = ld16(vb + 8 * r);
  const uint32_t vw[4] = {e.x, e.y, e.z, e.w};
  const uint32_t ks = fp4_scale_byte(halves_max(bf16_any_amax_pair(kw)));
  const uint32_t vs = fp4_scale_byte(dpp_max_u32<kDppXor2>(dpp_max_u32<kDppXor1>(halves_max(bf16_any_amax_pair(vw)))));
  uint32_t kc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) kc[i] = fp4_codes8(kw[4 * i], kw[4 * i + 1], kw[4 * i + 2], kw[4 * i + 3], ks);
  const uint32_t vc = fp4_codes8(vw[0], vw[1], vw[2], vw[3], vs);
  const uint4 codes = make_uint4(kc[0], kc[1], kc[2], kc[3]);
  {
    const int64_t at = (int64_t)page * a.sp + (int64_t)off * a.st;
    const int64_t sat = (int64_t)page * a.ss_p + off;
    if (r == 0) {
      st16(a.kc + at + 16 * g, codes);
      a.ks[sat + g * a.page_size] = (uint8_t)ks;
    }
    if (g == 0) {
      *reinterpret_cast<uint32_t*>(a.vc + at + 4 * r) = vc;
      if ((r & 3) == 0) a.vs[sat + (r >> 2) * a.page_size] = (uint8_t)vs;
    }
  }
  float s[kT][kSub];
  float same[kT];  // of every key alike
  scores<kT>(w, codes, ks, q, same);
#pragma unroll
  for (int t = 0; t < kT; ++t) s[t][0] = same[t], s[t][1] = s[t][2] = s[t][3] = -INFINITY;
  const int valid[kSub] = {1, 0, 0, 0};
  softmax<kT>(valid, a.scale_log2, a.ahead, s, st);
  store_p<kT>(s, lane, lds);
  const Pairs pairs = pairs_of(lane);
  const float f = fp8_scale(vs);
#pragma unroll
  for (int t = 0; t < kT; ++t) {
    const uint32_t p = *reinterpret_cast<const uint32_t*>(lds[8 * t + (r >> 1)] + 32 * g);
    const bf16x8_t pa = __builtin_bit_cast(bf16x8_t, make_uint4(perm_b32(0u, p, pairs.of[0]), 0u, 0u, 0u));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bf16x8_t v = __builtin_bit_cast(bf16x8_t, make_uint4(g == 0 ? pair_at(vc, j, f) : 0u, 0u, 0u, 0u));
      st.o[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pa, v, st.o[t][j], 0, 0, 0);
    }
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
  const int row = thread >> 4, d0 = 8 * (thread & 15);
  if (row >= args_again().M) return;  // at most 4 kT rows
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kW; ++i) top = fmaxf(top, lds.m[i][row]);
  const float base = top == -INFINITY ? 0.f : top;
  float acc[8] = {}, sum = 0.f;
#pragma unroll
  for (int i = 0; i < kW; ++i) {
    const float f = fast_exp2(lds.m[i][row] - base);
    sum += f * lds.l[i][row];
#pragma unroll
    for (int d = 0; d < 8; ++d) acc[d] += f * so[i][row][d0 + d];
  }
  if (rec == nullptr) {
    store_out(out_row(w.b, w.h, row) + d0, acc, sum);
  } else {
    float* o = rec + row * kRecord;
    if (d0 == 0) *reinterpret_cast<float2*>(o + kD) = make_float2(top, sum);
#pragma unroll
    for (int d = 0; d < 8; d += 2) *reinterpret_cast<float2*>(o + d0 + d) = make_float2(acc[d], acc[d + 1]);
  }
}

// One workgroup a (row, KV head), its kW waves taking the row's steps in turn; or (kChunked) one of a chunk of a row's steps, which
// leaves a record for the join unless it is the row's only one.
template <int kMode, int kT, int kW, bool kChunked>
__global__ __launch_bounds__(64 * kW, kT == 1 ? 4 : 3) void fp4_decode_kernel(const TreeArgs args) {
  __shared__ Lds<kT, kW> lds;
  __shared__ __align__(16) float s_o[kW][4 * kT][kD + 4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Work w;
  int unit;
  unit_of(args, w.h, w.mb, unit);
  if (unit >= args.units) return;
  Window win;
  uint4 raw[kT];
  auto load_q = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < kT; ++t) raw[t] = ld16(q_row(w, 4 * t + (lane >> 4)) + 8 * (lane & 15));
  };
  int s0 = 0, s1;  // the chunk's steps
  float* rec = nullptr;
  if constexpr (kChunked) {
    const Chunk c = chunk_at<kStep * kW>(args, (uint32_t)unit, kMode);
    if (c.row < 0) return;
    w.b = c.row;
    w.L = c.L;
    const int T = steps_of<kStep>(w.L, kMode);
    w.Tc = w.L > 0 ? (w.L + kStep - 1) / kStep : 0;
    const int steps = (int)((rounds_of<kStep * kW>(args, w.L, kMode) + c.count - 1) / c.count) * kW;
    s0 = min(w.Tc, c.index * steps);
    s1 = c.index == c.count - 1 ? T : min(w.Tc, s0 + steps);  // the last one has the own step
    if (c.count > 1) rec = args_again().rec + ((int64_t)unit * args_again().hkv + w.h) * (int64_t)(16 * kRecord);
    if (c.index == 0 && w.h == 0 && threadIdx.x == 0) reinterpret_cast<Joined*>(args_again().ws)[w.b] = Joined{unit - c.index, c.count};
    const int s = s0 + wave + kW * (lane >> 2);
    const Entry e = entry_of<kSub>(w.b, s, lane);
    load_q();
    win = window_of<kFp4Pool>(e, w.L, s < min(s1, w.Tc));
  } else {
    w.b = unit;
    const int row0 = max(0, args.batch - 64 * kW);
    if (args.order && unit >= row0) w.b = kth_longest<kW>(args, row0, unit - row0, wave);
    // The first window's page ids do not wait for the row's length.
    const Entry e = entry_of<kSub>(w.b, wave + kW * (lane >> 2), lane);
    load_q();
    win = window_of<kFp4Pool>(e, INT_MAX, true);
    w.L = __builtin_amdgcn_readfirstlane(row_tokens(w.b, kMode));
    w.Tc = w.L > 0 ? (w.L + kStep - 1) / kStep : 0;
    s1 = steps_of<kStep>(w.L, kMode);
  }
  const TreeArgs a = at_head(args, w.h);
  if (s1 == 0 && rec == nullptr) {
    zero_rows(w.b, w.h, w.mb, 16);
    return;
  }
  const int first = s0 + wave;
  const int n = max(0, (min(s1, w.Tc) - first + kW - 1) / kW);  // this wave's cached steps: first, first + kW, ...
  int64_t at[kSub];
  uint32_t sat[kSub];
  int seen[kSub];
  auto place = [&](int j) __attribute__((always_inline)) {
    if ((j & (kWindow - 1)) == 0 && j > 0 && j < n) {
      const int l = lane_now();
      win = window_of<kFp4Pool>(entry_of<kSub>(w.b, first + kW * (j + (l >> 2)), l), w.L, j + (l >> 2) < n);
    }
    const int slot = kSub * (j & (kWindow - 1)), tokens = w.L - kStep * (first + kW * j);
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      at[u] = (int64_t)(uint32_t)readlane((int)win.at, slot + u) << 4;
      sat[u] = (uint32_t)readlane((int)win.sat, slot + u);
      const int k = readlane(win.valid, slot + u), left = tokens - 16 * u;
      seen[u] = j < n ? (k < left ? k : left < 0 ? 0 : left) : 0;  // (min as a chain of scalar selects)
    }
  };
  Tile x;
  place(0);
  x.load_k(a, at, sat, seen, lane);
  x.load_v(a, at, sat, seen, lane);
  Query<kT> q;
  prepare_q<kT, kW>(w, raw, wave, lds, q);
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
  if constexpr (kMode == kAppend) {
    if (first + n * kW == s1 - 1) append_step<kT>(a, w, q, lds.p[wave], st);  // the row's own step is this wave's
  }
  const TreeArgs again = at_head(args_again(), w.h);  // (not held in registers, and spilled, since the kernel's start)
  for (int i = 0; i < n; ++i) {
    float s[kT][kSub];
    place(i + 1);
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      float one[kT];
      scores<kT>(w, x.k[u], x.ks[u], q, one);
#pragma unroll
      for (int t = 0; t < kT; ++t) s[t][u] = one[t];
    }
    __builtin_amdgcn_sched_barrier(0);
    x.load_k(again, at, sat, seen, lane);
    __builtin_amdgcn_sched_barrier(0);
    softmax<kT>(x.valid, again.scale_log2, again.ahead, s, st);
    values<kT>(x, s, lane, lds.p[wave], st);
    __builtin_amdgcn_sched_barrier(0);
    x.load_v(again, at, sat, seen, lane);
    __builtin_amdgcn_sched_barrier(0);
  }
  merge_waves<kT, kW>(w, st, rec, wave, s_o, lds);
}

template <int kMode, int kT>
void launch(const TreeArgs& a, dim3 grid, hipStream_t stream) {
  if (a.target == 0) hipLaunchKernelGGL((fp4_decode_kernel<kMode, kT, 4, false>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((fp4_decode_kernel<kMode, kT, 4, true>), grid, dim3(256), 0, stream, a);
}

}  // namespace

hipError_t launch_fp4_decode(const TreeArgs& a, int mode, dim3 grid, hipStream_t stream) {
  if (a.group <= 4) {
    if (mode == kAppend) launch<kAppend, 1>(a, grid, stream);
    else launch<kNoKeys, 1>(a, grid, stream);
  } else {
    if (mode == kAppend) launch<kAppend, 2>(a, grid, stream);
    else launch<kNoKeys, 2>(a, grid, stream);
  }
  return hipGetLastError();
}

}  // namespace q3a
