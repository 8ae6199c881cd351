// Attention of a few query tokens per row over the paged K/V pool, on MFMA (gfx950): decode over the 8-bit pool (plain, and
// with the step's quantising write) and attention for trees of drafted tokens over the 8-bit or the bf16 pool.
//
// Row b has N query tokens (nodes) and ctx cached tokens, all visible to every node, and N keys of its own of which node n
// sees those that its mask row allows (decode: N = 1 and no own key, or its own one as the pool will hold it).  With
// G = Hq / Hkv the M = N G query rows m = (n, g) of a KV head share every key:
//   s_mj = scale q_m . k_j,   o_m = sum_j exp(s_mj - max_j s_mj) v_j / sum_j exp(s_mj - max_j s_mj);   zeros if nothing is seen.
//
// A step is 32 keys (two 16-token subtiles, each inside one page) by 16 kMT query rows, on one wave, from registers alone:
//   S^T = K Q^T   v_mfma_f32_16x16x32_bf16, A = 16 keys x 32 dims, B = Q^T.  Lane l holds key l % 16 and, of each 32 dims,
//                 the 8 that its quarter g = l / 16 takes: any split of the 128 dims over (step, quarter) is right as long
//                 as Q has the same, so each quarter takes 16 codes in a row and a load is 16 B (8-bit), 8 dims (bf16).
//   O^T = V^T P^T A = V^T: lane l holds for dim index l % 16 the 8 keys 4 g .. 4 g + 3 of both subtiles, which are the keys
//                 whose P its S^T registers hold, so P needs no lane moves.  Row i of MFMA j stands for dim 8 i + j: the
//                 lane loads 8 dims in a row of its 8 keys, and the transpose is byte permutes within the lane.
// Lane l of O^T then holds 32 dims in a row of query row l % 16.  K is multiplied by its scale as it is converted (exact);
// V's scale goes onto P.  Scores, statistics and O are fp32; P is rounded to bf16 for the product (2^-8 of each term at
// worst, the sum l is of the unrounded ones), as the prefill kernel does.
#include <algorithm>

#include "fp8_common.h"
#include "../../include/q3attn.h"

namespace q3a {

int check_fp8_pool(const char* who, const void* kc, const void* vc, int64_t sp, int64_t st, int64_t sh, const void* ks,
                   const void* vs, int64_t ss_p, int64_t ss_h, int num_pages, int page_size, int hkv);

namespace {

constexpr int kD = kRowDims;
constexpr int kStep = 32;       // keys per step
constexpr int kWindow = 32;     // steps whose page ids a wave holds at once (one id a lane)
constexpr int kMergeRow = kD + 4;  // floats per row of the merge buffer (16-byte rows off the bank period)
enum { kNoKeys = 0, kTree = 1, kAppend = 2 };

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
  const int32_t* seqlens;
  const int32_t* bt;
  int64_t bt_sb;
  int max_pages;
  uint16_t* out;
  int64_t o_sb, o_sn, o_sh;
  float* ws;
  int nodes, group, hkv, M;
  int mblocks, nchunk, min_steps;
  float scale_log2;
};

__device__ __forceinline__ int readlane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// The first of the 8 dims that MFMA step c's operand holds in quarter g, and the 16 B piece of the row it lies in.
template <bool kFp8>
__device__ __forceinline__ int dim_of(int c, int g) {
  return kFp8 ? (c >> 1) * 64 + g * 16 + (c & 1) * 8 : c * 32 + g * 8;
}

// A step's keys in registers: the 8-bit pool's codes, or bf16.
template <bool kFp8>
struct Keys;
template <>
struct Keys<true> {
  uint4 k[2][2];
  uint2 v[2][4];
  uint32_t ks[2], vs[2];  // K: the scale byte of key l % 16; V: those of keys 4 g .. 4 g + 3
  int valid[2];           // keys of the subtile that are seen
};
template <>
struct Keys<false> {
  uint4 k[2][4];
  uint4 v[2][4];
  int valid[2];
};

// One row (b), KV head and block of 16 kMT query rows: where its steps are.
struct Work {
  int b, h, mb;
  int L;       // cached tokens that are attended; < 0: the row is skipped
  int Tc, T;   // steps of cached keys, and with the own keys'
};

template <int kMT>
struct State {
  f32x4_t o[kMT][8];
  float m[kMT], l[kMT];  // of query row l % 16; l: this quarter's keys only, until the merge
};

// How the row's T steps split over chunks: `size` steps each, the first `live` chunks not empty.
__device__ __forceinline__ void split_of(const TreeArgs& a, int T, int& size, int& live) {
  size = max((T + a.nchunk - 1) / a.nchunk, a.min_steps);
  live = (T + size - 1) / size;
}

__device__ __forceinline__ int row_tokens(const TreeArgs& a, int b, int mode) {
  const int n = a.seqlens[b];
  const int cap = a.max_pages * a.page_size;
  if (mode == kAppend) return n < cap ? n : -1;  // no room for the new row: skipped
  return min(n, cap);
}

__device__ __forceinline__ int steps_of(const TreeArgs& a, int L, int mode) {
  if (L < 0) return 0;
  return (L + kStep - 1) / kStep + (mode == kTree ? (a.nodes + kStep - 1) / kStep : mode == kAppend ? 1 : 0);
}

template <bool kFp8>
__device__ __forceinline__ void load_cached(const TreeArgs& a, const Work& w, int step, int slot, int pid, int poff, int lane,
                                            Keys<kFp8>& x) {
  const int r = lane & 15, g = lane >> 4;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int page = readlane(pid, 2 * slot + u), off = readlane(poff, 2 * slot + u);
    int nv = min(16, w.L - (kStep * step + 16 * u));
    if ((unsigned)page >= (unsigned)a.num_pages) nv = 0;
    nv = max(nv, 0);
    x.valid[u] = nv;
    // Descriptors that end with the last seen key: what lies past it is not read and comes as zeros.
    const int64_t at = nv > 0 ? (int64_t)page * a.sp + (int64_t)w.h * a.sh + (int64_t)off * a.st : 0;
    const uint32_t bytes = nv > 0 ? (uint32_t)(nv - 1) * (uint32_t)a.st + (kFp8 ? kD : 2 * kD) : 0u;
    const auto rk = make_rsrc(a.kc + at, bytes), rv = make_rsrc(a.vc + at, bytes);
    const uint32_t krow = (uint32_t)r * (uint32_t)a.st, vrow = (uint32_t)(4 * g) * (uint32_t)a.st;
    if constexpr (kFp8) {
#pragma unroll
      for (int i = 0; i < 2; ++i) x.k[u][i] = buffer_load16(rk, krow + 64 * i + 16 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x.v[u][i] = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rv, (int)(vrow + i * a.st + 8 * r), 0, 0));
      const int64_t sat = nv > 0 ? (int64_t)page * a.ss_p + (int64_t)w.h * a.ss_h + off : 0;
      const auto rs = make_rsrc(a.ks + sat, nv > 0 ? 16 : 0), rt = make_rsrc(a.vs + sat, nv > 0 ? 16 : 0);
      x.ks[u] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(rs, r, 0, 0);
      x.vs[u] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rt, 4 * g, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) x.k[u][i] = buffer_load16(rk, krow + 64 * i + 16 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) x.v[u][i] = buffer_load16(rv, vrow + i * a.st + 16 * r);
    }
  }
}

// The A operand of S^T at MFMA step c.
__device__ __forceinline__ bf16x8_t k_operand(const Keys<true>& x, int u, int c) {
  const uint4 w = x.k[u][c >> 1];
  const uint32_t lo = (c & 1) ? w.z : w.x, hi = (c & 1) ? w.w : w.y;
  const float f = fp8_scale(x.ks[u]);
  return __builtin_bit_cast(bf16x8_t, make_uint4(fp8_pair<false>(lo, f), fp8_pair<true>(lo, f), fp8_pair<false>(hi, f),
                                                 fp8_pair<true>(hi, f)));
}
__device__ __forceinline__ bf16x8_t k_operand(const Keys<false>& x, int u, int c) {
  return __builtin_bit_cast(bf16x8_t, x.k[u][c]);
}

// The A operands of O^T for dims 8 i + j, j = jj and jj + 1 (jj even): the pairs of keys (0, 1), (2, 3) of both subtiles.
__device__ __forceinline__ void v_operands(const Keys<true>& x, int jj, bf16x8_t& a0, bf16x8_t& a1) {
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
__device__ __forceinline__ void v_operands(const Keys<false>& x, int jj, bf16x8_t& a0, bf16x8_t& a1) {
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

__device__ __forceinline__ float v_scale(const Keys<true>& x, int u, int i) { return fp8_scale((x.vs[u] >> (8 * i)) & 0xffu); }
__device__ __forceinline__ float v_scale(const Keys<false>&, int, int) { return 1.f; }

// One step.  kMasked: seen[t] tells which of the lane's 8 keys (bit 4 u + i) its query row sees; else every valid one.
template <bool kFp8, bool kScaledV, bool kMasked, int kMT>
__device__ __forceinline__ void step(const Keys<kFp8>& x, const bf16x8_t (&q)[kMT][4], const uint32_t (&seen)[kMT], float scale,
                                     int lane, State<kMT>& st) {
  const int g = lane >> 4;
  f32x4_t s[kMT][2];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const bf16x8_t kf = k_operand(x, u, c);
#pragma unroll
      for (int t = 0; t < kMT; ++t)
        s[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, q[t][c], c == 0 ? f32x4_t{0.f, 0.f, 0.f, 0.f} : s[t][u], 0, 0, 0);
    }
  bf16x8_t pb[kMT];
#pragma unroll
  for (int t = 0; t < kMT; ++t) {
    float y[2][4], top = -INFINITY;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool ok = kMasked ? ((seen[t] >> (4 * u + i)) & 1) != 0 : 4 * g + i < x.valid[u];
        y[u][i] = ok ? s[t][u][i] * scale : -INFINITY;
        top = fmaxf(top, y[u][i]);
      }
    top = max_xor32(max_xor16(top));
    const float m = fmaxf(st.m[t], top);
    const float base = m == -INFINITY ? 0.f : m;  // nothing seen so far: every exp2 below is of -inf
    const float alpha = fast_exp2(st.m[t] - base);
    st.m[t] = m;
    float sum = 0.f;
    uint32_t pk[4];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float pv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = fast_exp2(y[u][i] - base);
        sum += p;
        const bool ok = kMasked ? ((seen[t] >> (4 * u + i)) & 1) != 0 : 4 * g + i < x.valid[u];
        pv[i] = kScaledV ? (ok ? p * v_scale(x, u, i) : 0.f) : p;  // the scale byte of a key not seen may be anything
      }
      pk[2 * u] = pack_bf16x2(pv[0], pv[1]);
      pk[2 * u + 1] = pack_bf16x2(pv[2], pv[3]);
    }
    st.l[t] = st.l[t] * alpha + sum;
    pb[t] = __builtin_bit_cast(bf16x8_t, make_uint4(pk[0], pk[1], pk[2], pk[3]));
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) st.o[t][j][i] *= alpha;
  }
#pragma unroll
  for (int jj = 0; jj < 8; jj += 2) {
    bf16x8_t a0, a1;
    v_operands(x, jj, a0, a1);
#pragma unroll
    for (int t = 0; t < kMT; ++t) {
      st.o[t][jj] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, pb[t], st.o[t][jj], 0, 0, 0);
      st.o[t][jj + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1, pb[t], st.o[t][jj + 1], 0, 0, 0);
    }
  }
}

__device__ __forceinline__ bool not_finite_pair(uint32_t w) {
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
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
// zeros and ones counts them.
template <int kMT>
__device__ __forceinline__ void add_not_finite(const Keys<false>& v, const uint32_t (&seen)[kMT], State<kMT>& st) {
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
    const float what = kind == 0 ? INFINITY : kind == 1 ? -INFINITY : __builtin_nanf("");
    Keys<false> x;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 e = v.v[u][i];
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
__device__ void tree_step(const TreeArgs& a, const Work& w, int ts, const bf16x8_t (&q)[kMT][4], int lane, State<kMT>& st) {
  const int r = lane & 15, g = lane >> 4;
  const uint16_t* kb = a.kn + (int64_t)w.b * a.kn_sb + (int64_t)w.h * a.kn_sh;
  const uint16_t* vb = a.vn + (int64_t)w.b * a.vn_sb + (int64_t)w.h * a.vn_sh;
  Keys<false> x;
  bool odd = false;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int j0 = kStep * ts + 16 * u;
    x.valid[u] = max(0, min(16, a.nodes - j0));
    const int jk = j0 + r;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      x.k[u][c] = make_uint4(0u, 0u, 0u, 0u);
      if (jk < a.nodes) x.k[u][c] = ld16(kb + (int64_t)jk * a.kn_sn + dim_of<kFp8>(c, g));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int jv = j0 + 4 * g + i;
      x.v[u][i] = make_uint4(0u, 0u, 0u, 0u);
      if (jv < a.nodes) x.v[u][i] = ld16(vb + (int64_t)jv * a.vn_sn + 8 * r);
      const uint4 e = x.v[u][i];
      odd = odd || not_finite_pair(e.x) || not_finite_pair(e.y) || not_finite_pair(e.z) || not_finite_pair(e.w);
    }
  }
  const bool any_odd = __builtin_amdgcn_ballot_w64(odd) != 0;
  Keys<false> kinds;
  if (any_odd) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 e = x.v[u][i];
        kinds.v[u][i] = e;
        x.v[u][i] = make_uint4(finite_halves(e.x), finite_halves(e.y), finite_halves(e.z), finite_halves(e.w));
      }
  }
  uint32_t seen[kMT];
#pragma unroll
  for (int t = 0; t < kMT; ++t) {
    const int m = (w.mb * kMT + t) * 16 + r;
    const int n = m / a.group;
    seen[t] = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = kStep * ts + 16 * u + 4 * g + i;
        bool ok = n < a.nodes && j < a.nodes;
        if (ok) ok = a.mask != nullptr ? a.mask[(int64_t)w.b * a.m_sb + (int64_t)n * a.m_sn + j] != 0 : j <= n;
        seen[t] |= ok ? 1u << (4 * u + i) : 0u;
      }
  }
  step<false, false, true, kMT>(x, q, seen, a.scale_log2, lane, st);
  if (any_odd) add_not_finite<kMT>(kinds, seen, st);
}

// The append form's new row, quantised as the write kernel does and stored, then attended as a cached subtile of one key.
__device__ __forceinline__ void append_keys(const TreeArgs& a, const Work& w, int lane, bool store, Keys<true>& x) {
  const int r = lane & 15, g = lane >> 4;
  const uint16_t* kb = a.kn + (int64_t)w.b * a.kn_sb + (int64_t)w.h * a.kn_sh;
  const uint16_t* vb = a.vn + (int64_t)w.b * a.vn_sb + (int64_t)w.h * a.vn_sh;
  const int pi = w.L / a.page_size, off = w.L - pi * a.page_size;
  const int page = a.bt[(int64_t)w.b * a.bt_sb + pi];
  const bool ok = (unsigned)page < (unsigned)a.num_pages;
  uint32_t kw[16], vw[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint4 e = ld16(kb + 64 * (i >> 1) + 16 * g + 8 * (i & 1));
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
  uint32_t km = halves_max(bf16_amax_pair(kw)), vm = halves_max(bf16_amax_pair(vw));
  km = (uint32_t)__float_as_int(max_xor32(max_xor16(__int_as_float((int)km))));  // small integers order as floats do
  vm = dpp_max_u32<kDppXor1>(vm);
  vm = dpp_max_u32<kDppXor2>(vm);
  vm = dpp_max_u32<kDppHalfMirror>(vm);
  vm = dpp_max_u32<kDppMirror>(vm);
  const uint32_t ks = fp8_scale_byte(km), vs = fp8_scale_byte(vm);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    x.valid[u] = 0;
    x.ks[u] = ks;
    x.vs[u] = vs;
#pragma unroll
    for (int i = 0; i < 2; ++i) x.k[u][i] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int i = 0; i < 4; ++i) x.v[u][i] = make_uint2(0u, 0u);
  }
  uint4 kc[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    kc[i] = make_uint4(fp8_codes4(kw[8 * i], kw[8 * i + 1], ks), fp8_codes4(kw[8 * i + 2], kw[8 * i + 3], ks),
                       fp8_codes4(kw[8 * i + 4], kw[8 * i + 5], ks), fp8_codes4(kw[8 * i + 6], kw[8 * i + 7], ks));
  const uint2 vc = make_uint2(fp8_codes4(vw[0], vw[1], vs), fp8_codes4(vw[2], vw[3], vs));
  x.valid[0] = ok ? 1 : 0;
  if (r == 0) {
    x.k[0][0] = kc[0];
    x.k[0][1] = kc[1];
  }
  if (g == 0) x.v[0][0] = vc;
  if (store && ok) {
    const int64_t at = (int64_t)page * a.sp + (int64_t)w.h * a.sh + (int64_t)off * a.st;
    const int64_t sat = (int64_t)page * a.ss_p + (int64_t)w.h * a.ss_h + off;
    if (r == 0) {
      st16(a.kc + at + 16 * g, kc[0]);
      st16(a.kc + at + 64 + 16 * g, kc[1]);
    }
    if (g == 0) *reinterpret_cast<u32x2*>(a.vc + at + 8 * r) = __builtin_bit_cast(u32x2, vc);
    if (lane == 0) {
      a.ks[sat] = (uint8_t)ks;
      a.vs[sat] = (uint8_t)vs;
    }
  }
}

// Workgroup: (chunk of a row's steps, KV head, block of 16 kMT query rows).  Its kW waves take the chunk's steps in turn,
// each with a state of its own, and merge in LDS.  A row of one live chunk is finished here; otherwise the chunk's
// (m, l, o) goes into the workspace for the merge kernel.  The KV head is the fastest grid dimension: workgroups go to the
// 8 XCDs in turn, so with 8 heads each L2 holds one head's keys for all their readers.
template <bool kFp8, int kMode, int kMT, int kW>
__global__ __launch_bounds__(64 * kW) void tree_kernel(const TreeArgs a) {
  __shared__ __align__(16) float s_o[kW][16][kMergeRow];
  __shared__ float s_m[kW][16], s_l[kW][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  Work w;
  int x = blockIdx.x;
  w.h = x % a.hkv;
  x /= a.hkv;
  w.mb = x % a.mblocks;
  const int chunk = x / a.mblocks;
  w.b = blockIdx.y;
  w.L = row_tokens(a, w.b, kMode);
  w.T = steps_of(a, w.L, kMode);
  w.Tc = w.L > 0 ? (w.L + kStep - 1) / kStep : 0;
  int size, live;
  split_of(a, w.T, size, live);
  if (chunk >= max(live, 1)) return;
  const int s0 = chunk * size, s1 = min(w.T, s0 + size);

  State<kMT> st;
#pragma unroll
  for (int t = 0; t < kMT; ++t) {
    st.m[t] = -INFINITY;
    st.l[t] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) st.o[t][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  if (s0 + wave < s1) {
    bf16x8_t q[kMT][4];
#pragma unroll
    for (int t = 0; t < kMT; ++t) {
      const int m = (w.mb * kMT + t) * 16 + r;
      const int n = m / a.group;
      const uint16_t* qp = a.q + (int64_t)w.b * a.q_sb + (int64_t)n * a.q_sn + (int64_t)(w.h * a.group + m - n * a.group) * a.q_sh;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (m < a.M) v = ld16(qp + dim_of<kFp8>(c, g));
        q[t][c] = __builtin_bit_cast(bf16x8_t, v);
      }
    }
    uint32_t all[kMT] = {};
    const int c1 = min(s1, w.Tc);  // cached steps end here
    int s = s0 + wave;
    while (s < c1) {
      // The page ids of this wave's next kWindow steps, one subtile a lane.
      const int n_here = min(kWindow, (c1 - s + kW - 1) / kW);
      int pid = -1, poff = 0;
      {
        const int tok = kStep * (s + kW * (lane >> 1)) + 16 * (lane & 1);
        if ((lane >> 1) < n_here && tok < w.L) {
          const int pi = tok / a.page_size;
          poff = tok - pi * a.page_size;
          pid = a.bt[(int64_t)w.b * a.bt_sb + pi];
        }
      }
      // Two register tiles in turn: the next step's loads are issued before this step is computed.
      Keys<kFp8> ka, kb;
      load_cached<kFp8>(a, w, s, 0, pid, poff, lane, ka);
      for (int i = 0; i < n_here; i += 2) {
        if (i + 1 < n_here) load_cached<kFp8>(a, w, s + kW * (i + 1), i + 1, pid, poff, lane, kb);
        __builtin_amdgcn_sched_barrier(0);
        step<kFp8, kFp8, false, kMT>(ka, q, all, a.scale_log2, lane, st);
        if (i + 1 < n_here) {
          if (i + 2 < n_here) load_cached<kFp8>(a, w, s + kW * (i + 2), i + 2, pid, poff, lane, ka);
          __builtin_amdgcn_sched_barrier(0);
          step<kFp8, kFp8, false, kMT>(kb, q, all, a.scale_log2, lane, st);
        }
      }
      s += kW * n_here;
    }
    if constexpr (kMode == kTree) {
      for (; s < s1; s += kW) tree_step<kFp8, kMT>(a, w, s - w.Tc, q, lane, st);
    }
    if constexpr (kMode == kAppend) {
      if (s < s1) {
        Keys<true> kn;
        append_keys(a, w, lane, w.mb == 0, kn);
        step<true, true, false, kMT>(kn, q, all, a.scale_log2, lane, st);
      }
    }
  }

  // Merge the waves: 16 query rows at a time through LDS.
  float* rec = nullptr;
  if (live > 1) rec = a.ws + (((int64_t)w.b * a.hkv + w.h) * a.nchunk + chunk) * (int64_t)a.M * (kD + 2);
#pragma unroll
  for (int t = 0; t < kMT; ++t) {
    if ((w.mb * kMT + t) * 16 >= a.M) break;
    if (t > 0) __syncthreads();
    const float l = sum_xor32(sum_xor16(st.l[t]));
    if (g == 0) {
      s_m[wave][r] = st.m[t];
      s_l[wave][r] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      *reinterpret_cast<f32x4_t*>(&s_o[wave][r][32 * g + 8 * i]) =
          f32x4_t{st.o[t][0][i], st.o[t][1][i], st.o[t][2][i], st.o[t][3][i]};
      *reinterpret_cast<f32x4_t*>(&s_o[wave][r][32 * g + 8 * i + 4]) =
          f32x4_t{st.o[t][4][i], st.o[t][5][i], st.o[t][6][i], st.o[t][7][i]};
    }
    __syncthreads();
    if (threadIdx.x < 256) {
      const int row = threadIdx.x >> 4, d0 = 8 * (threadIdx.x & 15);
      const int m = (w.mb * kMT + t) * 16 + row;
      if (m < a.M) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < kW; ++i) top = fmaxf(top, s_m[i][row]);
        const float base = top == -INFINITY ? 0.f : top;
        float acc[8] = {}, sum = 0.f;
#pragma unroll
        for (int i = 0; i < kW; ++i) {
          const float f = fast_exp2(s_m[i][row] - base);
          sum += f * s_l[i][row];
#pragma unroll
          for (int d = 0; d < 8; ++d) acc[d] += f * s_o[i][row][d0 + d];
        }
        if (rec == nullptr) {
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          const int n = m / a.group;
          uint16_t* op = a.out + (int64_t)w.b * a.o_sb + (int64_t)n * a.o_sn +
                         (int64_t)(w.h * a.group + m - n * a.group) * a.o_sh + d0;
          st16(op, make_uint4(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv),
                              pack_bf16x2(acc[4] * inv, acc[5] * inv), pack_bf16x2(acc[6] * inv, acc[7] * inv)));
        } else {
          float* o = rec + (int64_t)m * (kD + 2);
          if (d0 == 0) {
            o[kD] = top;
            o[kD + 1] = sum;
          }
          // rows of 130 floats: 8-byte aligned
#pragma unroll
          for (int d = 0; d < 8; d += 2) *reinterpret_cast<float2*>(o + d0 + d) = make_float2(acc[d], acc[d + 1]);
        }
      }
    }
  }
}

// Merges the chunks' records of rows that have more than one: 16 lanes a query row, 8 dims a lane.
template <int kMode>
__global__ __launch_bounds__(256) void tree_merge_kernel(const TreeArgs a) {
  const int b = blockIdx.y;
  const int mt = (a.M + 15) / 16;
  const int h = blockIdx.x / mt, m = (blockIdx.x - h * mt) * 16 + (threadIdx.x >> 4), d0 = 8 * (threadIdx.x & 15);
  int size, live;
  split_of(a, steps_of(a, row_tokens(a, b, kMode), kMode), size, live);
  if (live <= 1 || m >= a.M) return;
  const int64_t rec = (int64_t)a.M * (kD + 2);
  const float* base = a.ws + ((int64_t)b * a.hkv + h) * a.nchunk * rec + (int64_t)m * (kD + 2);
  float top = -INFINITY;
  for (int c = 0; c < live; ++c) top = fmaxf(top, base[c * rec + kD]);
  const float ref = top == -INFINITY ? 0.f : top;
  float acc[8] = {}, sum = 0.f;
  for (int c = 0; c < live; ++c) {
    const float* o = base + c * rec;
    const float f = fast_exp2(o[kD] - ref);
    sum += f * o[kD + 1];
#pragma unroll
    for (int d = 0; d < 8; d += 2) {
      const float2 e = *reinterpret_cast<const float2*>(o + d0 + d);
      acc[d] += f * e.x;
      acc[d + 1] += f * e.y;
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int n = m / a.group;
  uint16_t* op = a.out + (int64_t)b * a.o_sb + (int64_t)n * a.o_sn + (int64_t)(h * a.group + m - n * a.group) * a.o_sh + d0;
  st16(op, make_uint4(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv),
                      pack_bf16x2(acc[4] * inv, acc[5] * inv), pack_bf16x2(acc[6] * inv, acc[7] * inv)));
}

// ---------------------------------------------------------------------------------------------------- host side

constexpr int kWaves = 4;

int tiles_per_wave(int M) { return M <= 16 ? 1 : M <= 32 ? 2 : 4; }

// Chunks a row's steps are split into at most, from the shape alone (the lengths are on the device).
int chunks_of(int batch, int hkv, int mblocks, int64_t capacity, int nodes) {
  const int64_t steps = (capacity + kStep - 1) / kStep + (nodes + kStep - 1) / kStep;
  const int64_t groups = (int64_t)batch * hkv * mblocks;
  const int64_t want = std::max<int64_t>(1, (int64_t)num_cus() * 4 / std::max<int64_t>(groups, 1));
  const int64_t most = std::max<int64_t>(1, steps / (2 * kWaves));
  return (int)std::min<int64_t>(std::min(want, most), 256);
}

template <bool kFp8, int kMode>
int launch(const TreeArgs& a, int batch, const char* who, hipStream_t stream) {
  const dim3 grid((unsigned)(a.hkv * a.mblocks * a.nchunk), (unsigned)batch);
  const int tiles = tiles_per_wave(a.M);
  if constexpr (kMode == kTree) {
    if (tiles == 2) hipLaunchKernelGGL((tree_kernel<kFp8, kMode, 2, kWaves>), grid, dim3(64 * kWaves), 0, stream, a);
    if (tiles == 4) hipLaunchKernelGGL((tree_kernel<kFp8, kMode, 4, kWaves>), grid, dim3(64 * kWaves), 0, stream, a);
  }
  if (tiles == 1) hipLaunchKernelGGL((tree_kernel<kFp8, kMode, 1, kWaves>), grid, dim3(64 * kWaves), 0, stream, a);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && a.nchunk > 1) {
    hipLaunchKernelGGL((tree_merge_kernel<kMode>), dim3((unsigned)(a.hkv * ((a.M + 15) / 16)), (unsigned)batch), dim3(256), 0,
                       stream, a);
    e = hipGetLastError();
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
  if (max_pages < 0 || (int64_t)max_pages * page_size > (1 << 30))
    return fail(Q3A_EINVAL, "%s: table of %d pages of %d tokens (at most 2^30 tokens a row)", who, max_pages, page_size);
  return Q3A_OK;
}

size_t workspace_of(int batch, int nodes, int hq, int hkv, int64_t capacity) {
  const int M = nodes * (hq / hkv);
  const int per = 16 * tiles_per_wave(M);
  const int n = chunks_of(batch, hkv, (M + per - 1) / per, capacity, nodes);
  return n > 1 ? (size_t)batch * hkv * n * M * (kD + 2) * sizeof(float) : 0;
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
  const int per = 16 * tiles_per_wave(a.M);
  a.mblocks = (a.M + per - 1) / per;
  const int64_t capacity = (int64_t)a.max_pages * a.page_size;
  a.nchunk = chunks_of(batch, a.hkv, a.mblocks, capacity, a.nodes);
  a.min_steps = kWaves;
  const size_t need = workspace_of(batch, a.nodes, hq, a.hkv, capacity);
  if (need > 0 && (a.ws == nullptr || workspace_bytes < need || ((uintptr_t)a.ws & 15) != 0))
    return fail(Q3A_ESPACE, "%s: workspace of %zu bytes, %zu needed (16-byte aligned)", who, workspace_bytes, need);
  a.sp = kv_page * elem;
  a.st = (int)(kv_tok * elem);
  a.sh = kv_head * elem;
  a.scale_log2 = softmax_scale * kLog2e;
  const hipStream_t s = (hipStream_t)stream;
  if (fp8) {
    if (mode == kNoKeys) return launch<true, kNoKeys>(a, batch, who, s);
    if (mode == kAppend) return launch<true, kAppend>(a, batch, who, s);
    return launch<true, kTree>(a, batch, who, s);
  }
  return launch<false, kTree>(a, batch, who, s);
}

}  // namespace
}  // namespace q3a

using namespace q3a;

extern "C" size_t q3a_paged_decode_tree_workspace_bytes(int batch, int num_nodes, int num_q_heads, int num_kv_heads, int head_dim,
                                                        int max_pages_per_seq, int page_size) {
  if (check_shape("q3a_paged_decode_tree_workspace_bytes", batch, num_nodes, num_q_heads, num_kv_heads, head_dim,
                  max_pages_per_seq, page_size) != Q3A_OK || batch == 0)
    return 0;
  return workspace_of(batch, num_nodes, num_q_heads, num_kv_heads, (int64_t)max_pages_per_seq * page_size);
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
  a.ws = (float*)workspace;
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
  a.ws = (float*)workspace;
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
  a.ws = (float*)workspace;
  a.nodes = num_nodes;
  a.hkv = num_kv_heads;
  return run(who, a, kTree, fp8, batch, num_q_heads, workspace_bytes, kv_stride_page, kv_stride_tok, kv_stride_head,
             softmax_scale, stream);
}
