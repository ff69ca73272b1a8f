// Cross attention kernels, included once per element type T (see cross_attn.h).
//
//   x_ij = scale q_i . k_j + bias_ij, -inf where key j is hidden;  P = softmax_j(x);  o_i = sum_j P_ij v_j
//   dv_j = sum_i P_ij do_i,  dS_ij = P_ij (do_i . v_j - delta_i),  delta_i = do_i . o_i,
//   dq_i = scale sum_j dS_ij k_j,  dk_j = scale sum_i dS_ij q_i,  dbias = dS
//
// Every product runs on 32x32x16 MFMA tiles (accumulators: lane l, register r hold column l & 31, row
// 8 (r >> 2) + 4 (l >> 5) + (r & 3)).  The forward and the dq kernel form S^T = K Q^T, so a lane's
// column is one query: its softmax statistics are the lane's own, and the accumulator of P^T (dS^T)
// is, as it stands, the right operand of O^T = V^T P^T (dQ^T = K^T dS^T), with the left operand read
// from LDS in the accumulators' key order.  The dk, dv kernel forms S = Q K^T: its lanes hold keys.
//
// Heads that share a key head are rows of one tile, so keys and values are read once for them.
//
// Measured (one MI355X, us a launch).  Forward: 4 x 2048 queries x 4096 keys, 16 heads x 64 channels, bf16 165
// to 190 (830 to 720 TFLOP/s; 4 x 32 channels 148, 128 channels 348 = 790 TFLOP/s); beside the MFMAs each
// score costs an exponential, a rounding and the sum, so matrix and vector units are both busy and the clock
// falls to what power allows.  512 windows of 32 x 128, 4 heads x 32 with bias 18.5 (75 MB: 4.1 TB/s, 15.5 at
// a copy's rate).  8 x 1 query x 1536 keys, 16 heads over 4: 7.0 and 3.3 for the join, both latency.  fp32,
// 384 x 2900 x 8 heads x 48: 29 and 5 (six products for one).
#pragma once
#include "cross_attn.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;

template <int V>
struct IntC { static constexpr int value = V; };

PF_DEV f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}
PF_DEV float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
PF_DEV float xor32_max(float v) { return fmaxf(v, __shfl_xor(v, 32)); }
PF_DEV float xor32_sum(float v) { return v + __shfl_xor(v, 32); }
PF_DEV int acc_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// ------------------------------------------------------------------------------ tiles
// Operands of 16-bit types are themselves.  fp32 operands are split into three bf16 parts, each the
// rounded rest of the ones before: x = h + m + l exactly, in bf16's exponent range, which is fp32's.  A
// product takes h h', h m', m h', m m', h l' and l h'; what is left out is below 2^-25 of it.  Six bf16
// MFMAs (192 cycles for 16 channels) take the place of eight fp32 ones (512).
//
// Op: 32 rows x 16 channels as an MFMA operand; lane (n, h) holds channels 8 h .. 8 h + 7 of row n.
template <typename T>
struct LdsType { typedef T type; };
template <>
struct LdsType<float> { typedef bhalf_t type; };

template <typename T>
struct Mma {
  static constexpr bool SPLIT = __is_same(T, float);
  static constexpr int PARTS = SPLIT ? 3 : 1, E = 8;
  typedef typename LdsType<T>::type L;   // what LDS tiles hold, PARTS planes of it
  typedef L part_t __attribute__((ext_vector_type(8)));
  typedef L quad_t __attribute__((ext_vector_type(4)));
  struct Op { part_t p[PARTS]; };
  struct Packed { Op f[2]; };   // an accumulator as the right operand of a product over its 32 rows

  static constexpr int row_stride(int dp) { return dp + 8; }   // rows land on distinct banks (16 lanes x 16 bytes)
  // read both ways: the same, and four rows x 32 channels of the transposing reads meet in two banks at most
  // (2 x 2048 x 2048, 16 heads over 4, 128 channels: dk, dv 176 us, with dp + 8 185; dq 115 and 118)
  static constexpr int both_stride(int dp) { return dp == 128 ? dp + 24 : dp + 8; }
  // only read in transposed 4 x 16 blocks: four rows x 32 channels on (nearly) distinct banks
  static constexpr int col_stride(int dp) { return dp == 32 ? 32 : dp == 64 ? 80 : dp + (SPLIT ? 8 : 32); }

  static PF_DEV f32x16 mma1(const part_t& a, const part_t& b, const f32x16& c) {
    if constexpr (__is_same(L, half_t)) return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static PF_DEV f32x16 mma(const Op& a, const Op& b, f32x16 c) {
    if constexpr (SPLIT) {
      c = mma1(a.p[2], b.p[0], c);
      c = mma1(a.p[0], b.p[2], c);
      c = mma1(a.p[1], b.p[1], c);
      c = mma1(a.p[1], b.p[0], c);
      c = mma1(a.p[0], b.p[1], c);
    }
    return mma1(a.p[0], b.p[0], c);
  }
  // x[i] into element i of p[0 .. PARTS)
  template <int N, typename V>
  static PF_DEV void put(const float (&x)[N], V* p) {
    if constexpr (!SPLIT) {
#pragma unroll
      for (int i = 0; i < N; ++i) p[0][i] = (L)x[i];
    } else {
      float r[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        p[0][i] = (L)x[i];
        r[i] = x[i] - (float)p[0][i];
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        p[1][i] = (L)r[i];
        p[2][i] = (L)(r[i] - (float)p[1][i]);
      }
    }
  }
  // the same for a caller's values: infinities, and what rounds to one, are not split
  template <int N, typename V>
  static PF_DEV void put_any(const float (&x)[N], V* p) {
    put(x, p);
    if constexpr (SPLIT) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) top = fmaxf(top, __builtin_fabsf(x[i]));
      if (top >= 3.38e38f) {   // bf16's largest value is 3.3895e38
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (__builtin_fabsf(x[i]) >= 3.38e38f) {
            const float t = __uint_as_float(__float_as_uint(x[i]) & 0xffff0000u), r = x[i] == t ? 0.f : x[i] - t;
            p[0][i] = (L)t, p[1][i] = (L)r, p[2][i] = (L)(r - (float)p[1][i]);
          }
        }
      }
    }
  }
  static PF_DEV Packed pack(const f32x16& x) {
    Packed b;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      float y[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) y[t] = x[8 * s + t];
      put(y, b.f[s].p);
    }
    return b;
  }
  // 16-bit types: x to fp32's accuracy in WHOLE roundings, each of the rest of the ones before
  static constexpr int WHOLE = __is_same(T, half_t) ? 2 : 3;
  static PF_DEV void pack_whole(const f32x16& x, Packed (&b)[WHOLE]) {
    f32x16 r = x;
#pragma unroll
    for (int k = 0; k < WHOLE; ++k) {
      b[k] = pack(r);
#pragma unroll
      for (int t = 0; t < 16; ++t) r[t] -= (float)b[k].f[t >> 3].p[0][t & 7];
    }
  }
  // 16-bit types: c + the sum of this lane's 16 values as they were rounded
  static PF_DEV float sum(const Packed& b, float c) {
    typedef L pair_t __attribute__((ext_vector_type(2)));
    const pair_t one = {(L)1.f, (L)1.f};
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int t = 0; t < 8; t += 2) {
        const pair_t v = {b.f[s].p[0][t], b.f[s].p[0][t + 1]};
        if constexpr (__is_same(L, half_t)) c = __builtin_amdgcn_fdot2(v, one, c, false);
        else c = __builtin_amdgcn_fdot2_f32_bf16(v, one, c, false);
      }
    return c;
  }
  // LDS tiles are PARTS planes, `plane` elements apart
  static PF_DEV Op load(const L* a, int plane) {
    Op o;
#pragma unroll
    for (int i = 0; i < PARTS; ++i) o.p[i] = *reinterpret_cast<const part_t*>(a + i * plane);
    return o;
  }
  // acc[r][dt] += X^T P[r] over 32 rows of the LDS tile X (row stride `st`), taken in P's order.  A transposing
  // read hands lane i of 16 the column i of a 4 x 16 block whose 8-byte pieces the lanes point at.
  template <int DT, int R>
  static PF_DEV void outer(const L* x, int plane, int st, int lane, const Packed (&p)[R], f32x16 (&acc)[R][DT]) {
    const int h = lane >> 5, i = lane & 15, c16 = (lane >> 4) & 1;
    const L* at = x + (4 * h + (i >> 2)) * st + 16 * c16 + 4 * (i & 3);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        Op a;
#pragma unroll
        for (int k = 0; k < PARTS; ++k) {
          const L* pl = at + k * plane + 32 * dt;
          const quad_t lo = tr_read(pl + (16 * s) * st), hi = tr_read(pl + (16 * s + 8) * st);
          a.p[k] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r][dt] = mma(a, p[r].f[s], acc[r][dt]);
      }
  }
  // 16-bit types: acc[dt] += X^T (P[0] + P[1] + ..)
  template <int DT, int K>
  static PF_DEV void outer_sum(const L* x, int st, int lane, const Packed (&p)[K], f32x16 (&acc)[DT]) {
    const int h = lane >> 5, i = lane & 15, c16 = (lane >> 4) & 1;
    const L* at = x + (4 * h + (i >> 2)) * st + 16 * c16 + 4 * (i & 3);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const quad_t lo = tr_read(at + 32 * dt + (16 * s) * st), hi = tr_read(at + 32 * dt + (16 * s + 8) * st);
        const part_t a = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
        for (int k = K - 1; k >= 0; --k) acc[dt] = mma1(a, p[k].f[s].p[0], acc[dt]);
      }
  }
  static PF_DEV quad_t tr_read(const L* p) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4 lds_t;
    return __builtin_bit_cast(quad_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)p));
  }
};

// 32 rows x DP channels in registers
template <typename T, int DP>
struct Frag {
  static constexpr int S = DP / 16;
  typename Mma<T>::Op f[S];
  // row `p` in global memory; channels >= D are zero, and all are where !ok
  PF_DEV void load(const T* p, int D, int h, bool ok, bool neg = false) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int d = 16 * s + 8 * h;
      if constexpr (Mma<T>::SPLIT) {
        f32x4 a = {}, b = {};
        if (ok && d < D) a = *reinterpret_cast<const f32x4*>(p + d), b = *reinterpret_cast<const f32x4*>(p + d + 4);
        const float g = neg ? -1.f : 1.f;
        const float x[8] = {a[0] * g, a[1] * g, a[2] * g, a[3] * g, b[0] * g, b[1] * g, b[2] * g, b[3] * g};
        Mma<T>::put_any(x, f[s].p);
      } else {
        const typename Mma<T>::part_t z = {};
        f[s].p[0] = ok && d < D ? *reinterpret_cast<const typename Mma<T>::part_t*>(p + d) : z;
        if (neg) f[s].p[0] = -f[s].p[0];
      }
    }
  }
};

// c += A B^T over channels: A the LDS tile's 32 rows at `a` (this lane's row, channel 8 h), B a fragment
template <typename T, int DP>
PF_DEV f32x16 inner(const typename Mma<T>::L* a, int plane, const Frag<T, DP>& b, f32x16 c) {
#pragma unroll
  for (int s = 0; s < Frag<T, DP>::S; ++s) c = Mma<T>::mma(Mma<T>::load(a + 16 * s, plane), b.f[s], c);
  return c;
}

// c[r] = A B[r]^T
template <typename T, int DP, int R>
PF_DEV void inner_rows(const typename Mma<T>::L* a, int plane, const Frag<T, DP> (&b)[R], f32x16 (&c)[R]) {
#pragma unroll
  for (int r = 0; r < R; ++r) c[r] = zero16();
#pragma unroll
  for (int s = 0; s < Frag<T, DP>::S; ++s) {
    const auto f = Mma<T>::load(a + 16 * s, plane);
#pragma unroll
    for (int r = 0; r < R; ++r) c[r] = Mma<T>::mma(f, b[r].f[s], c[r]);
  }
}

// A tile of ROWS rows x DP channels on its way from global memory to LDS: 16-byte pieces in registers,
// a thread's pieces in one column of pieces, 256 / PER rows apart.
template <typename T, int DP, int ROWS>
struct Stage {
  typedef typename Vec16<T>::type vec_t;
  typedef typename Mma<T>::L L;
  static constexpr int N = Vec16<T>::N, PER = DP / N, CH = ROWS * PER / 256, STEP = 256 / PER;
  static_assert(ROWS * PER % 256 == 0 && 256 % PER == 0, "whole pieces per thread");
  vec_t v[CH];
  static PF_DEV int row(int j) { return (int)threadIdx.x / PER + j * STEP; }
  static PF_DEV int chan() { return (int)threadIdx.x % PER * N; }
  // this thread's first piece, in bytes from the tile's first row (row strides are below 2^22 elements)
  static PF_DEV uint32_t first(int stride) { return ((uint32_t)row(0) * (uint32_t)stride + (uint32_t)chan()) * (uint32_t)sizeof(T); }
  // p: row 0 of the tile, rows `stride` apart; all rows are there
  PF_DEV void load(const T* p, int stride, int D) {
    if (chan() < D) {
      const uint32_t at = first(stride);
#pragma unroll
      for (int j = 0; j < CH; ++j) v[j] = *reinterpret_cast<const vec_t*>(reinterpret_cast<const char*>(p + j * STEP * stride) + at);
    } else {
      const vec_t z = {};
#pragma unroll
      for (int j = 0; j < CH; ++j) v[j] = z;
    }
  }
  // the rows for which there(row) holds, zeros for the others
  template <typename F>
  PF_DEV void load_some(const T* p, int stride, int D, F there) {
    const uint32_t at = first(stride);
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const vec_t z = {};
      v[j] = chan() < D && there(row(j))
                 ? *reinterpret_cast<const vec_t*>(reinterpret_cast<const char*>(p + j * STEP * stride) + at) : z;
    }
  }
  PF_DEV void store(L* lds, int stride) const {
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      L* const to = lds + row(j) * stride + chan();
      if constexpr (Mma<T>::SPLIT) {
        typename Mma<T>::quad_t q[3];
        const float x[4] = {v[j][0], v[j][1], v[j][2], v[j][3]};
        Mma<T>::put_any(x, q);
#pragma unroll
        for (int k = 0; k < 3; ++k) *reinterpret_cast<typename Mma<T>::quad_t*>(to + k * ROWS * stride) = q[k];
      } else {
        *reinterpret_cast<vec_t*>(to) = v[j];
      }
    }
  }
};

// Which of a tile's KT keys are seen, a bit each, the same in every wave.  `fetch` asks for a tile's mask
// bytes, `take` turns them into the bits an iteration later: nothing waits for them.
template <int KT>
struct Seen {
  static constexpr int W = KT / 64;
  uint64_t w[W];
  uint8_t byte[W];
  PF_DEV void fetch(int t, int len, const uint8_t* mask) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int key = t * KT + 64 * i + lane;
      byte[i] = key < len ? (mask ? mask[key] : 1) : 0;
    }
  }
  PF_DEV void take() {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = __ballot(byte[i] != 0);
  }
  PF_DEV bool all() const {
    uint64_t a = ~0ull;
#pragma unroll
    for (int i = 0; i < W; ++i) a &= w[i];
    return a == ~0ull;
  }
  // bits of keys 32 k .. + 31
  PF_DEV uint32_t part(int k) const { return (uint32_t)((W == 2 && k >= 2 ? w[W - 1] : w[0]) >> (32 * (k & 1))); }
  PF_DEV bool at(int key) const { return ((W == 2 && key >= 64 ? w[W - 1] : w[0]) >> (key & 63)) & 1; }
};

// Key tile t of one key head: rows of hidden keys are zeros (what stands there, NaN say, takes no part).
template <typename T, int DP, int KT>
PF_DEV void load_keys(Stage<T, DP, KT>& s, const T* base, int stride, int D, int t, const Seen<KT>& seen) {
  const T* p = base + (long)t * KT * stride;
  if (seen.all()) s.load(p, stride, D);
  else s.load_some(p, stride, D, [&](int row) __attribute__((always_inline)) { return seen.at(row); });
}

// Workgroup w runs on XCD w % 8: neighbouring ids go to one XCD, so the workgroups of a (batch, key head)
// share its keys and values in one L2 (4 x 2048 x 4096: 167 us, in launch order 178; windows 13.4 and 16.7).
PF_DEV int xcd_remap(int w, int total) {
  const int x = w % 8, q = total / 8, rem = total % 8;
  return x * q + min(x, rem) + w / 8;
}

struct Block { int rt, z, b, hk; };
PF_DEV Block block_of(const XaParams& p, int tiles) {
  const int id = xcd_remap(blockIdx.x, gridDim.x);
  const int rt = id % tiles, rest = id / tiles, z = rest % p.splits, bh = rest / p.splits;
  return {rt, z, bh / p.Hk, bh % p.Hk};
}

PF_DEV int length_of(const XaParams& p, int b) { return p.lens ? max(0, min(p.Lk, p.lens[b])) : p.Lk; }

// 4 elements that need not begin on a multiple of their size together
template <typename T>
struct Any4 { typedef T type __attribute__((ext_vector_type(4), aligned(sizeof(T)))); };

// bias[row, key .. key + 3] of a lane's query (0 outside the tensor); dense: neighbouring keys adjoin
template <typename B>
PF_DEV void load_bias4(const B* a, int key, int Lk, bool dense, long bk, float (&x)[4]) {
  if (dense && key + 3 < Lk) {
    const auto v = *reinterpret_cast<const typename Any4<B>::type*>(a + key);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = (float)v[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = key + e < Lk ? (float)a[(key + e) * bk] : 0.f;
  }
}
template <typename T>
PF_DEV void load_bias(const XaParams& p, const char* row, int key, bool ok, float (&x)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = 0.f;
  if (!ok) return;
  if (p.bias_f32) load_bias4(reinterpret_cast<const float*>(row), key, p.Lk, p.bk == 1, p.bk, x);
  else load_bias4(reinterpret_cast<const T*>(row), key, p.Lk, p.bk == 1, p.bk, x);
}
// its keys key0 .. + 3, + 8 .. + 11, ..: a lane's 16 values of a 32-key tile
template <typename T>
PF_DEV void load_bias16(const XaParams& p, const char* row, int key0, bool ok, float (&x)[16]) {
#pragma unroll
  for (int run = 0; run < 4; ++run) {
    float y[4];
    load_bias<T>(p, row, key0 + 8 * run, ok, y);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[4 * run + e] = y[e];
  }
}
// a lane's row of the bias
template <typename T>
PF_DEV const char* bias_row(const XaParams& p, int b, int head, int i) {
  return (const char*)p.bias + (b * p.bb + head * p.bh + i * p.bq) * (p.bias_f32 ? 4 : (long)sizeof(T));
}

// c s - m, the exponent of a probability without a bias.  fp32 tensors: the product is rounded before
// the difference, so the largest logit gives exactly 0 (a query that sees one key gets that value, bit
// for bit); of 16-bit tensors one fused step is as good (2^-24 of the logit) and half the work.
template <typename T>
PF_DEV float exponent(float s, float c, float m) {
  if constexpr (__is_same(T, float)) {
#pragma clang fp contract(off)
    const float x = s * c;
    return x - m;
  } else {
    return fmaf(s, c, -m);
  }
}

// 4 consecutive results of a row
template <typename T>
PF_DEV void store4(T* p, const float (&x)[4]) {
  typedef T quad __attribute__((ext_vector_type(4)));
  quad v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (T)x[e];
  *reinterpret_cast<quad*>(p) = v;
}

// ------------------------------------------------------------------------------ forward
// FEW = false: every wave over the tile's 64 keys with R tiles of 32 rows.  FEW = true (at most 32 rows): the
// waves share one 32-row tile and take 32 of the tile's 128 keys each; their results are joined through LDS
// (512 windows of 32 x 128: 13.5 us, as rows of a 128-row tile 15.5; 8 requests of one query: 10.4 and 12.0).
//
// LDS buffers of a tile: two, so that a tile needs one barrier (128 channels: 85 us, with one buffer 129), or
// one where the tiles are large and more workgroups per CU are worth more (single rows stream keys at memory's
// rate; fp32's three parts).
template <typename T, bool FEW>
constexpr int buffers() { return FEW || __is_same(T, float) ? 1 : 2; }

// Waves per SIMD that the forward kernel's registers are kept to: the most that holds its accumulators and
// the tile on its way without spilling.
template <typename T, int DP, bool BIAS, bool FEW, int R, bool WHOLE>
constexpr int fwd_waves() {
  if (WHOLE && DP <= 64) return FEW && DP == 32 ? 3 : 2;
  if (DP == 128) return FEW || __is_same(T, float) ? 1 : 2;
  if (R == 2) return 2;
  return __is_same(T, float) ? 2 : DP == 64 ? (BIAS ? 2 : FEW ? 3 : 4) : BIAS && !FEW ? 3 : 4;
}

// WHOLE (16-bit types): P enters the product with the values to fp32's accuracy.  A bias's gradient is
// dS = P (dP - delta) itself, fp32 as a rule, and delta = do . o of an o made from rounded P would leave it
// with 2^-9 or 2^-12 of delta.  (2 x 512 x 765, 16 heads x 24, fp16: 17.6 us.)
template <typename T, int DP, bool BIAS, bool FEW, int R, bool WHOLE>
__global__ __launch_bounds__(256, (fwd_waves<T, DP, BIAS, FEW, R, WHOLE>())) void xa_fwd_kernel(XaParams p) {
  using M = Mma<T>;
  constexpr int KT = FEW ? XA_KT_FEW : XA_KT, NSUB = FEW ? 1 : 2, DT = DP / 32;
  constexpr int KS = M::row_stride(DP), VS = M::col_stride(DP);
  extern __shared__ __align__(16) char smem[];
  typedef typename M::L L;
  constexpr int PK = KT * KS, PV = KT * VS, BUF = M::PARTS * (PK + PV), NBUF = buffers<T, FEW>();
  L* const ks0 = reinterpret_cast<L*>(smem);   // per buffer: the parts of the keys, then of the values
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, n = lane & 31, h = lane >> 5;
  constexpr int ROWS = FEW ? 32 : 128 * R;
  const Block blk = block_of(p, (p.rows + ROWS - 1) / ROWS);
  const int b = blk.b, hk = blk.hk;
  const int sub0 = FEW ? 32 * wid : 0;
  int row[R], i[R], head[R];   // a lane's rows
  bool row_ok[R];
  Frag<T, DP> q[R];
  const char* bias[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    row[r] = blk.rt * ROWS + (FEW ? 0 : 32 * (R * wid + r)) + n;
    row_ok[r] = row[r] < p.rows;
    i[r] = row_ok[r] ? row[r] / p.G : 0;
    head[r] = hk * p.G + (row_ok[r] ? row[r] - i[r] * p.G : 0);
    q[r].load((const T*)p.q + b * p.qb + (long)i[r] * p.ql + head[r] * p.qh, p.D, h, row_ok[r], p.neg);
    if constexpr (BIAS) bias[r] = bias_row<T>(p, b, head[r], i[r]);
  }
  const int len = length_of(p, b);
  const int t0 = blk.z * p.per, t1 = min(t0 + p.per, (len + KT - 1) / KT);
  const uint8_t* mask = p.mask ? p.mask + b * p.mb : nullptr;
  const T* const kb = (const T*)p.k + b * p.kb + hk * p.kh;
  const T* const vb = (const T*)p.v + b * p.vb + hk * p.vh;

  Stage<T, DP, KT> sk, sv;
  Seen<KT> now, next;
  auto load_tile = [&](int t, const Seen<KT>& seen) __attribute__((always_inline)) {
    load_keys(sk, kb, p.kl, p.D, t, seen);
    load_keys(sv, vb, p.vl, p.D, t, seen);
  };

  const float c = BIAS ? p.scale : p.scale * LOG2E;   // x in units of 1 (bias) or log2
  // the reference of the exponentials follows the maximum when that has grown by SLACK: p <= 2^8
  constexpr float SLACK = BIAS ? 5.f : 8.f;
  float m[R], l[R];                                   // l: this lane's half of the keys
  f32x16 o[R][DT];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -INFINITY, l[r] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[r][dt] = zero16();
  }

  // the next tile's bias is on its way while this one's softmax and product run
  float bs[NSUB][R][16];
  auto fetch_bias = [&](int t) __attribute__((always_inline)) {
    if constexpr (BIAS) {
#pragma unroll
      for (int u = 0; u < NSUB; ++u)
#pragma unroll
        for (int r = 0; r < R; ++r) load_bias16<T>(p, bias[r], t * KT + sub0 + 32 * u + 4 * h, row_ok[r], bs[u][r]);
    }
  };
  if (t0 < t1) {
    now.fetch(t0, len, mask);
    next.fetch(t0 + 1, len, mask);
    now.take();
    load_tile(t0, now);
    fetch_bias(t0);
    sk.store(ks0, KS);
    sv.store(ks0 + M::PARTS * PK, VS);
  }
  __syncthreads();
  for (int t = t0; t < t1; ++t) {
    const L* const ks = ks0 + (NBUF == 2 ? (t - t0) % 2 * BUF : 0);
    const L* const vs = ks + M::PARTS * PK;
    next.take();
    if (t + 1 < t1) load_tile(t + 1, next);
    Seen<KT> then;
    then.fetch(t + 2, len, mask);
    // the keys of this wave that are seen, bit j: key sub0 + j of the tile
    const uint64_t word = FEW ? now.part(wid) : now.w[0];
    f32x16 x[NSUB][R];
    if (word) {
#pragma unroll
      for (int u = 0; u < NSUB; ++u) {
        inner_rows<T, DP, R>(ks + (sub0 + 32 * u + n) * KS + M::E * h, PK, q, x[u]);
        if constexpr (BIAS) {
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int k = 0; k < 16; ++k) x[u][r][k] = fmaf(x[u][r][k], c, bs[u][r][k]);
        }
        const uint32_t w = (uint32_t)(word >> (FEW ? 0 : 32 * u));
        if (w != 0xffffffffu) {
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int k = 0; k < 16; ++k) x[u][r][k] = (w >> (4 * h) >> acc_row(k, 0)) & 1 ? x[u][r][k] : -INFINITY;
        }
      }
    }
    if (t + 1 < t1) fetch_bias(t + 1);
    if (word) {
      typename M::Packed pk[NSUB][R];
      typename M::Packed whole[NSUB][M::WHOLE];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < NSUB; ++u)
#pragma unroll
          for (int k = 0; k < 16; ++k) mx = fmaxf(mx, x[u][r][k]);
        mx = xor32_max(mx);
        if (!BIAS) mx *= c;
        if (__any(mx > m[r] + SLACK)) {
          const float m_new = fmaxf(m[r], mx);
          const float a = m_new > m[r] ? exp2_fast(BIAS ? (m[r] - m_new) * LOG2E : m[r] - m_new) : 1.f;
          l[r] *= a;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int k = 0; k < 16; ++k) o[r][dt][k] *= a;
          m[r] = m_new;
        }
        const float mu = m[r] == -INFINITY ? 0.f : m[r];   // nothing seen so far: every p is 0
#pragma unroll
        for (int u = 0; u < NSUB; ++u) {
          f32x16 pr;
#pragma unroll
          for (int k = 0; k < 16; ++k) pr[k] = exp2_fast(BIAS ? (x[u][r][k] - mu) * LOG2E : exponent<T>(x[u][r][k], c, mu));
          if constexpr (WHOLE) M::pack_whole(pr, whole[u]);
          else pk[u][r] = M::pack(pr);
          if constexpr (BIAS || M::SPLIT) {   // a bias's gradient wants P, and so the sum, to fp32
#pragma unroll
            for (int k = 0; k < 16; ++k) l[r] += pr[k];
          } else {
            l[r] = M::sum(pk[u][r], l[r]);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < NSUB; ++u) {
        if constexpr (WHOLE) M::template outer_sum<DT, M::WHOLE>(vs + (sub0 + 32 * u) * VS, VS, lane, whole[u], o[0]);
        else M::template outer<DT, R>(vs + (sub0 + 32 * u) * VS, PV, VS, lane, pk[u], o);
      }
    }
    if constexpr (NBUF == 1) __syncthreads();
    if (t + 1 < t1) {
      L* const to = ks0 + (NBUF == 2 ? (t + 1 - t0) % 2 * BUF : 0);
      sk.store(to, KS);
      sv.store(to + M::PARTS * PK, VS);
    }
    now = next, next = then;
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < R; ++r) l[r] = xor32_sum(l[r]);
  const long part_rows = (long)p.splits * p.B * p.Hk * p.rows;
  const long part_row0 = ((long)blk.z * p.B * p.Hk + (long)b * p.Hk + hk) * p.rows;

  if constexpr (FEW) {
    // join the four waves: their maxima and sums, then thread (row, 4 channels) adds the four parts
    constexpr int OS = DP + 4;
    float* const os = reinterpret_cast<float*>(smem);       // [4][32][OS]
    float* const ms = os + 4 * 32 * OS;                     // [4][32][2]
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int run = 0; run < 4; ++run) {
        const f32x4 v = {o[0][dt][4 * run], o[0][dt][4 * run + 1], o[0][dt][4 * run + 2], o[0][dt][4 * run + 3]};
        *reinterpret_cast<f32x4*>(os + (32 * wid + n) * OS + 32 * dt + 8 * run + 4 * h) = v;
      }
    if (h == 0) {
      ms[(32 * wid + n) * 2] = m[0];
      ms[(32 * wid + n) * 2 + 1] = l[0];
    }
    __syncthreads();
    const int tr = threadIdx.x >> 3, sub = threadIdx.x & 7, rr = blk.rt * ROWS + tr;
    if (rr >= p.rows) return;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, ms[(32 * w + tr) * 2]);
    float f[4], ll = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      // (a wave that saw nothing has sums of 0, or NaN where its scores were: that has to spread)
      const float mw = ms[(32 * w + tr) * 2];
      f[w] = mw == -INFINITY ? 0.f : exp2_fast(BIAS ? (mw - mm) * LOG2E : mw - mm);
      ll += f[w] * ms[(32 * w + tr) * 2 + 1];
    }
    const int ri = rr / p.G, rh = hk * p.G + rr - ri * p.G;
    const long row_at = ((long)b * p.Lq + ri) * p.H + rh;
    const float inv = ll > 0.f || ll != ll ? 1.f / ll : 0.f;
    for (int d = 4 * sub; d < p.D; d += 32) {
      float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] += f[w] * os[(32 * w + tr) * OS + d + e];
      if (p.splits > 1) {
        store4<float>(p.part + (part_row0 + rr) * p.D + d, a);
        continue;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] *= inv;
      store4<T>((T*)p.o + row_at * p.D + d, a);
      if (p.o32) store4<float>(p.o32 + row_at * p.D + d, a);
    }
    if (sub == 0) {
      if (p.splits > 1) {
        p.part[part_rows * p.D + 2 * (part_row0 + rr)] = mm;
        p.part[part_rows * p.D + 2 * (part_row0 + rr) + 1] = ll;
      } else if (p.st_m) {
        const long at = ((long)b * p.H + rh) * p.Lq + ri;
        p.st_m[at] = mm == -INFINITY ? 0.f : mm;
        p.st_l[at] = ll == 0.f ? INFINITY : __builtin_amdgcn_logf(ll);
      }
    }
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (!row_ok[r]) continue;
      const float inv = l[r] > 0.f || l[r] != l[r] ? 1.f / l[r] : 0.f;
      const long row_at = ((long)b * p.Lq + i[r]) * p.H + head[r];
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int run = 0; run < 4; ++run) {
          const int d = 32 * dt + 8 * run + 4 * h;
          if (d >= p.D) continue;
          float a[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) a[e] = o[r][dt][4 * run + e] * (p.splits > 1 ? 1.f : inv);
          if (p.splits > 1) {
            store4<float>(p.part + (part_row0 + row[r]) * p.D + d, a);
          } else {
            store4<T>((T*)p.o + row_at * p.D + d, a);
            if (p.o32) store4<float>(p.o32 + row_at * p.D + d, a);
          }
        }
      if (h == 0) {
        if (p.splits > 1) {
          p.part[part_rows * p.D + 2 * (part_row0 + row[r])] = m[r];
          p.part[part_rows * p.D + 2 * (part_row0 + row[r]) + 1] = l[r];
        } else if (p.st_m) {
          const long at = ((long)b * p.H + head[r]) * p.Lq + i[r];
          p.st_m[at] = m[r] == -INFINITY ? 0.f : m[r];
          p.st_l[at] = l[r] == 0.f ? INFINITY : __builtin_amdgcn_logf(l[r]);
        }
      }
    }
  }
}

// The splits of a row joined: `slices` threads for 4 channels, each over a contiguous part of the splits,
// then joined through LDS in order.  Eight splits a thread at least: a thread alone on 64 splits waits for
// memory again and again (32 rows x 8 heads over 8192 keys, both kernels: 13.5 us with 8 slices, 31.3 with
// 1), for few splits the second join costs more (12 splits: 11.1 us with 8 slices, 9.8 with 1).
inline int join_slices(int splits, int D) {
  int s = 1;
  while (16 * s <= splits && 2 * s * (D / 4) <= 256) s *= 2;
  return s;
}

template <typename T, bool BIAS>
__global__ __launch_bounds__(256) void xa_join_kernel(XaParams p, int slices) {
  __shared__ float sm[256], sl[256], sa[256][4];
  const int per = p.D / 4, per_row = per * slices, rows = 256 / per_row;
  const int r0 = (int)threadIdx.x / per_row, e = (int)threadIdx.x - r0 * per_row, slice = e / per, d = (e - slice * per) * 4;
  const long row = (long)blockIdx.x * rows + r0;   // (b, hk, r)
  const long all = (long)p.B * p.Hk * p.rows;
  const bool ok = r0 < rows && row < all;
  const float* ml = p.part + all * p.splits * p.D;
  float mm = -INFINITY, l = 0.f, a[4] = {0.f, 0.f, 0.f, 0.f};
  // what a part that saw nothing holds are zeros, or NaN where its scores were: that has to spread
  auto factor = [](float m, float top) __attribute__((always_inline)) {
    return m == -INFINITY ? 0.f : exp2_fast(BIAS ? (m - top) * LOG2E : m - top);
  };
  if (ok) {
    const int n = (p.splits + slices - 1) / slices, z0 = slice * n, z1 = min(z0 + n, p.splits);
#pragma unroll 4
    for (int z = z0; z < z1; ++z) mm = fmaxf(mm, ml[2 * (z * all + row)]);
#pragma unroll 4
    for (int z = z0; z < z1; ++z) {
      const float f = factor(ml[2 * (z * all + row)], mm);
      l += f * ml[2 * (z * all + row) + 1];
      const f32x4 v = *reinterpret_cast<const f32x4*>(p.part + (z * all + row) * p.D + d);
#pragma unroll
      for (int k = 0; k < 4; ++k) a[k] += f * v[k];
    }
  }
  if (slices > 1) {
    sm[threadIdx.x] = mm, sl[threadIdx.x] = l;
#pragma unroll
    for (int k = 0; k < 4; ++k) sa[threadIdx.x][k] = a[k];
    __syncthreads();
    if (!ok || slice) return;
    for (int s = 1; s < slices; ++s) mm = fmaxf(mm, sm[threadIdx.x + s * per]);
    l = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) a[k] = 0.f;
    for (int s = 0; s < slices; ++s) {
      const int at = (int)threadIdx.x + s * per;
      const float f = factor(sm[at], mm);
      l += f * sl[at];
#pragma unroll
      for (int k = 0; k < 4; ++k) a[k] += f * sa[at][k];
    }
  } else if (!ok) {
    return;
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) a[k] *= inv;
  const long bh = row / p.rows;
  const int r = (int)(row - bh * p.rows), i = r / p.G, b = (int)(bh / p.Hk), head = (int)(bh % p.Hk) * p.G + r - i * p.G;
  const long at = (((long)b * p.Lq + i) * p.H + head) * p.D + d;
  store4<T>((T*)p.o + at, a);
  if (p.o32) store4<float>(p.o32 + at, a);
  if (d == 0 && p.st_m) {
    const long s = ((long)b * p.H + head) * p.Lq + i;
    p.st_m[s] = mm == -INFINITY ? 0.f : mm;
    p.st_l[s] = l == 0.f ? INFINITY : __builtin_amdgcn_logf(l);
  }
}

template <typename T, int DP, bool FEW>
size_t fwd_lds() {
  constexpr int KT = FEW ? XA_KT_FEW : XA_KT;
  const size_t tiles = (size_t)KT * (Mma<T>::row_stride(DP) + Mma<T>::col_stride(DP)) * 2 * Mma<T>::PARTS * buffers<T, FEW>();
  const size_t join = FEW ? (size_t)4 * 32 * (DP + 4 + 2) * 4 : 0;
  return tiles > join ? tiles : join;
}

template <typename T, int DP, bool BIAS, bool FEW, int R, bool WHOLE = false>
int fwd_launch(const XaParams& p, hipStream_t st) {
  const size_t lds = fwd_lds<T, DP, FEW>();
  const auto kernel = xa_fwd_kernel<T, DP, BIAS, FEW, R, WHOLE>;
  if (int rc = pf_reserve_lds((const void*)kernel, lds, "xa_fwd_kernel")) return rc;
  constexpr int ROWS = FEW ? 32 : 128 * R;
  const int tiles = (p.rows + ROWS - 1) / ROWS;
  kernel<<<(unsigned)((long)tiles * p.splits * p.B * p.Hk), 256, lds, st>>>(p);
  PF_CHECK_LAUNCH("xa_fwd_kernel");
  if (p.splits > 1) {
    const int slices = join_slices(p.splits, p.D), rows = 256 / (p.D / 4 * slices);
    xa_join_kernel<T, BIAS><<<(unsigned)(((long)p.B * p.Hk * p.rows + rows - 1) / rows), 256, 0, st>>>(p, slices);
    PF_CHECK_LAUNCH("xa_join_kernel");
  }
  return PF_OK;
}

// Whether the waves of a workgroup may share a row tile: three parts of 128 keys x 128 channels exceed LDS.
template <typename T, int DP>
constexpr bool has_few() { return !(Mma<T>::SPLIT && DP == 128); }

template <typename T, int DP>
int fwd_dp(const XaParams& p, hipStream_t st) {
  if constexpr (!Mma<T>::SPLIT) {
    if (p.bias && p.whole) return p.few ? fwd_launch<T, DP, true, true, 1, true>(p, st) : fwd_launch<T, DP, true, false, 1, true>(p, st);
  }
  if constexpr (has_few<T, DP>()) {
    if (p.few) return p.bias ? fwd_launch<T, DP, true, true, 1>(p, st) : fwd_launch<T, DP, false, true, 1>(p, st);
  }
  if (p.bias) return fwd_launch<T, DP, true, false, 1>(p, st);
  if constexpr (DP == 64 && !Mma<T>::SPLIT) {
    if (p.wide) return fwd_launch<T, DP, false, false, 2>(p, st);
  }
  return fwd_launch<T, DP, false, false, 1>(p, st);
}

template <typename T>
int fwd_type(const XaParams& p, hipStream_t st) {
  return p.D <= 32 ? fwd_dp<T, 32>(p, st) : p.D <= 64 ? fwd_dp<T, 64>(p, st) : fwd_dp<T, 128>(p, st);
}

}  // namespace
