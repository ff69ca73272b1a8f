// Backward pass of cross attention, included once per element type after cross_kernels.h (see there).
//
// Two kernels, neither with atomics, so gradients are the same bits each time: xa_dq_kernel (a
// workgroup has queries, walks over keys; also writes the logits' gradient where a bias wants it) and
// xa_dkv_kernel (a workgroup has 128 keys, walks over the rows of all heads that share them).
//
// fp16: dS and P are products' operands and far smaller than 1, where fp16 has few bits left (below
// 2^-14) or none (2^-25).  P is taken 2^15 times larger, and dS by the power of two that brings its
// bound max|do_i| max|v_j| 2 to 2^14 or less; both factors are divided out of the fp32 sums.
//
// Measured (one MI355X, us a launch): 2 x 2048 queries x 2048 keys of which about three quarters are seen, 16
// heads over 4, 128 channels, bf16: dq 115, dk and dv 176 and 12.5 for the sum of their four splits, delta 10
// (50 MB).  2 x 512 x 765, 16 heads x 24, fp16 with a bias whose gradient is wanted: dq 31 (50 MB of bias and
// dS), dk and dv 26, delta 5, sums 4.5 each.  fp32, 384 x 2900 x 8 heads x 48: dq 36, dk and dv 43, delta 4,
// sums 5 each.  Both large kernels hold two waves per SIMD (accumulators and operands fill the registers),
// which leaves LDS reads and MFMAs of one wave waiting for each other part of the time.
#pragma once
#include "cross_kernels.h"

namespace {

template <typename T>
constexpr bool SCALED = __is_same(T, half_t);

// power of two that brings 2 |do| |v| to (2^13, 2^14] (1 where the bound is 0 or not finite)
PF_DEV float ds_scale(const XaParams& p, int b, int hk) {
  const float* a = p.amax + ((long)b * p.Hk + hk) * p.chunks * 2;
  const int lane = threadIdx.x & 63;
  float g = lane < p.chunks ? a[2 * lane] : 0.f, v = lane < p.chunks ? a[2 * lane + 1] : 0.f;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) g = fmaxf(g, __shfl_xor(g, o)), v = fmaxf(v, __shfl_xor(v, o));
  const float bound = 2.f * __fsqrt_rn(g) * __fsqrt_rn(v);
  if (!(bound > 0.f) || !(bound < 3.0e38f)) return 1.f;
  int e;
  (void)frexpf(bound, &e);
  return ldexpf(1.f, max(-100, min(14 - e, 100)));
}

// ------------------------------------------------------------------------------ delta
// delta_i = do_i . o_i in fp32 from the unrounded o, 8 lanes a row; fp16:
// also the largest |do_i|^2 and |v_j|^2 of the workgroup's part of a key head (ds_scale joins the parts).
// blockIdx.x: batch element and key head, and its part (at most 64).
template <typename T>
__global__ __launch_bounds__(256) void xa_delta_kernel(XaParams p, float* __restrict__ amax) {
  __shared__ float top[2][4];
  const int sub = threadIdx.x & 7;
  const int bh = blockIdx.x / p.chunks, chunk = blockIdx.x - bh * p.chunks, hk = bh % p.Hk;
  const long b = bh / p.Hk;
  const float* o32 = p.o32 ? p.o32 : (const float*)p.o;
  float g_top = 0.f, v_top = 0.f;
  for (int r = chunk * 32 + (threadIdx.x >> 3); r < p.rows; r += 32 * p.chunks) {
    const int i = r / p.G, head = hk * p.G + r - i * p.G;
    const long at = ((b * p.Lq + i) * p.H + head) * p.D;
    float dot = 0.f, sq = 0.f;
    for (int d = 4 * sub; d < p.D; d += 32) {
      typedef T quad __attribute__((ext_vector_type(4)));
      const quad g4 = *reinterpret_cast<const quad*>((const T*)p.dout + at + d);
      const f32x4 o4 = *reinterpret_cast<const f32x4*>(o32 + at + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        dot = fmaf((float)g4[e], o4[e], dot);
        sq = fmaf((float)g4[e], (float)g4[e], sq);
      }
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      dot += __shfl_xor(dot, o);
      sq += __shfl_xor(sq, o);
    }
    if (sub == 0) p.delta[(b * p.H + head) * p.Lq + i] = dot;
    g_top = fmaxf(g_top, sq);
  }
  if constexpr (SCALED<T>) {
    const int len = length_of(p, (int)b);
    for (int key = chunk * 32 + (threadIdx.x >> 3); key < len; key += 32 * p.chunks) {
      float sq = 0.f;
      if (!p.mask || p.mask[b * p.mb + key]) {
        const T* v = (const T*)p.v + b * p.vb + (long)key * p.vl + hk * p.vh;
        for (int d = 4 * sub; d < p.D; d += 32) {
          typedef T quad __attribute__((ext_vector_type(4)));
          const quad v4 = *reinterpret_cast<const quad*>(v + d);
#pragma unroll
          for (int e = 0; e < 4; ++e) sq = fmaf((float)v4[e], (float)v4[e], sq);
        }
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) sq += __shfl_xor(sq, o);
      v_top = fmaxf(v_top, sq);
    }
#pragma unroll
    for (int o = 8; o < 64; o <<= 1) g_top = fmaxf(g_top, __shfl_xor(g_top, o)), v_top = fmaxf(v_top, __shfl_xor(v_top, o));
    if ((threadIdx.x & 63) == 0) top[0][threadIdx.x >> 6] = g_top, top[1][threadIdx.x >> 6] = v_top;
    __syncthreads();
    if (threadIdx.x < 2) {
      const float* t = top[threadIdx.x];
      amax[(long)blockIdx.x * 2 + threadIdx.x] = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
    }
  }
}

// ------------------------------------------------------------------------------ dq, dS
template <typename T, int DP, bool BIAS, bool FEW>
constexpr int dq_waves() {
  if (DP == 128) return FEW || __is_same(T, float) ? 1 : 2;
  return __is_same(T, float) || DP == 64 || BIAS ? 2 : FEW ? 3 : 4;
}

template <typename T, int DP, bool BIAS, bool FEW>
__global__ __launch_bounds__(256, (dq_waves<T, DP, BIAS, FEW>())) void xa_dq_kernel(XaParams p) {
  using M = Mma<T>;
  constexpr int KT = FEW ? XA_KT_FEW : XA_KT, NSUB = FEW ? 1 : 2, DT = DP / 32;
  constexpr int KS = M::both_stride(DP);
  extern __shared__ __align__(16) char smem[];
  typedef typename M::L L;
  constexpr int PK = KT * KS, BUF = 2 * M::PARTS * PK, NBUF = buffers<T, FEW>();
  L* const ks0 = reinterpret_cast<L*>(smem);   // per buffer: the parts of the keys, then of the values
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, n = lane & 31, h = lane >> 5;
  constexpr int ROWS = FEW ? 32 : 128;
  const Block blk = block_of(p, (p.rows + ROWS - 1) / ROWS);
  const int b = blk.b, hk = blk.hk;
  const int r = blk.rt * ROWS + (FEW ? 0 : 32 * wid) + n;
  const bool row_ok = r < p.rows;
  const int i = row_ok ? r / p.G : 0, head = hk * p.G + (row_ok ? r - i * p.G : 0);
  const int sub0 = FEW ? 32 * wid : 0;
  const long row_at = ((long)b * p.Lq + i) * p.H + head;
  Frag<T, DP> q, g;
  q.load((const T*)p.q + b * p.qb + (long)i * p.ql + head * p.qh, p.D, h, row_ok, p.neg);
  g.load((const T*)p.dout + row_at * p.D, p.D, h, row_ok);
  const long stat = ((long)b * p.H + head) * p.Lq + i;
  const float m = row_ok ? p.st_m[stat] : 0.f, ll = row_ok ? p.st_l[stat] : INFINITY;
  const float m_ll = m + ll;   // 16-bit types without a bias (2^-24 of the logit is nothing there)
  const float delta = row_ok ? p.delta[stat] : 0.f;
  const float sf = SCALED<T> ? ds_scale(p, b, hk) : 1.f;
  const char* bias = nullptr;
  if constexpr (BIAS) bias = bias_row<T>(p, b, head, i);
  float* const ds = p.ds && row_ok ? p.ds + stat * p.Lk : nullptr;
  const int len = length_of(p, b);
  // the logits' gradient has zeros at hidden keys, so its writer goes on to the end
  const int t0 = blk.z * p.per, t1 = min(t0 + p.per, ((p.ds ? p.Lk : len) + KT - 1) / KT);
  const uint8_t* mask = p.mask ? p.mask + b * p.mb : nullptr;
  const T* const kb = (const T*)p.k + b * p.kb + hk * p.kh;
  const T* const vb = (const T*)p.v + b * p.vb + hk * p.vh;

  Stage<T, DP, KT> sk, sv;
  Seen<KT> now, next;
  auto load_tile = [&](int t, const Seen<KT>& seen) __attribute__((always_inline)) {
    load_keys(sk, kb, p.kl, p.D, t, seen);
    load_keys(sv, vb, p.vl, p.D, t, seen);
  };

  const float c = BIAS ? p.scale : p.scale * LOG2E;
  f32x16 dq[1][DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) dq[0][dt] = zero16();

  float bs[NSUB][16];
  auto fetch_bias = [&](int t, int u) __attribute__((always_inline)) {
    if constexpr (BIAS) load_bias16<T>(p, bias, t * KT + sub0 + 32 * u + 4 * h, row_ok, bs[u]);
  };
  if (t0 < t1) {
    now.fetch(t0, len, mask);
    next.fetch(t0 + 1, len, mask);
    now.take();
    load_tile(t0, now);
#pragma unroll
    for (int u = 0; u < NSUB; ++u) fetch_bias(t0, u);
    sk.store(ks0, KS);
    sv.store(ks0 + M::PARTS * PK, KS);
  }
  __syncthreads();
  for (int t = t0; t < t1; ++t) {
    const L* const ks = ks0 + (NBUF == 2 ? (t - t0) % 2 * BUF : 0);
    const L* const vs = ks + M::PARTS * PK;
    next.take();
    if (t + 1 < t1) load_tile(t + 1, next);
    Seen<KT> then;
    then.fetch(t + 2, len, mask);
    const uint64_t word = FEW ? now.part(wid) : now.w[0];
#pragma unroll
    for (int u = 0; u < NSUB; ++u) {
      const uint32_t word_u = (uint32_t)(word >> (FEW ? 0 : 32 * u));
      if (!word_u && !p.ds) {
        if (t + 1 < t1) fetch_bias(t + 1, u);
        continue;
      }
      const int key0 = t * KT + sub0 + 32 * u + 4 * h;
      const int at = (sub0 + 32 * u + n) * KS + M::E * h;
      const f32x16 s = inner<T, DP>(ks + at, PK, q, zero16());
      f32x16 y;
#pragma unroll
      for (int k = 0; k < 16; ++k) y[k] = -delta;
      y = inner<T, DP>(vs + at, PK, g, y);
#pragma unroll
      for (int k = 0; k < 16; ++k)
        y[k] *= exp2_fast(BIAS ? fmaf(fmaf(s[k], c, bs[u][k]) - m, LOG2E, -ll)
                               : M::SPLIT ? exponent<T>(s[k], c, m) - ll : fmaf(s[k], c, -m_ll));
      if (t + 1 < t1) fetch_bias(t + 1, u);
      if (word_u != 0xffffffffu) {
#pragma unroll
        for (int k = 0; k < 16; ++k) y[k] = (word_u >> (4 * h) >> acc_row(k, 0)) & 1 ? y[k] : 0.f;
      }
      if (ds) {
#pragma unroll
        for (int run = 0; run < 4; ++run) {
          const int key = key0 + 8 * run;
          if (key + 3 < p.Lk) {
            const typename Any4<float>::type v = {y[4 * run], y[4 * run + 1], y[4 * run + 2], y[4 * run + 3]};
            *reinterpret_cast<typename Any4<float>::type*>(ds + key) = v;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (key + e < p.Lk) ds[key + e] = y[4 * run + e];
          }
        }
      }
      if constexpr (SCALED<T>) {
#pragma unroll
        for (int k = 0; k < 16; ++k) y[k] *= sf;
      }
      if (word_u) {
        const typename M::Packed pk[1] = {M::pack(y)};
        M::template outer<DT, 1>(ks + (sub0 + 32 * u) * KS, PK, KS, lane, pk, dq);
      }
    }
    if constexpr (NBUF == 1) __syncthreads();
    if (t + 1 < t1) {
      L* const to = ks0 + (NBUF == 2 ? (t + 1 - t0) % 2 * BUF : 0);
      sk.store(to, KS);
      sv.store(to + M::PARTS * PK, KS);
    }
    now = next, next = then;
    __syncthreads();
  }

  const float out_scale = p.grad_scale / sf;
  if constexpr (FEW) {
    constexpr int OS = DP + 4;
    float* const os = reinterpret_cast<float*>(smem);       // [4][32][OS]
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int run = 0; run < 4; ++run) {
        const f32x4 v = {dq[0][dt][4 * run], dq[0][dt][4 * run + 1], dq[0][dt][4 * run + 2], dq[0][dt][4 * run + 3]};
        *reinterpret_cast<f32x4*>(os + (32 * wid + n) * OS + 32 * dt + 8 * run + 4 * h) = v;
      }
    __syncthreads();
    const int row = threadIdx.x >> 3, sub = threadIdx.x & 7, rr = blk.rt * ROWS + row;
    if (rr >= p.rows) return;
    const int ri = rr / p.G, rh = hk * p.G + rr - ri * p.G;
    const long to = ((long)b * p.Lq + ri) * p.H + rh;
    for (int d = 4 * sub; d < p.D; d += 32) {
      float a[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) a[e] += os[(32 * w + row) * OS + d + e];
        a[e] *= out_scale;
      }
      if (p.splits > 1) store4<float>(p.part + ((long)blk.z * p.B * p.Lq * p.H + to) * p.D + d, a);
      else store4<T>((T*)p.dq + to * p.D + d, a);
    }
  } else {
    if (!row_ok) return;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int run = 0; run < 4; ++run) {
        const int d = 32 * dt + 8 * run + 4 * h;
        if (d >= p.D) continue;
        float a[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = dq[0][dt][4 * run + e] * out_scale;
        if (p.splits > 1) store4<float>(p.part + ((long)blk.z * p.B * p.Lq * p.H + row_at) * p.D + d, a);
        else store4<T>((T*)p.dq + row_at * p.D + d, a);
      }
  }
}

// ------------------------------------------------------------------------------ dk, dv
// 4 waves x 32 keys; a tile is RT consecutive queries of one head, the heads of the key head one after
// the other.  A wave's values stay in registers; its keys do too where those suffice for two waves per
// SIMD, else (128 channels, fp32 from 64) they are read from LDS for each tile
// (fp32: without padding, so that two workgroups share a CU's LDS; the 16-byte pieces of a row are
// permuted by the row's low bits instead, and 16 rows still land on distinct banks).
template <typename T, int DP>
constexpr bool keys_in_lds() { return DP == 128 || (Mma<T>::SPLIT && DP == 64); }

// 128 channels of 16 bits: half of the values as well, and one buffer, so that 80 KB of LDS and 256
// registers hold a workgroup without spilling (a reload waits for every load before it: 230 -> 185 us at
// 8192 rows x 2048 keys, 2 x 4 key heads).
template <typename T, int DP>
constexpr int dkv_buffers() { return DP == 128 ? 1 : buffers<T, false>(); }
template <typename T, int DP>
constexpr int v_steps() { return DP == 128 && !Mma<T>::SPLIT ? 4 : DP / 16; }

template <typename T, int DP, bool BIAS>
__global__ __launch_bounds__(256, DP == 128 && __is_same(T, float) ? 1 : 2) void xa_dkv_kernel(XaParams p) {
  using M = Mma<T>;
  constexpr int RT = xa_rt(DP, __is_same(T, float)), DT = DP / 32, S = M::both_stride(DP);
  typedef typename M::L L;
  constexpr int PT = RT * S, STATS = 3 * RT * 2, NBUF = dkv_buffers<T, DP>(), BUF = 2 * M::PARTS * PT + STATS;
  constexpr bool KLDS = keys_in_lds<T, DP>();
  extern __shared__ __align__(16) char smem[];
  L* const buf0 = reinterpret_cast<L*>(smem);   // per buffer: q, do, then fp32 [3][RT] maximum, log2 of the sum, delta
  L* const kl = buf0 + NBUF * BUF;              // parts of the keys
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, n = lane & 31, h = lane >> 5;
  const Block blk = block_of(p, (p.Lk + XA_KEYS - 1) / XA_KEYS);
  const int b = blk.b, hk = blk.hk;
  const int key = blk.rt * XA_KEYS + 32 * wid + n;
  const int len = length_of(p, b);
  const uint8_t* mask = p.mask ? p.mask + b * p.mb : nullptr;
  const bool seen = key < len && (!mask || mask[key]);
  Frag<T, DP> kf, vf;
  kf.load((const T*)p.k + b * p.kb + (long)key * p.kl + hk * p.kh, p.D, h, seen, p.neg);
  vf.load((const T*)p.v + b * p.vb + (long)key * p.vl + hk * p.vh, p.D, h, seen);
  constexpr int KLS = M::SPLIT ? DP : M::row_stride(DP);
  auto kl_at = [&](int s) __attribute__((always_inline)) {
    const int piece = M::SPLIT ? (2 * s + h) ^ (n & (DP / 8 - 1)) : 2 * s + h;
    return kl + (32 * wid + n) * KLS + 8 * piece;
  };
  if constexpr (KLDS) {
#pragma unroll
    for (int s = 0; s < Frag<T, DP>::S; ++s)
#pragma unroll
      for (int k = 0; k < M::PARTS; ++k) *reinterpret_cast<typename M::part_t*>(kl_at(s) + k * XA_KEYS * KLS) = kf.f[s].p[k];
  }
  constexpr int VST = v_steps<T, DP>(), VLS = DP - 16 * VST + 8;
  L* const vl_row = kl + (KLDS ? M::PARTS * XA_KEYS * KLS : 0) + (32 * wid + n) * VLS + 8 * h;
  if constexpr (VST < DP / 16) {
#pragma unroll
    for (int s = VST; s < DP / 16; ++s) *reinterpret_cast<typename M::part_t*>(vl_row + 16 * (s - VST)) = vf.f[s].p[0];
  }
  const float sf = SCALED<T> ? ds_scale(p, b, hk) : 1.f;
  // 16-bit types without a bias: maximum and log2 of the sum as one (2^-24 of the logit is nothing there)
  constexpr bool ONE_STAT = !BIAS && !M::SPLIT;
  constexpr float P_UP = SCALED<T> ? 15.f : 0.f, P_FACTOR = SCALED<T> ? 32768.f : 1.f;
  const float ds_f = sf / P_FACTOR;
  const bool any_seen = __any(seen), all_seen = __all(seen);
  const int head_tiles = (p.Lq + RT - 1) / RT;
  // nothing of this workgroup's keys is seen by anyone: its sums are zero
  const int t0 = blk.z * p.per, t1 = blk.rt * XA_KEYS < len ? min(t0 + p.per, p.G * head_tiles) : t0;

  Stage<T, DP, RT> sq, sg;
  float stat = 0.f;   // threads 0 .. 3 RT: one value of the tile's statistics
  const int sw = threadIdx.x / RT, sr = threadIdx.x % RT;
  auto load_tile = [&](int t) __attribute__((always_inline)) {
    const int g = t / head_tiles, i0 = (t - g * head_tiles) * RT, head = hk * p.G + g, left = p.Lq - i0;
    const T* qp = (const T*)p.q + b * p.qb + (long)i0 * p.ql + head * p.qh;
    const T* gp = (const T*)p.dout + (((long)b * p.Lq + i0) * p.H + head) * p.D;
    if (left >= RT) {
      sq.load(qp, p.ql, p.D);
      sg.load(gp, p.H * p.D, p.D);
    } else {
      auto there = [&](int row) __attribute__((always_inline)) { return row < left; };
      sq.load_some(qp, p.ql, p.D, there);
      sg.load_some(gp, p.H * p.D, p.D, there);
    }
    if (sw < 3) {
      stat = sw == 1 ? INFINITY : 0.f;   // a row behind the last: P = 0
      const long at = ((long)b * p.H + head) * p.Lq + i0 + sr;
      if constexpr (ONE_STAT) {
        if (sw == 0) stat = sr < left ? p.st_m[at] + (p.st_l[at] - P_UP) : INFINITY;
        else if (sw == 2 && sr < left) stat = p.delta[at];
      } else if (sr < left) {
        stat = (sw == 0 ? p.st_m : sw == 1 ? p.st_l : p.delta)[at];
      }
    }
  };
  auto store_tile = [&](int t) __attribute__((always_inline)) {
    L* const to = buf0 + (NBUF == 2 ? (t - t0) % 2 * BUF : 0);
    sq.store(to, S);
    sg.store(to + M::PARTS * PT, S);
    if (sw < 3) reinterpret_cast<float*>(to + 2 * M::PARTS * PT)[sw * RT + sr] = stat;
  };

  const float c = BIAS ? p.scale : p.scale * LOG2E;
  f32x16 dk[1][DT], dv[1][DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) dk[0][dt] = zero16(), dv[0][dt] = zero16();

  float bs[RT / 32][16];
  auto fetch_bias = [&](int t, int u) __attribute__((always_inline)) {
    if constexpr (BIAS) {
      const int g = t / head_tiles, i0 = (t - g * head_tiles) * RT + 32 * u, head = hk * p.G + g;
      const long ba = b * p.bb + head * p.bh + (i0 + 4 * h) * p.bq + key * p.bk;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        bs[u][k] = 0.f;
        if (i0 + acc_row(k, h) < p.Lq && seen) {
          const long e = ba + acc_row(k, 0) * p.bq;
          bs[u][k] = p.bias_f32 ? ((const float*)p.bias)[e] : (float)((const T*)p.bias)[e];
        }
      }
    }
  };
  if (t0 < t1) {
    load_tile(t0);
#pragma unroll
    for (int u = 0; u < RT / 32; ++u) fetch_bias(t0, u);
    store_tile(t0);
  }
  __syncthreads();
  for (int t = t0; t < t1; ++t) {
    const L* const qs = buf0 + (NBUF == 2 ? (t - t0) % 2 * BUF : 0);
    const L* const gs = qs + M::PARTS * PT;
    const float* const st = reinterpret_cast<const float*>(gs + M::PARTS * PT);
    if (t + 1 < t1) load_tile(t + 1);
    if (any_seen) {
#pragma unroll
      for (int u = 0; u < RT / 32; ++u) {
        const int at = (32 * u + n) * S + M::E * h;
        f32x16 pr = zero16(), dp;
        if constexpr (KLDS) {
#pragma unroll
          for (int s = 0; s < Frag<T, DP>::S; ++s)
            pr = M::mma(M::load(qs + at + 16 * s, PT), M::load(kl_at(s), XA_KEYS * KLS), pr);
        } else {
          pr = inner<T, DP>(qs + at, PT, kf, pr);
        }
#pragma unroll
        for (int run = 0; run < 4; ++run) {
          const f32x4 m = *reinterpret_cast<const f32x4*>(st + 32 * u + 8 * run + 4 * h);
          f32x4 ll = {};
          if constexpr (!ONE_STAT) ll = *reinterpret_cast<const f32x4*>(st + RT + 32 * u + 8 * run + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int k = 4 * run + e;
            pr[k] = exp2_fast(BIAS ? fmaf(fmaf(pr[k], c, bs[u][k]) - m[e], LOG2E, P_UP - ll[e])
                                   : ONE_STAT ? fmaf(pr[k], c, -m[e]) : exponent<T>(pr[k], c, m[e]) - ll[e]);
          }
        }
        if (t + 1 < t1) fetch_bias(t + 1, u);
        if (!all_seen) {
#pragma unroll
          for (int k = 0; k < 16; ++k) pr[k] = seen ? pr[k] : 0.f;
        }
        const typename M::Packed pv[1] = {M::pack(pr)};
        M::template outer<DT, 1>(gs + 32 * u * S, PT, S, lane, pv, dv);
#pragma unroll
        for (int run = 0; run < 4; ++run) {
          const f32x4 dl = *reinterpret_cast<const f32x4*>(st + 2 * RT + 32 * u + 8 * run + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) dp[4 * run + e] = -dl[e];
        }
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
          dp = M::mma(M::load(gs + at + 16 * s, PT), s < VST ? vf.f[s] : M::load(vl_row + 16 * (s - VST), 0), dp);
#pragma unroll
        for (int k = 0; k < 16; ++k) dp[k] = pr[k] * (SCALED<T> ? dp[k] * ds_f : dp[k]);
        const typename M::Packed pd[1] = {M::pack(dp)};
        M::template outer<DT, 1>(qs + 32 * u * S, PT, S, lane, pd, dk);
      }
    }
    if constexpr (NBUF == 1) __syncthreads();
    if (t + 1 < t1) store_tile(t + 1);
    __syncthreads();
  }

  if (key >= p.Lk) return;
  const float k_scale = p.grad_scale / sf, v_scale = 1.f / P_FACTOR;
  const long at = ((long)b * p.Lk + key) * p.Hk + hk, all = (long)p.B * p.Lk * p.Hk;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int run = 0; run < 4; ++run) {
      const int d = 32 * dt + 8 * run + 4 * h;
      if (d >= p.D) continue;
      float x[4], y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = seen ? dk[0][dt][4 * run + e] * k_scale : 0.f;
        y[e] = seen ? dv[0][dt][4 * run + e] * v_scale : 0.f;
      }
      if (p.splits > 1) {
        store4<float>(p.part + (2l * blk.z * all + at) * p.D + d, x);
        store4<float>(p.part + ((2l * blk.z + 1) * all + at) * p.D + d, y);
      } else {
        store4<T>((T*)p.dk + at * p.D + d, x);
        store4<T>((T*)p.dv + at * p.D + d, y);
      }
    }
}

// out = the sum over `splits` of part[z * step + e], e < n, four elements a thread; blockIdx.y = 1: the
// second result, its parts n behind the first's
template <typename T>
__global__ __launch_bounds__(256) void xa_sum_kernel(const float* __restrict__ part, long step, int splits, T* __restrict__ out0,
                                                     T* __restrict__ out1, long n) {
  T* const out = blockIdx.y ? out1 : out0;
  part += blockIdx.y * n;
  const long e = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (e >= n) return;
  float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int z = 0; z < splits; ++z) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(part + z * step + e);
#pragma unroll
    for (int k = 0; k < 4; ++k) a[k] += v[k];
  }
  store4<T>(out + e, a);
}

template <typename T>
int sum_launch(const float* part, long step, int splits, void* out0, void* out1, long n, hipStream_t st) {
  xa_sum_kernel<T><<<dim3((unsigned)((n + 1023) / 1024), out1 ? 2 : 1), 256, 0, st>>>(part, step, splits, (T*)out0, (T*)out1, n);
  PF_CHECK_LAUNCH("xa_sum_kernel");
  return PF_OK;
}

template <typename T, int DP, bool BIAS, bool FEW>
int dq_launch(const XaParams& p, hipStream_t st) {
  constexpr int KT = FEW ? XA_KT_FEW : XA_KT;
  const size_t tiles = (size_t)2 * KT * Mma<T>::both_stride(DP) * 2 * Mma<T>::PARTS * buffers<T, FEW>(),
               join = FEW ? (size_t)4 * 32 * (DP + 4) * 4 : 0, lds = tiles > join ? tiles : join;
  if (int rc = pf_reserve_lds((const void*)xa_dq_kernel<T, DP, BIAS, FEW>, lds, "xa_dq_kernel")) return rc;
  const int rt = (p.rows + (FEW ? 31 : 127)) / (FEW ? 32 : 128);
  xa_dq_kernel<T, DP, BIAS, FEW><<<(unsigned)((long)rt * p.splits * p.B * p.Hk), 256, lds, st>>>(p);
  PF_CHECK_LAUNCH("xa_dq_kernel");
  const long n = (long)p.B * p.Lq * p.H * p.D;
  return p.splits > 1 ? sum_launch<T>(p.part, n, p.splits, p.dq, nullptr, n, st) : PF_OK;
}

template <typename T, int DP>
int dq_dp(const XaParams& p, hipStream_t st) {
  if constexpr (has_few<T, DP>()) {
    if (p.few) return p.bias ? dq_launch<T, DP, true, true>(p, st) : dq_launch<T, DP, false, true>(p, st);
  }
  return p.bias ? dq_launch<T, DP, true, false>(p, st) : dq_launch<T, DP, false, false>(p, st);
}

template <typename T>
int dq_type(const XaParams& p, hipStream_t st) {
  return p.D <= 32 ? dq_dp<T, 32>(p, st) : p.D <= 64 ? dq_dp<T, 64>(p, st) : dq_dp<T, 128>(p, st);
}

template <typename T, int DP, bool BIAS>
int dkv_launch(const XaParams& p, hipStream_t st) {
  constexpr int RT = xa_rt(DP, __is_same(T, float)), S = Mma<T>::both_stride(DP);
  const size_t lds = dkv_buffers<T, DP>() * ((size_t)4 * Mma<T>::PARTS * RT * S + 3 * RT * 4) +
                     (keys_in_lds<T, DP>() ? (size_t)2 * Mma<T>::PARTS * XA_KEYS * (Mma<T>::SPLIT ? DP : Mma<T>::row_stride(DP)) : 0) +
                     (v_steps<T, DP>() < DP / 16 ? (size_t)2 * XA_KEYS * (DP - 16 * v_steps<T, DP>() + 8) : 0);
  if (int rc = pf_reserve_lds((const void*)xa_dkv_kernel<T, DP, BIAS>, lds, "xa_dkv_kernel")) return rc;
  const int tiles = (p.Lk + XA_KEYS - 1) / XA_KEYS;
  xa_dkv_kernel<T, DP, BIAS><<<(unsigned)((long)tiles * p.splits * p.B * p.Hk), 256, lds, st>>>(p);
  PF_CHECK_LAUNCH("xa_dkv_kernel");
  if (p.splits == 1) return PF_OK;
  const long n = (long)p.B * p.Lk * p.Hk * p.D;
  return sum_launch<T>(p.part, 2 * n, p.splits, p.dk, p.dv, n, st);
}

template <typename T, int DP>
int dkv_dp(const XaParams& p, hipStream_t st) {
  return p.bias ? dkv_launch<T, DP, true>(p, st) : dkv_launch<T, DP, false>(p, st);
}

template <typename T>
int dkv_type(const XaParams& p, hipStream_t st) {
  return p.D <= 32 ? dkv_dp<T, 32>(p, st) : p.D <= 64 ? dkv_dp<T, 64>(p, st) : dkv_dp<T, 128>(p, st);
}

template <typename T>
int delta_type(const XaParams& p, float* amax, hipStream_t st) {
  xa_delta_kernel<T><<<(unsigned)((long)p.chunks * p.B * p.Hk), 256, 0, st>>>(p, amax);
  PF_CHECK_LAUNCH("xa_delta_kernel");
  return PF_OK;
}

}  // namespace
