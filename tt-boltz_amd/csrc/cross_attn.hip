// Cross attention entry points: argument checks, the split of the work, and the sum of the logits'
// gradient over a bias's broadcast dimensions (kernels: cross_kernels.h, cross_bwd.h).
#include "cross_attn.h"

namespace {

// Workgroups wanted: two for each of 256 CUs, what most kernels' registers and LDS allow.  (dk, dv of 2 x 2048
// keys, 4 key heads x 128 channels: 176 us, with one per CU 262; the parts of more are more to join.)
constexpr long WANT = 512;

struct Split { int splits, per; };

// `tiles` of one axis split so that `base` workgroups become up to WANT (a few more than that wait for all
// the others: fp32 dk, dv of 184 workgroups 51 us in 3 parts, 42 in 2), at least `least` tiles each
Split split_of(long base, long tiles, long least) {
  long s = base > 0 ? WANT / base : 1;
  if (s > tiles / least) s = tiles / least;
  if (s > 64) s = 64;
  if (s < 1) s = 1;
  const long per = (tiles + s - 1) / s;
  return {(int)(per > 0 ? (tiles + per - 1) / per : 1), (int)(per > 0 ? per : 1)};
}

long up256(long b) { return (b + 255) & ~255l; }

int check(const pf_cross_attn_args* a, const char* fn) {
  if (!a) return pf_fail(PF_E_INVALID, "%s: null args", fn);
  if (a->dtype < PF_FP32 || a->dtype > PF_BF16) return pf_fail(PF_E_INVALID, "%s: unknown dtype %d", fn, a->dtype);
  if (a->B < 0 || a->Lq < 0 || a->Lk < 0 || a->H < 0 || a->Hk < 1 || a->H % a->Hk)
    return pf_fail(PF_E_INVALID, "%s: bad shape (B=%d Lq=%d Lk=%d H=%d Hk=%d; H a multiple of Hk)", fn, a->B, a->Lq, a->Lk, a->H,
                   a->Hk);
  if (a->D < 8 || a->D > 128 || a->D % 8) return pf_fail(PF_E_INVALID, "%s: D must be a multiple of 8 up to 128 (got %d)", fn, a->D);
  if (!__builtin_isfinite(a->scale)) return pf_fail(PF_E_INVALID, "%s: scale is not finite", fn);
  if ((long)a->Lq * (a->H / a->Hk) > 0x3fffffffl || a->Lk > 0x3fffffff)
    return pf_fail(PF_E_INVALID, "%s: too long (Lq=%d Lk=%d)", fn, a->Lq, a->Lk);
  if (a->bias && a->bias_dtype != PF_FP32 && a->bias_dtype != a->dtype)
    return pf_fail(PF_E_INVALID, "%s: the bias must be fp32 or the tensors' type", fn);
  return PF_OK;
}

int check_data(const pf_cross_attn_args* a, const char* fn) {
  const long unit = 16 / pf_elem_size(a->dtype);
  if (!a->q || (a->Lk > 0 && (!a->k || !a->v))) return pf_fail(PF_E_INVALID, "%s: null pointer", fn);
  if (!pf_aligned16(a->q) || !pf_aligned16(a->k) || !pf_aligned16(a->v))
    return pf_fail(PF_E_INVALID, "%s: q, k and v must be 16-byte aligned", fn);
  for (long s : {a->q_b, a->q_l, a->q_h, a->k_b, a->k_l, a->k_h, a->v_b, a->v_l, a->v_h})
    if (s % unit) return pf_fail(PF_E_INVALID, "%s: strides must be multiples of 16 bytes", fn);
  for (long s : {a->q_l, a->k_l, a->v_l, (long)a->H * a->D})
    if (s < 0 || s >= 1l << 22) return pf_fail(PF_E_INVALID, "%s: row strides must be below 2^22 elements (got %ld)", fn, s);
  return PF_OK;
}

XaParams params_of(const pf_cross_attn_args* a) {
  XaParams p = {};
  p.B = a->B, p.Lq = a->Lq, p.Lk = a->Lk, p.H = a->H, p.Hk = a->Hk, p.D = a->D, p.G = a->H / a->Hk;
  p.rows = p.G * p.Lq;
  p.neg = a->scale < 0.f, p.grad_scale = a->scale;
  p.scale = __builtin_fabsf(a->scale);
  if (p.scale < 1e-30f) p.scale = 1e-30f;   // 0: all logits equal (0 times a hidden key's -inf would not be)
  p.q = a->q, p.k = a->k, p.v = a->v;
  p.qb = a->q_b, p.ql = (int)a->q_l, p.qh = a->q_h, p.kb = a->k_b, p.kl = (int)a->k_l, p.kh = a->k_h;
  p.vb = a->v_b, p.vl = (int)a->v_l, p.vh = a->v_h;
  p.bias = a->bias, p.bias_f32 = a->bias_dtype == PF_FP32;
  p.bb = a->bias_b, p.bh = a->bias_h, p.bq = a->bias_q, p.bk = a->bias_k;
  p.mask = a->mask, p.mb = a->mask_b, p.lens = a->k_lens;
  p.o = a->o, p.o32 = a->o32;
  if (a->stats) p.st_m = a->stats, p.st_l = a->stats + (long)a->B * a->H * a->Lq;
  p.few = p.rows <= 32 && !(a->dtype == PF_FP32 && p.D > 64);
  p.splits = p.per = 1;
  const int longest = p.rows > p.Lk ? p.rows : p.Lk;
  p.chunks = longest > 64 * 32 ? 64 : (longest + 31) / 32;
  return p;
}

// the split over key tiles of the forward and the dq kernel.  Three tiles of 16 bits a part at least: 2 x 512
// x 765, 16 heads, four parts of 3 tiles 17.4 us, three of 4 20.6; 64 rows x 8 heads over 8192 keys 14.9 in
// 32 or 42 parts, 17.3 in 64.  An fp32 tile is worth several (2, 1 and 4 within a microsecond of each other).
Split key_split(const XaParams& p, int dtype) {
  const long rows = p.few ? 32 : 128, kt = p.few ? XA_KT_FEW : XA_KT;
  return split_of((p.rows + rows - 1) / rows * p.B * p.Hk, (p.Lk + kt - 1) / kt, p.few ? 1 : dtype == PF_FP32 ? 2 : 3);
}
// the split over row tiles of the dk, dv kernel
Split row_split(const XaParams& p, int dtype) {
  const int rt = xa_rt(p.D <= 32 ? 32 : p.D <= 64 ? 64 : 128, dtype == PF_FP32);
  return split_of((long)(p.Lk + XA_KEYS - 1) / XA_KEYS * p.B * p.Hk, ((long)p.Lq + rt - 1) / rt * p.G, dtype == PF_FP32 ? 2 : 256 / rt);
}

long fwd_part_bytes(const XaParams& p, const Split& s) {
  return s.splits > 1 ? (long)s.splits * p.B * p.Hk * p.rows * (p.D + 2) * 4 : 0;
}

struct BwdLayout { long delta, amax, ds, part, bytes; };

BwdLayout bwd_layout(const pf_cross_attn_args* a, const XaParams& p) {
  BwdLayout l;
  l.delta = 0;
  l.amax = up256((long)p.B * p.H * p.Lq * 4);
  l.ds = l.amax + up256((long)p.B * p.Hk * p.chunks * 8);
  const bool own = a->dbias_B > 0 && !(a->bias_dtype == PF_FP32 && a->dbias_B == a->B && a->dbias_H == a->H);
  l.part = l.ds + (own ? up256((long)p.B * p.H * p.Lq * p.Lk * 4) : 0);
  const Split ks = key_split(p, a->dtype), rs = row_split(p, a->dtype);
  const long dq = ks.splits > 1 ? (long)ks.splits * p.B * p.Lq * p.H * p.D * 4 : 0;
  const long dkv = rs.splits > 1 ? 2l * rs.splits * p.B * p.Lk * p.Hk * p.D * 4 : 0;
  l.bytes = l.part + (dq > dkv ? dq : dkv);
  return l;
}

// A launch holds fewer than 2^32 threads: 2^24 workgroups (splits are made where there are few), and
// element-wise launches of a thread for four channels.
bool grid_fits(const XaParams& p, bool backward) {
  const long rt = ((long)p.rows + (p.few ? 31 : 127)) / (p.few ? 32 : 128);
  const long kt = backward ? ((long)p.Lk + XA_KEYS - 1) / XA_KEYS : 0, chunks = backward ? p.chunks : 0;
  long most = rt > kt ? rt : kt;
  if (chunks > most) most = chunks;
  if (most >= 1l << 24 || most * p.B >= 1l << 24 || most * p.B * p.Hk >= 1l << 24) return false;
  const long q = (long)p.B * p.Lq * p.H, k = (long)p.B * p.Lk * p.Hk;
  return q < 1l << 31 && k < 1l << 31 && q * p.D < 1l << 34 && k * p.D < 1l << 34;
}

// dbias[bb, hh, e] = sum of ds[b, h, e] over the dimensions of size 1, e < Lq Lk: lanes on neighbouring
// elements, each adding its batch elements and heads in order.
template <typename T>
__global__ __launch_bounds__(256) void xa_dbias_kernel(const float* __restrict__ ds, T* __restrict__ out, int B, int H, int oB,
                                                       int oH, long n) {
  const long e = (long)blockIdx.x * 256 + threadIdx.x;
  if (e >= n) return;
  const int ob = blockIdx.y / oH, oh = blockIdx.y % oH;
  const int b0 = oB == 1 ? 0 : ob, b1 = oB == 1 ? B : ob + 1, h0 = oH == 1 ? 0 : oh, h1 = oH == 1 ? H : oh + 1;
  float a = 0.f;
  for (int b = b0; b < b1; ++b)
#pragma unroll 4
    for (int h = h0; h < h1; ++h) a += ds[((long)b * H + h) * n + e];
  out[(long)blockIdx.y * n + e] = (T)a;
}

template <typename T>
int dbias_launch(const float* ds, void* out, const pf_cross_attn_args* a, hipStream_t st) {
  const long n = (long)a->Lq * a->Lk;
  xa_dbias_kernel<T><<<dim3((unsigned)((n + 255) / 256), (unsigned)(a->dbias_B * a->dbias_H)), 256, 0, st>>>(
      ds, (T*)out, a->B, a->H, a->dbias_B, a->dbias_H, n);
  PF_CHECK_LAUNCH("xa_dbias_kernel");
  return PF_OK;
}

}  // namespace

extern "C" size_t pf_cross_attn_workspace_size(const pf_cross_attn_args* a) {
  if (check(a, "pf_cross_attn_workspace_size")) return 0;
  const XaParams p = params_of(a);
  return (size_t)fwd_part_bytes(p, key_split(p, a->dtype));
}

extern "C" int pf_cross_attn_fwd(const pf_cross_attn_args* a) {
  const char* fn = "pf_cross_attn_fwd";
  if (int rc = check(a, fn)) return rc;
  if (a->B == 0 || a->Lq == 0 || a->H == 0) return PF_OK;
  if (int rc = check_data(a, fn)) return rc;
  if (!a->o) return pf_fail(PF_E_INVALID, "%s: null pointer", fn);
  if (!pf_aligned16(a->o) || !pf_aligned16(a->o32)) return pf_fail(PF_E_INVALID, "%s: o must be 16-byte aligned", fn);
  XaParams p = params_of(a);
  if (!grid_fits(p, false)) return pf_fail(PF_E_INVALID, "%s: too large (B=%d Lq=%d Lk=%d H=%d)", fn, a->B, a->Lq, a->Lk, a->H);
  const Split s = key_split(p, a->dtype);
  const size_t need = (size_t)fwd_part_bytes(p, s);
  if (need && (!a->workspace || a->workspace_bytes < need))
    return pf_fail(PF_E_INVALID, "%s: workspace too small (%zu < %zu bytes)", fn, a->workspace_bytes, need);
  if (need && !pf_aligned16(a->workspace)) return pf_fail(PF_E_INVALID, "%s: workspace not 16-byte aligned", fn);
  p.splits = s.splits, p.per = s.per, p.part = (float*)a->workspace;
  p.whole = a->o32_whole != 0;
  // Two row tiles per wave (64 channels without a bias: each LDS read serves two products) where
  // workgroups of 256 rows still come to two per CU: 16 heads x 2048 rows x 4096 keys, batch 4 (512
  // workgroups) 185 against 198 us, batch 2 (256) 113 against 109.
  p.wide = s.splits == 1 && (long)(p.rows + 255) / 256 * p.B * p.Hk >= 512;
  hipStream_t st = (hipStream_t)a->stream;
  return a->dtype == PF_FP32 ? pf_xa_fwd_fp32(p, st) : a->dtype == PF_FP16 ? pf_xa_fwd_fp16(p, st) : pf_xa_fwd_bf16(p, st);
}

extern "C" size_t pf_cross_attn_bwd_workspace_size(const pf_cross_attn_args* a) {
  if (check(a, "pf_cross_attn_bwd_workspace_size")) return 0;
  return (size_t)bwd_layout(a, params_of(a)).bytes;
}

extern "C" int pf_cross_attn_bwd(const pf_cross_attn_args* a) {
  const char* fn = "pf_cross_attn_bwd";
  if (int rc = check(a, fn)) return rc;
  if (a->dbias && (!a->bias || (a->dbias_B != 1 && a->dbias_B != a->B) || (a->dbias_H != 1 && a->dbias_H != a->H)))
    return pf_fail(PF_E_INVALID, "%s: dbias [%d][%d] does not belong to a bias of B=%d H=%d", fn, a->dbias_B, a->dbias_H, a->B, a->H);
  if ((a->dbias != nullptr) != (a->dbias_B > 0)) return pf_fail(PF_E_INVALID, "%s: dbias and dbias_B do not agree", fn);
  if (a->B == 0 || a->Lq == 0 || a->H == 0)
    return a->Lk == 0 || a->B == 0 || (!a->dk && !a->dbias) ? PF_OK
                                                            : pf_fail(PF_E_INVALID, "%s: no queries (the caller clears dk and dv)", fn);
  if (int rc = check_data(a, fn)) return rc;
  const float* o32 = a->dtype == PF_FP32 ? (const float*)a->o : a->o32;
  if (!a->dout || !o32 || !a->stats) return pf_fail(PF_E_INVALID, "%s: dout, the unrounded o and the statistics are needed", fn);
  if ((a->dk != nullptr) != (a->dv != nullptr)) return pf_fail(PF_E_INVALID, "%s: dk and dv come together", fn);
  if (a->dbias && !a->dq) return pf_fail(PF_E_INVALID, "%s: dbias comes with dq", fn);
  if (!pf_aligned16(a->dout) || !pf_aligned16(o32) || !pf_aligned16(a->dq) || !pf_aligned16(a->dk) || !pf_aligned16(a->dv) ||
      !pf_aligned16(a->dbias) || !pf_aligned16(a->workspace))
    return pf_fail(PF_E_INVALID, "%s: gradients and workspace must be 16-byte aligned", fn);
  XaParams p = params_of(a);
  if (!grid_fits(p, true)) return pf_fail(PF_E_INVALID, "%s: too large (B=%d Lq=%d Lk=%d H=%d)", fn, a->B, a->Lq, a->Lk, a->H);
  if (a->dbias && ((long)a->Lq * a->Lk > (1l << 32) - 256 || (long)a->dbias_B * a->dbias_H > 65535))
    return pf_fail(PF_E_INVALID, "%s: bias gradient too large (Lq=%d Lk=%d B=%d H=%d)", fn, a->Lq, a->Lk, a->dbias_B, a->dbias_H);
  const BwdLayout l = bwd_layout(a, p);
  if (!a->workspace || a->workspace_bytes < (size_t)l.bytes)
    return pf_fail(PF_E_INVALID, "%s: workspace too small (%zu < %ld bytes)", fn, a->workspace_bytes, l.bytes);
  hipStream_t st = (hipStream_t)a->stream;
  char* ws = (char*)a->workspace;
  float* delta = (float*)(ws + l.delta);
  float* amax = (float*)(ws + l.amax);
  p.dout = a->dout, p.amax = amax, p.part = (float*)(ws + l.part);
  p.dq = a->dq, p.dk = a->dk, p.dv = a->dv;
  const int t = a->dtype;
  p.delta = delta;
  if (int rc = t == PF_FP32 ? pf_xa_delta_fp32(p, amax, st) : t == PF_FP16 ? pf_xa_delta_fp16(p, amax, st) : pf_xa_delta_bf16(p, amax, st))
    return rc;
  if (a->dq) {
    const Split s = key_split(p, a->dtype);
    XaParams d = p;
    d.splits = s.splits, d.per = s.per;
    const bool own = a->dbias && !(a->bias_dtype == PF_FP32 && a->dbias_B == a->B && a->dbias_H == a->H);
    d.ds = own ? (float*)(ws + l.ds) : (float*)a->dbias;
    if (int rc = t == PF_FP32 ? pf_xa_dq_fp32(d, st) : t == PF_FP16 ? pf_xa_dq_fp16(d, st) : pf_xa_dq_bf16(d, st)) return rc;
    if (own && a->Lk > 0) {
      const int bt = a->bias_dtype;
      if (int rc = bt == PF_FP32 ? dbias_launch<float>(d.ds, a->dbias, a, st)
                                 : bt == PF_FP16 ? dbias_launch<half_t>(d.ds, a->dbias, a, st)
                                                 : dbias_launch<bhalf_t>(d.ds, a->dbias, a, st))
        return rc;
    }
  }
  if (a->dk && a->Lk > 0) {
    const Split s = row_split(p, t);
    XaParams d = p;
    d.splits = s.splits, d.per = s.per;
    if (int rc = t == PF_FP32 ? pf_xa_dkv_fp32(d, st) : t == PF_FP16 ? pf_xa_dkv_fp16(d, st) : pf_xa_dkv_bf16(d, st)) return rc;
  }
  return PF_OK;
}
