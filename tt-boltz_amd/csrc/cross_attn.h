// Cross attention on gfx950: what the host entry points (cross_attn.hip) and the kernels, one source
// per element type (cross_fp32.hip, cross_fp16.hip, cross_bf16.hip), share.
#pragma once
#include "pf_elem.h"

struct XaParams {
  int B, Lq, Lk, H, Hk, D, G;    // G = H / Hk heads share a key head
  int rows;                      // G * Lq rows of a key head: row r is query r / G of head hk G + r % G
  float scale;                   // |scale| (at least 1e-30); `neg`: q is negated as it is loaded
  int neg;
  float grad_scale;              // the caller's scale, a factor of dq and dk
  const void *q, *k, *v;
  long qb, qh, kb, kh, vb, vh;   // strides in elements, channels contiguous
  int ql, kl, vl;                // (from row to row: below 2^22)
  const void* bias;
  int bias_f32;                  // fp32, else the element type
  long bb, bh, bq, bk;
  const uint8_t* mask;           // [B] rows of Lk bytes, mb apart; 0 = hidden
  long mb;
  const int* lens;               // [B]
  void* o;                       // [B][Lq][H][D]
  float* o32;                    // the same before rounding (for the backward pass of 16-bit types), or null
  float *st_m, *st_l;            // [B][H][Lq]: a row's maximum and log2 of its sum (+inf: nothing seen), or null
  float* part;                   // splits > 1: partial results
  int splits, per;               // key tiles (dkv: row tiles) per split
  int few;                       // the waves of a workgroup share a 32-row tile
  int wide;                      // forward: two 32-row tiles per wave
  int whole;                     // forward, 16-bit types with a bias: o32 to fp32's accuracy
  // backward
  const void* dout;              // [B][Lq][H][D]
  float* delta;                  // [B][H][Lq]
  const float* amax;             // [B][Hk][chunks][2]: largest |dout_i|^2 and |v_j|^2 of a chunk (fp16)
  int chunks;                    // <= 64
  float* ds;                     // [B][H][Lq][Lk] gradient of the logits, or null
  void *dq, *dk, *dv;            // contiguous
};

constexpr int XA_KT = 64, XA_KT_FEW = 128;    // keys per tile
constexpr int XA_KEYS = 128;                  // keys per workgroup of the dk, dv kernel
constexpr int xa_rt(int dp, bool fp32) { return dp == 128 || fp32 ? 32 : 64; }   // its rows per tile

int pf_xa_fwd_fp32(const XaParams& p, hipStream_t st);
int pf_xa_delta_fp32(const XaParams& p, float* amax, hipStream_t st);
int pf_xa_dq_fp32(const XaParams& p, hipStream_t st);
int pf_xa_dkv_fp32(const XaParams& p, hipStream_t st);
int pf_xa_fwd_fp16(const XaParams& p, hipStream_t st);
int pf_xa_delta_fp16(const XaParams& p, float* amax, hipStream_t st);
int pf_xa_dq_fp16(const XaParams& p, hipStream_t st);
int pf_xa_dkv_fp16(const XaParams& p, hipStream_t st);
int pf_xa_fwd_bf16(const XaParams& p, hipStream_t st);
int pf_xa_delta_bf16(const XaParams& p, float* amax, hipStream_t st);
int pf_xa_dq_bf16(const XaParams& p, hipStream_t st);
int pf_xa_dkv_bf16(const XaParams& p, hipStream_t st);
