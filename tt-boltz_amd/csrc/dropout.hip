// Residual dropout with a counter-based generator (get_dropout_mask, tt_bio/boltz2.py:293-304, and
// the z + dropout * update of tt_bio/reference.py:877-903) for gfx950.
//
//   out[e] = r[e] + (u(g(e)) >= t ? x[e] / (1 - p) : 0),   t = p 2^32,
// u(g) = word g % 4 of Philox4x32-10 (Salmon, Moraes, Dror and Shaw, SC 2011) at counter
// (g / 4, offset) under the key `seed`; g is the element, or the (batch, row) or (batch, column) of
// a pair tensor.  The mask is a function of (seed, offset, g) alone, so the backward pass makes it
// again (x = the gradient, r = none) and nothing of it is ever stored.
//
// Memory's rate bounds it.  Measured (one MI355X): 33.5 M bf16 elements with residual 29 us (201 MB: 6.9 TB/s,
// part of it from cache; 37 from memory), its gradient 24; 512 x 512 x 128 fp32 by rows or columns 67 us
// (370 MB: 5.5 TB/s), a quarter of x not being read.
#include "pf_elem.h"

namespace {

struct Words { uint32_t w[4]; };

PF_DEV Words philox(uint64_t seed, uint64_t counter, uint64_t offset) {
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
  uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)b;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

struct DropShape {
  uint64_t total;        // elements
  uint64_t threshold;    // kept where a word is at least this (2^32: nothing is)
  float scale;           // 1 / (1 - p)
  uint64_t seed, offset;
  const uint64_t* seed_at;   // the seed in device memory (read when the kernel runs), or null
  uint32_t rows, cols, channels;   // I, J, C of a shared mask
};

template <typename T, int N>
PF_DEV void drop_store(const T* r, T* out, uint64_t e, const float (&y)[N]) {
  float a[N];
  if (r) {
    load_elems<T, N>(r + e, a);
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] += y[i];
    store_elems<T, N>(out + e, a);
  } else {
    store_elems<T, N>(out + e, y);
  }
}

// One mask value per element.  N elements a thread (16 bytes, or 1 where a pointer allows no more: N = 1
// makes a whole counter for each element, as do the last few of a number that N does not divide).  A second
// step a thread costs 31.5 us for 29, the smallest sizes (64 K elements) 3.0 for 2.4.
template <typename T, int N>
__global__ __launch_bounds__(256) void dropout_elem_kernel(const T* __restrict__ x, const T* __restrict__ r,
                                                           T* __restrict__ out, DropShape p) {
  const uint64_t e = ((uint64_t)blockIdx.x * 256 + threadIdx.x) * N;
  if (e >= p.total) return;
  const uint64_t seed = p.seed_at ? *p.seed_at : p.seed;
  if (N == 1 || e + N > p.total) {
    for (uint64_t k = e; k < p.total && k < e + N; ++k) {
      const Words w = philox(seed, k / 4, p.offset);
      const uint32_t c = (uint32_t)k & 3, lo = c & 1 ? w.w[1] : w.w[0], hi = c & 1 ? w.w[3] : w.w[2];
      const float y[1] = {(c & 2 ? hi : lo) >= p.threshold ? (float)x[k] * p.scale : 0.f};
      drop_store<T, 1>(r, out, k, y);
    }
    return;
  }
  float v[N];
  load_elems<T, N>(x + e, v);
#pragma unroll
  for (int q = 0; q < N / 4; ++q) {
    const Words w = philox(seed, e / 4 + q, p.offset);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[4 * q + i] = w.w[i] >= p.threshold ? v[4 * q + i] * p.scale : 0.f;
  }
  drop_store<T, N>(r, out, e, v);
}

// One mask value per (batch, row): blockIdx.y counts them (in steps of gridDim.y), so the generator
// runs on the scalar unit, and a dropped row of x is not read at all.  U steps a thread: two 67.7 us at 512 x
// 512 x 128 fp32 and 8.4 at 256 x 256 x 128 bf16, four 71.2 and 8.5, one 64.2 and 9.4.
template <typename T, int N, int U>
__global__ __launch_bounds__(256) void dropout_row_kernel(const T* __restrict__ x, const T* __restrict__ r,
                                                          T* __restrict__ out, DropShape p) {
  const uint64_t seed = p.seed_at ? *p.seed_at : p.seed;
  const uint64_t len = (uint64_t)p.cols * p.channels, groups = p.total / len;
  const uint64_t j0 = ((uint64_t)blockIdx.x * (256 * U) + threadIdx.x) * N;
  for (uint64_t g = blockIdx.y; g < groups; g += gridDim.y) {
    const Words w = philox(seed, g / 4, p.offset);
    const uint32_t c = (uint32_t)g & 3, lo = c & 1 ? w.w[1] : w.w[0], hi = c & 1 ? w.w[3] : w.w[2];
    const bool keep = (c & 2 ? hi : lo) >= p.threshold;
    float v[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t j = j0 + (uint64_t)u * 256 * N;
#pragma unroll
      for (int i = 0; i < N; ++i) v[u][i] = 0.f;
      if (keep && j < len) {
        load_elems<T, N>(x + g * len + j, v[u]);
#pragma unroll
        for (int i = 0; i < N; ++i) v[u][i] *= p.scale;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t j = j0 + (uint64_t)u * 256 * N;
      if (j < len) drop_store<T, N>(r, out, g * len + j, v[u]);
    }
  }
}

// One mask value per (batch, column): a thread makes the value of its column once and walks down
// ROWS rows with it (two 66.6 us and 8.9 at the sizes above, four 70.3 and 9.1, one 64.3 and 9.8).
template <typename T, int N, int ROWS>
__global__ __launch_bounds__(256) void dropout_col_kernel(const T* __restrict__ x, const T* __restrict__ r,
                                                          T* __restrict__ out, DropShape p) {
  const uint64_t seed = p.seed_at ? *p.seed_at : p.seed;
  const uint64_t len = (uint64_t)p.cols * p.channels;
  const uint32_t row_blocks = (p.rows + ROWS - 1) / ROWS;
  const uint64_t steps = p.total / len / p.rows * row_blocks;
  const uint64_t j = ((uint64_t)blockIdx.x * 256 + threadIdx.x) * N;
  if (j >= len) return;
  for (uint64_t s = blockIdx.y; s < steps; s += gridDim.y) {
    const uint64_t b = s / row_blocks;
    const uint32_t i0 = (uint32_t)(s - b * row_blocks) * ROWS;
    const uint64_t g = b * p.cols + j / p.channels;
    const Words w = philox(seed, g / 4, p.offset);
    const uint32_t c = (uint32_t)g & 3, lo = c & 1 ? w.w[1] : w.w[0], hi = c & 1 ? w.w[3] : w.w[2];
    const bool keep = (c & 2 ? hi : lo) >= p.threshold;
    const uint64_t e0 = (b * p.rows + i0) * len + j;
    float v[ROWS][N];
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[u][i] = 0.f;
      if (keep && i0 + u < p.rows) {
        load_elems<T, N>(x + e0 + u * len, v[u]);
#pragma unroll
        for (int i = 0; i < N; ++i) v[u][i] *= p.scale;
      }
    }
#pragma unroll
    for (int u = 0; u < ROWS; ++u)
      if (i0 + u < p.rows) drop_store<T, N>(r, out, e0 + u * len, v[u]);
  }
}

unsigned blocks_of(uint64_t n, uint64_t per) { return (unsigned)((n + per - 1) / per); }

template <typename T, int N>
int launch(const void* xv, const void* rv, void* ov, const DropShape& p, int shared, hipStream_t st) {
  const T *x = (const T*)xv, *r = (const T*)rv;
  T* out = (T*)ov;
  constexpr unsigned MOST_Y = 65535;
  const uint64_t len = (uint64_t)p.cols * p.channels;
  if (shared == PF_DROP_ELEMENT) {
    dropout_elem_kernel<T, N><<<blocks_of(p.total, 256 * N), 256, 0, st>>>(x, r, out, p);
  } else if (shared == PF_DROP_ROW) {
    constexpr int U = 2;
    const uint64_t groups = p.total / len;
    dropout_row_kernel<T, N, U><<<dim3(blocks_of(len, 256 * U * N), (unsigned)(groups < MOST_Y ? groups : MOST_Y)), 256, 0,
                                  st>>>(x, r, out, p);
  } else {
    constexpr int ROWS = 2;
    const uint64_t steps = p.total / len / p.rows * ((p.rows + ROWS - 1) / ROWS);
    dropout_col_kernel<T, N, ROWS><<<dim3(blocks_of(len, 256 * N), (unsigned)(steps < MOST_Y ? steps : MOST_Y)), 256, 0,
                                     st>>>(x, r, out, p);
  }
  PF_CHECK_LAUNCH("dropout_kernel");
  return PF_OK;
}

template <typename T>
int launch_type(const void* x, const void* r, void* out, const DropShape& p, int shared, hipStream_t st) {
  constexpr int N = Vec16<T>::N;
  const uint64_t inner = shared == PF_DROP_ELEMENT ? N : shared == PF_DROP_ROW ? (uint64_t)p.cols * p.channels : p.channels;
  if (pf_aligned16(x) && pf_aligned16(r) && pf_aligned16(out)) {
    if (inner % N == 0) return launch<T, N>(x, r, out, p, shared, st);
    // 8 bytes of 16-bit types: 512 x 512 x 132 bf16 by columns 32 us, one element a thread 92
    if constexpr (N == 8) {
      if (inner % 4 == 0) return launch<T, 4>(x, r, out, p, shared, st);
    }
  }
  if (p.total > (1ull << 32) - 256)   // a launch holds fewer than 2^32 threads
    return pf_fail(PF_E_INVALID, "pf_dropout_add_fwd: 2^32 elements need 16-byte aligned tensors");
  return launch<T, 1>(x, r, out, p, shared, st);
}

}  // namespace

extern "C" int pf_dropout_add_fwd(const pf_dropout_args* a) {
  if (!a) return pf_fail(PF_E_INVALID, "pf_dropout_add_fwd: null args");
  if (a->dtype < PF_FP32 || a->dtype > PF_BF16) return pf_fail(PF_E_INVALID, "pf_dropout_add_fwd: unknown dtype %d", a->dtype);
  if (a->shared < PF_DROP_ELEMENT || a->shared > PF_DROP_COLUMN)
    return pf_fail(PF_E_INVALID, "pf_dropout_add_fwd: unknown sharing %d", a->shared);
  if (!(a->p >= 0.0 && a->p <= 1.0)) return pf_fail(PF_E_INVALID, "pf_dropout_add_fwd: p must be in [0, 1] (got %g)", a->p);
  if (a->B < 0 || a->I < 0 || a->J < 0 || a->C < 0 || a->I > 0x7fffffff || a->J > 0x7fffffff || a->C > 0x7fffffff)
    return pf_fail(PF_E_INVALID, "pf_dropout_add_fwd: bad shape (B=%ld I=%ld J=%ld C=%ld)", a->B, a->I, a->J, a->C);
  unsigned long long total = 1;
  for (long d : {a->B, a->I, a->J, a->C})
    if (__builtin_mul_overflow(total, (unsigned long long)d, &total) || total > (1ull << 32))
      return pf_fail(PF_E_INVALID, "pf_dropout_add_fwd: more than 2^32 elements (B=%ld I=%ld J=%ld C=%ld)", a->B, a->I, a->J, a->C);
  if (total == 0) return PF_OK;
  if (!a->x || !a->out) return pf_fail(PF_E_INVALID, "pf_dropout_add_fwd: null pointer");
  const uint64_t threshold = (uint64_t)__builtin_rint(a->p * 4294967296.0);
  const DropShape p{total, threshold, a->p < 1.0 ? (float)(1.0 / (1.0 - a->p)) : 0.f, a->seed, a->offset,
                    (const uint64_t*)a->seed_at, (uint32_t)a->I, (uint32_t)a->J, (uint32_t)a->C};
  hipStream_t st = (hipStream_t)a->stream;
  if (a->dtype == PF_FP32) return launch_type<float>(a->x, a->residual, a->out, p, a->shared, st);
  if (a->dtype == PF_FP16) return launch_type<half_t>(a->x, a->residual, a->out, p, a->shared, st);
  return launch_type<bhalf_t>(a->x, a->residual, a->out, p, a->shared, st);
}
