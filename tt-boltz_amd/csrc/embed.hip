// Table lookup with a scale, and its transpose: the table's gradient, summed by sorted tokens
// (nn.Embedding; the token <-> atom broadcasts and the one-hot projections of tt_bio/boltz2.py) for
// gfx950.
//
//   forward    out[i, :] = scale * w[t_i, :]           (t_i outside [0, V): zeros)
//   gradient   dw[v, :]  = scale * sum_{i : t_i = v} g[i, :]
//
// The gradient reads every row of g once and writes every row of dw once, in fp32 sums whose order
// depends on the tokens alone (no float atomics: the same call gives the same bits).  Tokens are
// radix-sorted with their positions (stable, integer ranks), then
//   * embed_grad_kernel, part 1: a table row that at most CH of the sorted tokens name is summed and
//     written by one group of lanes (zeros where no token names it);
//   * part 2: the sorted list is cut into chunks of CH; where a row's run is longer than CH, each
//     chunk's part of it is summed into a workspace row (a chunk meets at most two such runs: one
//     that holds its first token and one that holds its last);
//   * embed_join_kernel adds a long run's parts, in the chunks' order.
#include "pf_elem.h"

namespace {

// ------------------------------------------------------------------------------ forward
// A group of TPR lanes (a power of two) copies U rows; N elements (16 bytes, or 1) a load.
template <typename T, int N, typename I>
__global__ __launch_bounds__(256) void embed_kernel(const I* __restrict__ t, const T* __restrict__ w, long ldw,
                                                    T* __restrict__ out, long n, long V, long C, float scale, int tpr_log2) {
  constexpr int U = 4;
  const int tpr = 1 << tpr_log2, groups = 256 >> tpr_log2;
  const int lane = threadIdx.x & (tpr - 1), group = threadIdx.x >> tpr_log2;
  const long i0 = (long)blockIdx.x * (groups * U) + group;
  long row[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long i = i0 + (long)u * groups;
    row[u] = i < n ? (long)t[i] : -1;
  }
  for (long c = (long)lane * N; c < C; c += (long)tpr * N) {
    float v[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int k = 0; k < N; ++k) v[u][k] = 0.f;
      if (row[u] >= 0 && row[u] < V) load_elems<T, N>(w + row[u] * ldw + c, v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long i = i0 + (long)u * groups;
      if (i >= n) continue;
#pragma unroll
      for (int k = 0; k < N; ++k) v[u][k] *= scale;
      store_elems<T, N>(out + i * C + c, v[u]);
    }
  }
}

// ------------------------------------------------------------------------------ sorting
// One pass of a stable least-significant-digit radix sort: at most SORT_BLOCKS workgroups, each with
// a contiguous part of the list.  A pass is two launches (counts per workgroup and digit, then the
// moves): every workgroup of the second adds up the others' counts itself, which at <= 512 digits
// x 256 workgroups (512 KB from L2) costs less than a third launch.
constexpr int SORT_BLOCKS = 256, SORT_TILE = 1024, SORT_BITS = 9;

struct SortPart {
  long n, per;    // tokens, and tokens per workgroup (a multiple of SORT_TILE)
  long V;
  int shift, bits;
};

// Key of token i: the token, or V (behind all others) where it lies outside the table.
template <typename I, bool FIRST>
PF_DEV uint32_t sort_key(const void* src, long i, long V) {
  if constexpr (FIRST) {
    const long t = (long)((const I*)src)[i];
    return (uint32_t)(t >= 0 && t < V ? t : V);
  } else {
    return ((const uint32_t*)src)[i];
  }
}

template <typename I, bool FIRST>
__global__ __launch_bounds__(256) void sort_count_kernel(const void* __restrict__ keys, uint32_t* __restrict__ counts,
                                                         SortPart p) {
  __shared__ uint32_t hist[1 << SORT_BITS];
  const int bins = 1 << p.bits;
  for (int d = threadIdx.x; d < bins; d += 256) hist[d] = 0;
  __syncthreads();
  const long i1 = min(p.n, ((long)blockIdx.x + 1) * p.per);
  for (long i = (long)blockIdx.x * p.per + threadIdx.x; i < i1; i += 256)
    atomicAdd(&hist[(sort_key<I, FIRST>(keys, i, p.V) >> p.shift) & (bins - 1)], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += 256) counts[(long)blockIdx.x * bins + d] = hist[d];
}

template <typename I, bool FIRST>
__global__ __launch_bounds__(256) void sort_move_kernel(const void* __restrict__ keys, const uint32_t* __restrict__ pos,
                                                        const uint32_t* __restrict__ counts, uint32_t* __restrict__ keys_out,
                                                        uint32_t* __restrict__ pos_out, SortPart p) {
  constexpr int BINS = 1 << SORT_BITS, ITEMS = SORT_TILE / 256;
  __shared__ uint32_t base[BINS];        // where the next token of a digit goes
  __shared__ uint32_t wave_n[4][BINS];   // tokens of a digit per wave of this tile, then their first place
  __shared__ uint32_t scan[256];
  const int bins = 1 << p.bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // totals per digit, and this workgroup's share before it
  uint32_t before[2] = {0, 0}, total[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int d = 2 * threadIdx.x + k;
    if (d < bins) {
#pragma unroll 8
      for (int b = 0; b < (int)gridDim.x; ++b) {
        const uint32_t c = counts[(long)b * bins + d];
        total[k] += c;
        before[k] += b < (int)blockIdx.x ? c : 0;
      }
    }
  }
  scan[threadIdx.x] = total[0] + total[1];
  __syncthreads();
  for (int o = 1; o < 256; o <<= 1) {
    const uint32_t v = threadIdx.x >= (unsigned)o ? scan[threadIdx.x - o] : 0;
    __syncthreads();
    scan[threadIdx.x] += v;
    __syncthreads();
  }
  const uint32_t first = scan[threadIdx.x] - total[0] - total[1];
  if (2 * (int)threadIdx.x < bins) base[2 * threadIdx.x] = first + before[0];
  if (2 * (int)threadIdx.x + 1 < bins) base[2 * threadIdx.x + 1] = first + total[0] + before[1];
  const long begin = (long)blockIdx.x * p.per, end = min(p.n, begin + p.per);
  for (long t0 = begin; t0 < end; t0 += SORT_TILE) {
    for (int d = threadIdx.x; d < 4 * BINS; d += 256) (&wave_n[0][0])[d] = 0;
    __syncthreads();
    // wave w ranks tokens t0 + 256 w .. + 255 in order, 64 at a time
    uint32_t key[ITEMS], at[ITEMS], rank[ITEMS];
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
      const long i = t0 + 256 * wave + 64 * u + lane;
      key[u] = i < end ? sort_key<I, FIRST>(keys, i, p.V) : 0;
      at[u] = i < end ? (FIRST ? (uint32_t)i : pos[i]) : 0;
    }
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
      const bool in = t0 + 256 * wave + 64 * u + lane < end;
      const uint32_t d = (key[u] >> p.shift) & (bins - 1);
      uint64_t same = __ballot(in);   // the lanes with this digit
      for (int b = 0; b < p.bits; ++b) {
        const uint64_t ones = __ballot((d >> b) & 1);
        same &= (d >> b) & 1 ? ones : ~ones;
      }
      const int lower = __popcll(same & ((1ull << lane) - 1));
      uint32_t seen = 0;
      if (in) seen = wave_n[wave][d];
      // the wave's LDS accesses run in order; the fences keep the compiler to it: every lane has read
      // before the first one adds, and the next 64 tokens read what was added
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (in && lower == 0) wave_n[wave][d] = seen + (uint32_t)__popcll(same);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      rank[u] = seen + lower;
    }
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += 256) {
      uint32_t s = base[d];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t c = wave_n[w][d];
        wave_n[w][d] = s;
        s += c;
      }
      base[d] = s;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
      if (t0 + 256 * wave + 64 * u + lane < end) {
        const uint32_t to = wave_n[wave][(key[u] >> p.shift) & (bins - 1)] + rank[u];
        keys_out[to] = key[u];
        pos_out[to] = at[u];
      }
    }
    __syncthreads();
  }
}

// First index of the sorted keys that is not below v.
PF_DEV long lower_bound(const uint32_t* __restrict__ keys, long n, uint32_t v) {
  long lo = 0, len = n;
  while (len > 0) {
    const long half = len >> 1;
    const bool below = keys[lo + half] < v;
    lo = below ? lo + half + 1 : lo;
    len = below ? len - half - 1 : half;
  }
  return lo;
}

// ------------------------------------------------------------------------------ sums
constexpr int GRAD_ROWS = 128;   // most table rows of a workgroup of part 1

struct GradPart {
  long n, V, C;
  long chunks;           // of CH sorted tokens
  int ch;                // CH
  int rows;              // table rows per workgroup of part 1
  long row_blocks;
  float scale;
  int tpr_log2;          // lanes per row, a power of two <= 256
};

// a += rows g[pos[i]], i = s, s + by, .. < e, at channels c .. c + N in fp32, U of them in flight.
template <typename T, int N>
PF_DEV void sum_rows(const T* __restrict__ g, const uint32_t* __restrict__ pos, long C, long s, long e, int by, long c,
                     float (&a)[N]) {
  constexpr int U = 8;
  for (long i0 = s; i0 < e; i0 += (long)by * U) {
    float v[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long i = i0 + (long)u * by;
#pragma unroll
      for (int k = 0; k < N; ++k) v[u][k] = 0.f;
      if (i < e) load_elems<T, N>(g + (long)pos[i] * C + c, v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < N; ++k) a[k] += v[u][k];
  }
}

template <typename T, int N>
__global__ __launch_bounds__(256) void embed_grad_kernel(const T* __restrict__ g, const uint32_t* __restrict__ keys,
                                                         const uint32_t* __restrict__ pos, T* __restrict__ dw,
                                                         float* __restrict__ parts, int* __restrict__ long_end, GradPart p) {
  __shared__ float part[N * 256];
  __shared__ long bound[GRAD_ROWS + 1];
  const int lane = threadIdx.x & ((1 << p.tpr_log2) - 1), group = threadIdx.x >> p.tpr_log2, groups = 256 >> p.tpr_log2;
  const long step = (long)N << p.tpr_log2;
  if ((long)blockIdx.x >= p.chunks) {   // part 1: table rows v0 .. v0 + rows
    const long v0 = ((long)blockIdx.x - p.chunks) * p.rows;
    const int rows = (int)min((long)p.rows, p.V - v0);
    if ((int)threadIdx.x <= rows) bound[threadIdx.x] = lower_bound(keys, p.n, (uint32_t)(v0 + threadIdx.x));
    __syncthreads();
    for (int r = group; r < rows; r += groups) {
      const long s = bound[r], e = bound[r + 1];
      if (e - s > p.ch) continue;
      for (long c = (long)lane * N; c < p.C; c += step) {
        float a[N];
#pragma unroll
        for (int i = 0; i < N; ++i) a[i] = 0.f;
        sum_rows<T, N>(g, pos, p.C, s, e, 1, c, a);
#pragma unroll
        for (int i = 0; i < N; ++i) a[i] *= p.scale;
        store_elems<T, N>(dw + (v0 + r) * p.C + c, a);
      }
    }
    return;
  }
  // part 2: what long runs have in this chunk
  const long i0 = (long)blockIdx.x * p.ch, i1 = min(p.n, i0 + p.ch);
  if (threadIdx.x < 4) {   // the runs of the first and of the last token
    const uint32_t v = keys[threadIdx.x < 2 ? i0 : i1 - 1];
    bound[threadIdx.x] = lower_bound(keys, p.n, v + (threadIdx.x & 1));
  }
  __syncthreads();
  const long s0 = bound[0], e0 = bound[1], s1 = bound[2], e1 = bound[3];
  const bool first = e0 - s0 > p.ch && keys[i0] < (uint32_t)p.V;
  const bool last = s1 > i0 && e1 - s1 > p.ch && keys[i1 - 1] < (uint32_t)p.V;
  // a long run that begins in this chunk: the join's work
  if (threadIdx.x == 0) long_end[blockIdx.x] = last ? (int)e1 : first && s0 == i0 ? (int)e0 : 0;
  for (int w = 0; w < 2; ++w) {
    if (!(w ? last : first)) continue;
    const long s = w ? s1 : i0, e = w ? i1 : min(i1, e0);
    // the groups take the rows in turn, and their sums are joined in the groups' order
    for (long c0 = 0; c0 < p.C; c0 += step) {
      const long c = c0 + (long)lane * N;
      float a[N];
#pragma unroll
      for (int i = 0; i < N; ++i) a[i] = 0.f;
      if (c < p.C) sum_rows<T, N>(g, pos, p.C, s + group, e, groups, c, a);
      if (groups > 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) part[i * 256 + threadIdx.x] = a[i];
        for (int o = groups >> 1; o >= 1; o >>= 1) {
          __syncthreads();
          if (group < o) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
              a[i] += part[i * 256 + threadIdx.x + (o << p.tpr_log2)];
              part[i * 256 + threadIdx.x] = a[i];
            }
          }
        }
        __syncthreads();
      }
      if (group == 0 && c < p.C) {
#pragma unroll
        for (int i = 0; i < N; ++i) parts[(2l * blockIdx.x + w) * p.C + c + i] = a[i];
      }
    }
  }
}

// The parts of the long run that begins in chunk blockIdx.x, if one does: its first part, then the
// first-token parts of the chunks up to its end.  One channel a lane.
template <typename T>
__global__ __launch_bounds__(256) void embed_join_kernel(const float* __restrict__ parts, const uint32_t* __restrict__ keys,
                                                         const int* __restrict__ long_end, T* __restrict__ dw, GradPart p) {
  __shared__ float part[256];
  const long c0 = blockIdx.x, e = long_end[c0];
  if (e == 0) return;
  const uint32_t v = keys[e - 1];
  const long c1 = (e - 1) / p.ch;
  const bool whole = keys[c0 * p.ch] == v;   // the run holds the chunk's first token too
  const int lane = threadIdx.x & ((1 << p.tpr_log2) - 1), group = threadIdx.x >> p.tpr_log2, groups = 256 >> p.tpr_log2;
  for (long c = (long)blockIdx.y << p.tpr_log2; c < p.C; c += (long)gridDim.y << p.tpr_log2) {
    const bool in = c + lane < p.C;
    float a = 0.f;
    if (in) {
#pragma unroll 8
      for (long k = c0 + group; k <= c1; k += groups) a += parts[(2 * k + (k == c0 && !whole)) * p.C + c + lane];
    }
    if (groups > 1) {
      part[threadIdx.x] = a;
      for (int o = groups >> 1; o >= 1; o >>= 1) {
        __syncthreads();
        if (group < o) part[threadIdx.x] = a = a + part[threadIdx.x + (o << p.tpr_log2)];
      }
      __syncthreads();
    }
    if (group == 0 && in) dw[(long)v * p.C + c + lane] = (T)(a * p.scale);
  }
}

// ------------------------------------------------------------------------------ host side
int log2_at_least(long n) {
  int b = 0;
  while ((1l << b) < n) ++b;
  return b;
}

struct GradLayout {
  int passes, bits, ch;
  long per, blocks, chunks;
  size_t keys, pos, counts, ends, parts, bytes;
};

GradLayout grad_layout(long n, long V, long C) {
  GradLayout l;
  const int all = log2_at_least(V + 1) > 0 ? log2_at_least(V + 1) : 1;
  l.passes = (all + SORT_BITS - 1) / SORT_BITS;
  l.bits = (all + l.passes - 1) / l.passes;
  const long tiles = n > 0 ? (n + SORT_TILE - 1) / SORT_TILE : 1;
  l.per = (tiles + SORT_BLOCKS - 1) / SORT_BLOCKS * SORT_TILE;
  l.blocks = (n + l.per - 1) / l.per;
  l.ch = n <= (1l << 17) ? 64 : 256;
  l.chunks = (n + l.ch - 1) / l.ch;
  auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
  const size_t list = up((size_t)n * 4);
  l.keys = 0;
  l.pos = 2 * list;
  l.counts = 4 * list;
  l.ends = l.counts + up(((size_t)l.blocks << l.bits) * 4);
  l.parts = l.ends + up((size_t)l.chunks * 4);
  l.bytes = l.parts + up((size_t)l.chunks * 2 * C * 4);
  return l;
}

int embed_check(const char* fn, const void* index, int index64, int dtype, long n, long V, long C) {
  if (dtype < PF_FP32 || dtype > PF_BF16) return pf_fail(PF_E_INVALID, "%s: unknown dtype %d", fn, dtype);
  if (index64 != 0 && index64 != 1) return pf_fail(PF_E_INVALID, "%s: index64 must be 0 or 1 (got %d)", fn, index64);
  if (n < 0 || V < 0 || C < 0 || n > 0x7fffff00l || V > 0x7ffffff0l || C > (1l << 24))
    return pf_fail(PF_E_INVALID, "%s: bad shape (n=%ld V=%ld C=%ld; n, V < 2^31, C <= 2^24)", fn, n, V, C);
  if (n > 0 && C > 0 && !index) return pf_fail(PF_E_INVALID, "%s: null pointer", fn);
  return PF_OK;
}

template <typename T, int N>
int embed_launch(const void* t, int index64, const T* w, long ldw, T* out, long n, long V, long C, float scale,
                 hipStream_t st) {
  const int units = (int)((C + N - 1) / N), tpr_log2 = units >= 256 ? 8 : log2_at_least(units);
  const long per = 4l * (256 >> tpr_log2);
  const long grid_l = (n + per - 1) / per;
  if (grid_l >> 24)   // a launch holds fewer than 2^32 threads
    return pf_fail(PF_E_INVALID, "pf_embedding_fwd: too many rows (n=%ld C=%ld)", n, C);
  const unsigned grid = (unsigned)grid_l;
  if (index64)
    embed_kernel<T, N, long><<<grid, 256, 0, st>>>((const long*)t, w, ldw, out, n, V, C, scale, tpr_log2);
  else
    embed_kernel<T, N, int><<<grid, 256, 0, st>>>((const int*)t, w, ldw, out, n, V, C, scale, tpr_log2);
  PF_CHECK_LAUNCH("embed_kernel");
  return PF_OK;
}

template <typename T>
int embed_type(const void* t, int index64, const void* w, long ldw, void* out, long n, long V, long C, float scale,
               hipStream_t st) {
  constexpr int N = Vec16<T>::N;
  if (C % N == 0 && ldw % N == 0 && pf_aligned16(w) && pf_aligned16(out))
    return embed_launch<T, N>(t, index64, (const T*)w, ldw, (T*)out, n, V, C, scale, st);
  return embed_launch<T, 1>(t, index64, (const T*)w, ldw, (T*)out, n, V, C, scale, st);
}

template <typename I>
int sort_tokens(const void* index, char* ws, const GradLayout& l, long n, long V, hipStream_t st, int* result) {
  uint32_t *keys[2], *pos[2], *counts = (uint32_t*)(ws + l.counts);
  const size_t list = (l.pos - l.keys) / 2;
  for (int k = 0; k < 2; ++k) {
    keys[k] = (uint32_t*)(ws + l.keys + k * list);
    pos[k] = (uint32_t*)(ws + l.pos + k * list);
  }
  for (int pass = 0; pass < l.passes; ++pass) {
    const SortPart p{n, l.per, V, pass * l.bits, l.bits};
    const int to = pass & 1, from = 1 - to;
    if (pass == 0) {
      sort_count_kernel<I, true><<<(unsigned)l.blocks, 256, 0, st>>>(index, counts, p);
      PF_CHECK_LAUNCH("sort_count_kernel");
      sort_move_kernel<I, true><<<(unsigned)l.blocks, 256, 0, st>>>(index, nullptr, counts, keys[to], pos[to], p);
    } else {
      sort_count_kernel<I, false><<<(unsigned)l.blocks, 256, 0, st>>>(keys[from], counts, p);
      PF_CHECK_LAUNCH("sort_count_kernel");
      sort_move_kernel<I, false><<<(unsigned)l.blocks, 256, 0, st>>>(keys[from], pos[from], counts, keys[to], pos[to], p);
    }
    PF_CHECK_LAUNCH("sort_move_kernel");
  }
  *result = (l.passes - 1) & 1;
  return PF_OK;
}

template <typename T, int N>
int grad_sums(const T* g, const uint32_t* keys, const uint32_t* pos, T* dw, char* ws, const GradLayout& l, long n, long V,
              long C, float scale, hipStream_t st) {
  const int units = (int)((C + N - 1) / N), tpr_log2 = units >= 256 ? 8 : log2_at_least(units);
  // a row for each group of lanes at least; more where eight workgroups per CU remain
  const long groups = 256 >> tpr_log2, share = V / 2048 < 64 ? V / 2048 : 64;
  const int rows = (int)(groups > GRAD_ROWS ? GRAD_ROWS : share < groups ? groups : share);
  GradPart p{n, V, C, l.chunks, l.ch, rows, (V + rows - 1) / rows, scale, tpr_log2};
  float* parts = (float*)(ws + l.parts);
  int* ends = (int*)(ws + l.ends);
  if ((p.chunks + p.row_blocks) >> 24) return pf_fail(PF_E_INVALID, "pf_embedding_grad: too many rows (n=%ld V=%ld C=%ld)", n, V, C);
  embed_grad_kernel<T, N><<<(unsigned)(p.chunks + p.row_blocks), 256, 0, st>>>(g, keys, pos, dw, parts, ends, p);
  PF_CHECK_LAUNCH("embed_grad_kernel");
  if (l.chunks == 0 || n <= l.ch) return PF_OK;   // no run can be longer than a chunk
  p.tpr_log2 = C >= 64 ? 6 : log2_at_least(C);
  const long cols = (C + (1l << p.tpr_log2) - 1) >> p.tpr_log2;
  embed_join_kernel<T><<<dim3((unsigned)l.chunks, (unsigned)(cols < 32 ? cols : 32)), 256, 0, st>>>(parts, keys, ends, dw, p);
  PF_CHECK_LAUNCH("embed_join_kernel");
  return PF_OK;
}

template <typename T>
int grad_type(const void* g, const uint32_t* keys, const uint32_t* pos, void* dw, char* ws, const GradLayout& l, long n,
              long V, long C, float scale, hipStream_t st) {
  constexpr int N = Vec16<T>::N;
  if (C % N == 0 && pf_aligned16(g) && pf_aligned16(dw))
    return grad_sums<T, N>((const T*)g, keys, pos, (T*)dw, ws, l, n, V, C, scale, st);
  return grad_sums<T, 1>((const T*)g, keys, pos, (T*)dw, ws, l, n, V, C, scale, st);
}

}  // namespace

extern "C" int pf_embedding_fwd(const void* index, int index64, const void* weight, long ldw, void* out, long n, long V,
                                long C, int dtype, float scale, void* stream) {
  if (int rc = embed_check("pf_embedding_fwd", index, index64, dtype, n, V, C)) return rc;
  if (n == 0 || C == 0) return PF_OK;
  if (!out || (V > 0 && !weight)) return pf_fail(PF_E_INVALID, "pf_embedding_fwd: null pointer");
  if (ldw < C) return pf_fail(PF_E_INVALID, "pf_embedding_fwd: row stride %ld below C = %ld", ldw, C);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == PF_FP32) return embed_type<float>(index, index64, weight, ldw, out, n, V, C, scale, st);
  if (dtype == PF_FP16) return embed_type<half_t>(index, index64, weight, ldw, out, n, V, C, scale, st);
  return embed_type<bhalf_t>(index, index64, weight, ldw, out, n, V, C, scale, st);
}

extern "C" size_t pf_embedding_grad_workspace_size(long n, long V, long C) {
  if (n <= 0 || V <= 0 || C <= 0 || n > 0x7fffff00l || V > 0x7ffffff0l || C > (1l << 24)) return 0;
  return grad_layout(n, V, C).bytes;
}

extern "C" int pf_embedding_grad(const void* index, int index64, const void* grad, void* dw, long n, long V, long C,
                                 int dtype, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = embed_check("pf_embedding_grad", index, index64, dtype, n, V, C)) return rc;
  if (V == 0 || C == 0) return PF_OK;
  if (!dw || (n > 0 && !grad)) return pf_fail(PF_E_INVALID, "pf_embedding_grad: null pointer");
  const GradLayout l = grad_layout(n, V, C);
  if (n > 0 && (!workspace || workspace_bytes < l.bytes))
    return pf_fail(PF_E_INVALID, "pf_embedding_grad: workspace too small (%zu < %zu bytes)", workspace_bytes, l.bytes);
  if (n > 0 && ((uintptr_t)workspace & 15)) return pf_fail(PF_E_INVALID, "pf_embedding_grad: workspace not 16-byte aligned");
  hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)workspace;
  int at = 0;
  if (n > 0) {
    if (int rc = index64 ? sort_tokens<long>(index, ws, l, n, V, st, &at) : sort_tokens<int>(index, ws, l, n, V, st, &at)) return rc;
  }
  const size_t list = (l.pos - l.keys) / 2;
  const uint32_t *keys = (const uint32_t*)(ws + l.keys + at * list), *pos = (const uint32_t*)(ws + l.pos + at * list);
  if (dtype == PF_FP32) return grad_type<float>(grad, keys, pos, dw, ws, l, n, V, C, scale, st);
  if (dtype == PF_FP16) return grad_type<half_t>(grad, keys, pos, dw, ws, l, n, V, C, scale, st);
  return grad_type<bhalf_t>(grad, keys, pos, dw, ws, l, n, V, C, scale, st);
}
