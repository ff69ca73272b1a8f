// Table lookup with a scale, and its transpose: the table's gradient, summed by sorted tokens
// (nn.Embedding; the token <-> atom broadcasts and the one-hot projections of tt_bio/boltz2.py) for
// gfx950.
//
//   forward    out[i, :] = scale * w[t_i, :]           (t_i outside [0, V): zeros)
//   gradient   dw[v, :]  = scale * sum_{i : t_i = v} g[i, :]
//
// The gradient reads every row of g once and writes every row of dw once, in fp32 sums whose order
// depends on the tokens alone (no float atomics: the same call gives the same bits).  Tokens are
// radix-sorted with their positions (stable, integer ranks) and cut into chunks; then
//   * embed_grad_kernel, part 1: a group of lanes streams a chunk's rows and writes a table row where the
//     token changes.  A run of one token that crosses a chunk's border goes to a workspace row instead (at
//     most two a chunk: the run that came in, the run that goes out);
//   * part 2: the rows that no token names get their zeros;
//   * embed_join_kernel adds the parts of each run that crossed, in the chunks' order.
//
// Memory's rate bounds all but the smallest.  Measured (one MI355X): lookup of 16384 rows of 2048 bf16 out of
// 32000 17 to 21 us (134 MB, rows that come again from cache), of 524288 x 64 fp32 out of 33 22.5 (134 MB
// written: 6.0 TB/s).  Gradient of the latter: sums 23 us (134 MB read), join 9.5, sort 16; of 16384 x 2048 bf16
// in 128000 rows: sums and zeros 106 to 114 (591 MB, of which the 524 written alone take a fill 76), join 8,
// sort 27 for its two digits.  Up to 4096 tokens 10 to 40 us, the launches' and the sort's latency.
#include "pf_elem.h"

namespace {

// ------------------------------------------------------------------------------ forward
// (two rows against one and four: within 2 % at 134 MB; 4608 x 128 fp32 2.6 us, with four 3.0)
constexpr int LOOKUP_ROWS = 2;

// A group of lanes (a power of two) copies LOOKUP_ROWS rows; N elements (16 bytes, or 1) a load.
template <typename T, int N, typename I>
__global__ __launch_bounds__(256) void embed_kernel(const I* __restrict__ t, const T* __restrict__ w, long ldw,
                                                    T* __restrict__ out, long n, long V, long C, float scale, int tpr_log2) {
  constexpr int U = LOOKUP_ROWS;
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
// Stable least-significant-digit radix sort of (token, position), digits of at most 9 bits.
//   * up to SORT_SMALL tokens: one workgroup, all passes in LDS, one launch (the whole gradient in the
//     launches below instead: 64 tokens of 30000 25.8 us for 15.8, 4096 tokens 34 for 25);
//   * else each pass is a launch that counts the digits per workgroup (at most 2^17 / digits
//     workgroups, each with a contiguous part of the list), one that turns the counts into first places,
//     and one that moves.
// A wave ranks 64 tokens at a time: the lanes with its digit come from one ballot per bit, and the
// digit's counter of the wave is read by all of them and raised by the first.
constexpr int SORT_TILE = 1024, SORT_BITS = 9, SORT_BINS = 1 << SORT_BITS, SORT_SMALL = 4096;

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

// Rank of this lane's token (`in`: there is one) among those of digit d that the wave has seen since its
// `counts` were cleared, and the counts with these 64 added.
PF_DEV uint32_t wave_rank(uint32_t* counts, uint32_t d, int bits, bool in, int lane) {
  uint64_t same = __ballot(in);   // the lanes with this digit
  for (int b = 0; b < bits; ++b) {
    const uint64_t ones = __ballot((d >> b) & 1);
    same &= (d >> b) & 1 ? ones : ~ones;
  }
  const int lower = __popcll(same & ((1ull << lane) - 1));
  uint32_t seen = 0;
  if (in) seen = counts[d];
  // the wave's LDS accesses run in order; the fences keep the compiler to it: every lane has read
  // before the first one adds, and the next 64 tokens read what was added
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  if (in && lower == 0) counts[d] = seen + (uint32_t)__popcll(same);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  return seen + lower;
}

// Inclusive sum over the lanes up to this one.
PF_DEV uint32_t wave_scan(uint32_t x, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(x, o);
    x += lane >= o ? y : 0;
  }
  return x;
}

constexpr int SMALL_WAVES = 16;
constexpr size_t SMALL_LDS = 4 * SORT_SMALL * 4 + SMALL_WAVES * SORT_BINS * 4 + 64;

template <typename I>
__global__ __launch_bounds__(64 * SMALL_WAVES) void sort_small_kernel(const void* __restrict__ tokens, uint32_t* __restrict__ keys_out,
                                                                      uint32_t* __restrict__ pos_out, SortPart p, int passes) {
  extern __shared__ __align__(16) char smem[];
  uint32_t* const keys = reinterpret_cast<uint32_t*>(smem);      // [2][SORT_SMALL]
  uint32_t* const pos = keys + 2 * SORT_SMALL;                   // [2][SORT_SMALL]
  uint32_t* const counts = pos + 2 * SORT_SMALL;                 // [SMALL_WAVES][SORT_BINS]
  uint32_t* const sums = counts + SMALL_WAVES * SORT_BINS;       // [SMALL_WAVES]
  const int n = (int)p.n, bins = 1 << p.bits, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  constexpr int NT = 64 * SMALL_WAVES, ITEMS = SORT_SMALL / NT;
  for (int i = tid; i < n; i += NT) {
    keys[i] = sort_key<I, true>(tokens, i, p.V);
    pos[i] = i;
  }
  // a wave's share of the list, whole 64s
  const int share = (n + 64 * SMALL_WAVES - 1) / (64 * SMALL_WAVES) * 64;
  for (int pass = 0; pass < passes; ++pass) {
    const uint32_t *ki = keys + (pass & 1) * SORT_SMALL, *pi = pos + (pass & 1) * SORT_SMALL;
    uint32_t *ko = keys + (1 - (pass & 1)) * SORT_SMALL, *po = pos + (1 - (pass & 1)) * SORT_SMALL;
    for (int d = tid; d < SMALL_WAVES * SORT_BINS; d += NT) counts[d] = 0;
    __syncthreads();
    uint32_t key[ITEMS], rank[ITEMS];
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
      const int i = wave * share + 64 * u + lane;
      const bool in = 64 * u < share && i < n;
      key[u] = in ? ki[i] : 0;
      if (64 * u < share) rank[u] = wave_rank(counts + wave * SORT_BINS, (key[u] >> (pass * p.bits)) & (bins - 1), p.bits, in, lane);
    }
    __syncthreads();
    // first places: the digits before, then the waves before
    uint32_t total = 0;
    if (tid < bins) {
      for (int w = 0; w < SMALL_WAVES; ++w) total += counts[w * SORT_BINS + tid];
    }
    const uint32_t upto = wave_scan(total, lane);
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    uint32_t at = upto - total;
    for (int w = 0; w < wave; ++w) at += sums[w];
    if (tid < bins) {
      for (int w = 0; w < SMALL_WAVES; ++w) {
        const uint32_t c = counts[w * SORT_BINS + tid];
        counts[w * SORT_BINS + tid] = at;
        at += c;
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
      const int i = wave * share + 64 * u + lane;
      if (64 * u < share && i < n) {
        const uint32_t to = counts[wave * SORT_BINS + ((key[u] >> (pass * p.bits)) & (bins - 1))] + rank[u];
        ko[to] = key[u];
        po[to] = pi[i];
      }
    }
    __syncthreads();
  }
  for (int i = tid; i < n; i += NT) {
    keys_out[i] = keys[(passes & 1) * SORT_SMALL + i];
    pos_out[i] = pos[(passes & 1) * SORT_SMALL + i];
  }
}

template <typename I, bool FIRST>
__global__ __launch_bounds__(256) void sort_count_kernel(const void* __restrict__ keys, uint32_t* __restrict__ counts,
                                                         SortPart p) {
  __shared__ uint32_t hist[SORT_BINS];
  const int bins = 1 << p.bits;
  for (int d = threadIdx.x; d < bins; d += 256) hist[d] = 0;
  __syncthreads();
  const long i1 = min(p.n, ((long)blockIdx.x + 1) * p.per);
  for (long i = (long)blockIdx.x * p.per + threadIdx.x; i < i1; i += 256)
    atomicAdd(&hist[(sort_key<I, FIRST>(keys, i, p.V) >> p.shift) & (bins - 1)], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += 256) counts[(long)d * gridDim.x + blockIdx.x] = hist[d];
}

// counts [digit][workgroup]: a wave per digit replaces them by the sums of the workgroups before, and
// leaves the digit's total behind them (totals[digit]).  A lane has U consecutive workgroups.
__global__ __launch_bounds__(64) void sort_scan_kernel(uint32_t* __restrict__ counts, uint32_t* __restrict__ totals, int blocks) {
  constexpr int U = 8;
  uint32_t* const c = counts + (long)blockIdx.x * blocks;
  const int lane = threadIdx.x;
  uint32_t before = 0;
  for (int b0 = 0; b0 < blocks; b0 += 64 * U) {
    const int b = b0 + U * lane;
    uint32_t x[U], sum = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = b + u < blocks ? c[b + u] : 0;
#pragma unroll
    for (int u = 0; u < U; ++u) sum += x[u];
    const uint32_t upto = wave_scan(sum, lane);
    uint32_t at = before + upto - sum;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (b + u < blocks) c[b + u] = at;
      at += x[u];
    }
    before += __shfl(upto, 63);
  }
  if (lane == 0) totals[blockIdx.x] = before;
}

template <typename I, bool FIRST>
__global__ __launch_bounds__(256) void sort_move_kernel(const void* __restrict__ keys, const uint32_t* __restrict__ pos,
                                                        const uint32_t* __restrict__ counts, const uint32_t* __restrict__ totals,
                                                        uint32_t* __restrict__ keys_out, uint32_t* __restrict__ pos_out, SortPart p) {
  constexpr int ITEMS = SORT_TILE / 256;
  __shared__ uint32_t base[SORT_BINS];        // where the next token of a digit goes
  __shared__ uint32_t wave_n[4][SORT_BINS];   // tokens of a digit per wave of this tile, then their first place
  __shared__ uint32_t sums[4];
  const int bins = 1 << p.bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t total[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) total[k] = 2 * (int)threadIdx.x + k < bins ? totals[2 * threadIdx.x + k] : 0;
  const uint32_t upto = wave_scan(total[0] + total[1], lane);
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  uint32_t first = upto - total[0] - total[1];
  for (int w = 0; w < wave; ++w) first += sums[w];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int d = 2 * threadIdx.x + k;
    if (d < bins) base[d] = first + counts[(long)d * gridDim.x + blockIdx.x];
    first += total[k];
  }
  const long begin = (long)blockIdx.x * p.per, end = min(p.n, begin + p.per);
  for (long t0 = begin; t0 < end; t0 += SORT_TILE) {
    for (int d = threadIdx.x; d < 4 * SORT_BINS; d += 256) (&wave_n[0][0])[d] = 0;
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
    for (int u = 0; u < ITEMS; ++u)
      rank[u] = wave_rank(wave_n[wave], (key[u] >> p.shift) & (bins - 1), p.bits, t0 + 256 * wave + 64 * u + lane < end, lane);
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
struct GradPart {
  long n, V, C;
  int ch;                // CH, a multiple of 8
  long chunks;           // of CH sorted tokens
  long chunk_blocks;     // workgroups of part 1
  int rows;              // table rows per workgroup of part 2, groups of lanes x a whole number
  long row_blocks;
  float scale;
  int tpr_log2;          // lanes per row, a power of two <= 256
};

constexpr int GRAD_ROWS = 128;   // most table rows of a workgroup of part 2

template <typename T, int N>
__global__ __launch_bounds__(256) void embed_grad_kernel(const T* __restrict__ g, const uint32_t* __restrict__ keys,
                                                         const uint32_t* __restrict__ pos, T* __restrict__ dw,
                                                         float* __restrict__ parts, GradPart p) {
  __shared__ long bound[2 * GRAD_ROWS];
  const int lane = threadIdx.x & ((1 << p.tpr_log2) - 1), group = threadIdx.x >> p.tpr_log2, groups = 256 >> p.tpr_log2;
  const long step = (long)N << p.tpr_log2;
  if ((long)blockIdx.x >= p.chunk_blocks) {
    // part 2: zeros for the rows that no token names.  Neighbouring workgroups take neighbouring rows (a
    // workgroup on consecutive rows of its own leaves the chip writing far-apart pieces at a time).
    const long k = (long)blockIdx.x - p.chunk_blocks;
    auto row_of = [&](int r) __attribute__((always_inline)) {
      return ((long)(r / groups) * p.row_blocks + k) * groups + r % groups;
    };
    if ((int)threadIdx.x < 2 * p.rows) {
      const long v = row_of(threadIdx.x >> 1);
      bound[threadIdx.x] = v < p.V ? lower_bound(keys, p.n, (uint32_t)(v + (threadIdx.x & 1))) : threadIdx.x & 1;
    }
    __syncthreads();
    float zero[N];
#pragma unroll
    for (int i = 0; i < N; ++i) zero[i] = 0.f;
    for (int r = group; r < p.rows; r += groups) {
      if (bound[2 * r] != bound[2 * r + 1]) continue;
      T* const to = dw + row_of(r) * p.C;
      for (long c = (long)lane * N; c < p.C; c += step) store_elems<T, N>(to + c, zero);
    }
    return;
  }
  // part 1: a group of lanes streams the CH tokens of a chunk in their sorted order, U rows in flight, and
  // writes a sum where the token changes (4 rows: 65536 x 2048 of 32000 131 us, with 8 152; 524288 x 64 of 33 47
  // and 50; 2^20 x 128 of 33 128 and 121)
  constexpr int U = 4;
  const long chunk = (long)blockIdx.x * groups + group;
  if (chunk >= p.chunks) return;
  const long i0 = chunk * p.ch, i1 = min(p.n, i0 + p.ch);
  const uint32_t none = (uint32_t)p.V;
  const bool goes_on = i0 > 0 && keys[i0 - 1] == keys[i0];   // its first run began before
  const bool reaches = i1 < p.n && keys[i1] == keys[i1 - 1] && keys[i1] < none;   // its last run goes on behind
  float* const part0 = parts + 2 * chunk * p.C;
  for (long c = (long)lane * N; c < p.C; c += step) {
    uint32_t cur = keys[i0];
    if (cur >= none) return;   // sorted behind all others: nothing here, or later
    bool first = goes_on;
    float a[N];
#pragma unroll
    for (int k = 0; k < N; ++k) a[k] = 0.f;
    auto flush = [&](bool part, float* to) __attribute__((always_inline)) {
      if (part) {
#pragma unroll
        for (int k = 0; k < N; ++k) to[c + k] = a[k];
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k) a[k] *= p.scale;
        store_elems<T, N>(dw + (long)cur * p.C + c, a);
      }
    };
    uint32_t key[U], at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long i = min(i0 + u, i1 - 1);
      key[u] = keys[i], at[u] = pos[i];
    }
    for (long i = i0; i < i1 && key[0] < none; i += U) {
      float v[U][N];
      uint32_t now[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int k = 0; k < N; ++k) v[u][k] = 0.f;
        now[u] = key[u];
        if (i + u < i1 && key[u] < none) load_elems<T, N>(g + (long)at[u] * p.C + c, v[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {   // the next tokens, behind the rows' loads
        const long j = min(i + U + u, i1 - 1);
        key[u] = keys[j], at[u] = pos[j];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (now[u] != cur) {
          if (cur < none) flush(first, part0);
          first = false;
          cur = now[u];
#pragma unroll
          for (int k = 0; k < N; ++k) a[k] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < N; ++k) a[k] += v[u][k];
      }
    }
    if (cur < none) flush(first || reaches, first ? part0 : part0 + p.C);
  }
}

// The runs that begin in a workgroup's JOIN chunks and go on behind their chunk: the run's own part, then
// the following chunks' first parts.  A wave adds a run of up to JOIN_SHORT parts by itself; a longer one
// is split over the waves.  N channels a lane, blockIdx.y counts blocks of 64 N channels.
constexpr int JOIN = 8, JOIN_WAVES = 8, JOIN_SHORT = 32;

template <typename T, int N>
__global__ __launch_bounds__(64 * JOIN_WAVES) void embed_join_kernel(const float* __restrict__ parts, const uint32_t* __restrict__ keys,
                                                                     T* __restrict__ dw, GradPart p) {
  __shared__ float part[JOIN_WAVES][N][64];
  __shared__ long last[JOIN];       // last chunk of the run that begins in a chunk (0: none does)
  __shared__ uint32_t token[JOIN];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long c00 = (long)blockIdx.x * JOIN;
  if (threadIdx.x < JOIN) {
    const long c0 = c00 + threadIdx.x, i0 = c0 * p.ch, i1 = i0 + p.ch;
    long end = 0;
    if (i1 < p.n) {
      const uint32_t v = keys[i1 - 1];
      if (v < (uint32_t)p.V && keys[i1] == v && !(i0 > 0 && keys[i0] == v && keys[i0 - 1] == v)) {
        end = c0 + 1;
        token[threadIdx.x] = v;
      }
    }
    last[threadIdx.x] = end;
  }
  if (!__syncthreads_or(threadIdx.x < JOIN && last[threadIdx.x])) return;
  // how far the runs go: 64 chunk beginnings at a time, 64 times as far apart while all of them match
  for (int j = wave; j < JOIN; j += JOIN_WAVES) {
    long lo = last[j];   // chunk lo begins with the token
    if (lo == 0) continue;
    const uint32_t v = token[j];
    bool grow = true;
    for (long hop = 1; hop >= 1;) {
      const long k = lo + hop * (lane + 1);
      const int match = __popcll(__ballot(k < p.chunks && keys[k < p.chunks ? k * p.ch : 0] == v));
      lo += hop * match;
      grow = grow && match == 64;
      hop = grow ? hop * 64 : hop / 64;
    }
    if (lane == 0) last[j] = lo;
  }
  __syncthreads();
  // lanes of a wave beyond a row's take further parts of the same run
  const int tpr = 1 << p.tpr_log2, sub = lane >> p.tpr_log2, subs = 64 >> p.tpr_log2;
  auto add = [&](long c0, long from, long to, int by, long c, float (&a)[N]) __attribute__((always_inline)) {
    constexpr int U = 8;
    for (long k0 = from; k0 <= to; k0 += (long)by * U) {
      float x[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long k = k0 + (long)u * by;
#pragma unroll
        for (int e = 0; e < N; ++e) x[u][e] = 0.f;
        if (k <= to) load_elems<float, N>(parts + (2 * k + (k == c0)) * p.C + c, x[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < N; ++e) a[e] += x[u][e];
    }
  };
  for (long cb = (long)blockIdx.y * tpr * N; cb < p.C; cb += (long)gridDim.y * tpr * N) {
    const long c = cb + (lane & (tpr - 1)) * N;
    const bool in = c < p.C;
    for (int j = wave; j < JOIN; j += JOIN_WAVES) {
      const long c0 = c00 + j, c1 = last[j];
      if (c1 == 0 || c1 - c0 >= JOIN_SHORT || !in || sub) continue;
      float a[N];
#pragma unroll
      for (int e = 0; e < N; ++e) a[e] = 0.f;
      add(c0, c0, c1, 1, c, a);
      T* const to = dw + (long)token[j] * p.C + c;
#pragma unroll
      for (int e = 0; e < N; ++e) to[e] = (T)(a[e] * p.scale);
    }
    for (int j = 0; j < JOIN; ++j) {
      const long c0 = c00 + j, c1 = last[j];
      if (c1 == 0 || c1 - c0 < JOIN_SHORT) continue;
      float a[N];
#pragma unroll
      for (int e = 0; e < N; ++e) a[e] = 0.f;
      if (in) add(c0, c0 + wave * subs + sub, c1, JOIN_WAVES * subs, c, a);
      for (int o = tpr; o < 64; o <<= 1) {
#pragma unroll
        for (int e = 0; e < N; ++e) a[e] += __shfl_xor(a[e], o);
      }
#pragma unroll
      for (int e = 0; e < N; ++e) part[wave][e][lane] = a[e];
      __syncthreads();
      if (wave == 0 && sub == 0 && in) {
        T* const to = dw + (long)token[j] * p.C + c;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          float s = 0.f;
#pragma unroll
          for (int w = 0; w < JOIN_WAVES; ++w) s += part[w][e][lane];
          to[e] = (T)(s * p.scale);
        }
      }
      __syncthreads();
    }
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
  size_t keys, pos, counts, totals, parts, bytes;
};

GradLayout grad_layout(long n, long V, long C) {
  GradLayout l;
  const int all = log2_at_least(V + 1) > 0 ? log2_at_least(V + 1) : 1;
  l.passes = (all + SORT_BITS - 1) / SORT_BITS;
  l.bits = (all + l.passes - 1) / l.passes;
  const long tiles = n > 0 ? (n + SORT_TILE - 1) / SORT_TILE : 1;
  const long most = (1l << 17) >> l.bits;   // workgroups: their counts stay within 512 KB
  l.per = (tiles + most - 1) / most * SORT_TILE;
  l.blocks = (n + l.per - 1) / l.per;
  // chunks of 16 tokens up to 2^16 lanes (4608 x 128 27.6 us, with 32 29.7; above, 16384 x 2048
  // into 128000 rows takes 158 with 16, 150 with 32), 32 above, and longer ones (fewer crossed borders) so that there are at most 8192 (524288 x 64
  // fp32 of 33 rows: 50 us with 64, 56 with 32 or 16; 65536 x 512 of 1000 46 with 32, 57 with 64)
  const int lanes = C >= 1024 ? 256 : 1 << log2_at_least((C + 3) / 4);
  l.ch = n / 16 * lanes <= (1l << 16) ? 16 : 32;
  while (l.ch < 256 && n / l.ch > 8192) l.ch *= 2;
  l.chunks = (n + l.ch - 1) / l.ch;
  auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
  const size_t list = up((size_t)n * 4);
  l.keys = 0;
  l.pos = 2 * list;
  l.counts = 4 * list;
  l.totals = l.counts + up(((size_t)l.blocks << l.bits) * 4);
  l.parts = l.totals + up((size_t)4 << l.bits);
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
  const long per = (long)LOOKUP_ROWS * (256 >> tpr_log2);
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
  // 8 bytes of 16-bit types: 16384 x 2044 bf16 out of 32000 22 us, one element a lane 31
  if constexpr (N == 8) {
    if (C % 4 == 0 && ldw % 4 == 0 && pf_aligned16(w) && pf_aligned16(out))
      return embed_launch<T, 4>(t, index64, (const T*)w, ldw, (T*)out, n, V, C, scale, st);
  }
  return embed_launch<T, 1>(t, index64, (const T*)w, ldw, (T*)out, n, V, C, scale, st);
}

template <typename I>
int sort_tokens(const void* index, char* ws, const GradLayout& l, long n, long V, hipStream_t st, int* result) {
  uint32_t *keys[2], *pos[2], *counts = (uint32_t*)(ws + l.counts), *totals = (uint32_t*)(ws + l.totals);
  const size_t list = (l.pos - l.keys) / 2;
  for (int k = 0; k < 2; ++k) {
    keys[k] = (uint32_t*)(ws + l.keys + k * list);
    pos[k] = (uint32_t*)(ws + l.pos + k * list);
  }
  if (n <= SORT_SMALL) {
    if (int rc = pf_reserve_lds((const void*)sort_small_kernel<I>, SMALL_LDS, "sort_small_kernel")) return rc;
    sort_small_kernel<I><<<1, 64 * SMALL_WAVES, SMALL_LDS, st>>>(index, keys[0], pos[0], SortPart{n, l.per, V, 0, l.bits}, l.passes);
    PF_CHECK_LAUNCH("sort_small_kernel");
    *result = 0;
    return PF_OK;
  }
  for (int pass = 0; pass < l.passes; ++pass) {
    const SortPart p{n, l.per, V, pass * l.bits, l.bits};
    const int to = pass & 1, from = 1 - to;
    const unsigned grid = (unsigned)l.blocks;
    if (pass == 0) sort_count_kernel<I, true><<<grid, 256, 0, st>>>(index, counts, p);
    else sort_count_kernel<I, false><<<grid, 256, 0, st>>>(keys[from], counts, p);
    PF_CHECK_LAUNCH("sort_count_kernel");
    sort_scan_kernel<<<1u << l.bits, 64, 0, st>>>(counts, totals, (int)l.blocks);
    PF_CHECK_LAUNCH("sort_scan_kernel");
    if (pass == 0) sort_move_kernel<I, true><<<grid, 256, 0, st>>>(index, nullptr, counts, totals, keys[to], pos[to], p);
    else sort_move_kernel<I, false><<<grid, 256, 0, st>>>(keys[from], pos[from], counts, totals, keys[to], pos[to], p);
    PF_CHECK_LAUNCH("sort_move_kernel");
  }
  *result = (l.passes - 1) & 1;
  return PF_OK;
}

template <typename T, int N>
int grad_sums(const T* g, const uint32_t* keys, const uint32_t* pos, T* dw, char* ws, const GradLayout& l, long n, long V,
              long C, float scale, hipStream_t st) {
  const int units = (int)((C + N - 1) / N), tpr_log2 = units >= 256 ? 8 : units <= 2 ? 1 : log2_at_least(units);
  const long groups = 256 >> tpr_log2;
  // part 2: a row for each group of lanes at least; up to 64 where four workgroups per CU remain
  long rows = V / 1024 < 64 ? V / 1024 / groups * groups : 64 / groups * groups;
  if (rows < groups) rows = groups;
  GradPart p{n, V, C, l.ch, l.chunks, (l.chunks + groups - 1) / groups, (int)rows, (V + rows - 1) / rows, scale, tpr_log2};
  float* parts = (float*)(ws + l.parts);
  if ((p.chunk_blocks + p.row_blocks) >> 24)
    return pf_fail(PF_E_INVALID, "pf_embedding_grad: too many rows (n=%ld V=%ld C=%ld)", n, V, C);
  embed_grad_kernel<T, N><<<(unsigned)(p.chunk_blocks + p.row_blocks), 256, 0, st>>>(g, keys, pos, dw, parts, p);
  PF_CHECK_LAUNCH("embed_grad_kernel");
  if (l.chunks <= 1) return PF_OK;   // no run crosses a border
  constexpr int J = N > 1 ? 4 : 1;
  p.tpr_log2 = C >= 64 * J ? 6 : log2_at_least((C + J - 1) / J);
  const long cols = (C + 64 * J - 1) / (64 * J), blocks = (l.chunks + JOIN - 1) / JOIN;
  embed_join_kernel<T, J><<<dim3((unsigned)blocks, (unsigned)(cols < 64 ? cols : 64)), 64 * JOIN_WAVES, 0, st>>>(parts, keys, dw, p);
  PF_CHECK_LAUNCH("embed_join_kernel");
  return PF_OK;
}

template <typename T>
int grad_type(const void* g, const uint32_t* keys, const uint32_t* pos, void* dw, char* ws, const GradLayout& l, long n,
              long V, long C, float scale, hipStream_t st) {
  constexpr int N = Vec16<T>::N;
  if (C % N == 0 && pf_aligned16(g) && pf_aligned16(dw))
    return grad_sums<T, N>((const T*)g, keys, pos, (T*)dw, ws, l, n, V, C, scale, st);
  if constexpr (N == 8) {   // (the same sizes: 71 us and 166)
    if (C % 4 == 0 && pf_aligned16(g) && pf_aligned16(dw))
      return grad_sums<T, 4>((const T*)g, keys, pos, (T*)dw, ws, l, n, V, C, scale, st);
  }
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
