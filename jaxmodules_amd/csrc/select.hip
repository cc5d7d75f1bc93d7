// Selection of key blocks for each query (mattn_block_means, mattn_select_blocks).
//
//   m_j = mean of the keys of block j (float64 sum, rounded once to float32)
//   s_qj = (sum over the group's query heads of q) . m_j, in float64
//   blocks of q: the `first` first and `last` newest visible ones, and the best by s of
//   the others, ties to the lower index; ascending, -1 behind
//
// A selection is whole numbers, and neighbours in the order of s lie closer than float32
// sums hold apart, so the scores are float64 products and sums (the order of additions then
// does not show).  Summing the group's queries first makes one cost 2 D flop whatever the
// group's size.  (Products of two bfloat16 pieces each on the faster matrix cores, with the
// rows they leave open scored again, took as long: 40 us against 36 at [1, 8192, 32/8, 128],
// and another 10 for those rows.)
//
// Scores go to a workspace, rows at a time, rounded to float32, which keeps their order but
// for ties; those at the cut are scored again in float64.  Choice: some lanes hold a row's
// scores in registers and halve the range of values, counting how many are at or above a
// trial: some 8 steps (a search over the bits of float64 keys took 25).  More than 2048
// blocks: float64 scores in memory and that search.
#include "elem.hpp"

namespace mattn {
namespace {

__device__ __forceinline__ int held_of(const int32_t* lengths, int b, int most) {
  return lengths ? min(max(lengths[b], 0), most) : most;
}

// ---- means ----------------------------------------------------------------------------

// A workgroup forms 32 chunks of V columns of one block: 8 threads a chunk, each every
// eighth key (32 chunks are 512 bytes of a row).  Bound by HBM: each key is read once.
template <class Tag, int V>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256)))
void block_means(mattn_means p, int nblk, uint32_t groups) {
  __shared__ double red[8][32 * V];
  const int cc = threadIdx.x & 31, kr = threadIdx.x >> 5;
  const int b = blockIdx.y, held = held_of(p.lengths, b, p.L);
  int j = (int)(blockIdx.x / groups);
  const int64_t c0 = 32 * (int64_t)(blockIdx.x % groups);  // first chunk
  if (p.new_keys > 0) {  // only the blocks that hold one of the newest keys
    j += max(held - p.new_keys, 0) / p.block_size;
    if ((int64_t)j * p.block_size >= held) return;
  }
  const int cpr = p.D / V;  // chunks of a head's row
  const int64_t c = c0 + cc;
  const int h = (int)(c / cpr), col = V * (int)(c % cpr);
  const int64_t k0 = (int64_t)j * p.block_size;
  const int n = (int)min((int64_t)p.block_size, max((int64_t)held - k0, (int64_t)0));
  double s[V];
#pragma unroll
  for (int e = 0; e < V; ++e) s[e] = 0.0;
  if (h < p.H) {
    const int64_t at = b * p.k_stride[0] + h * p.k_stride[2] + col;
    for (int i = kr; i < n; i += 8) {
      float x[V];
      load_v<Tag, V>(p.k, at + (k0 + i) * p.k_stride[1], x);
#pragma unroll
      for (int e = 0; e < V; ++e) s[e] += (double)x[e];
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) red[kr][cc + 32 * e] = s[e];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * V; i += 256) {
    const int64_t ci = c0 + i / V;
    const int hi = (int)(ci / cpr), e = i % V;
    if (hi >= p.H) continue;
    double t = 0.0;
#pragma unroll
    for (int r = 0; r < 8; ++r) t += red[r][i / V + 32 * e];
    p.means[(((int64_t)b * nblk + j) * p.H + hi) * p.D + V * (ci % cpr) + e] = n > 0 ? (float)(t / n) : 0.f;
  }
}

// ---- scores ---------------------------------------------------------------------------

struct SelArgs {
  mattn_select p;
  void* s;          // scores of rows [row0, row0 + rows) of each (b, hk): [B * Hkv][rows][nblk] floats (wide: doubles)
  int wide;
  int row0, rows;   // queries of this launch
};
constexpr int kWide = 2048;  // more blocks than this: float64 scores
__device__ __forceinline__ void put_score(const SelArgs& a, int64_t at, double x) {
  if (a.wide) ((double*)a.s)[at] = x;
  else ((float*)a.s)[at] = (float)x;
}

__device__ __forceinline__ int64_t position(const mattn_select& p, int b, int q) {
  return (int64_t)(p.starts ? p.starts[b] : 0) + q;
}
// Blocks that query q of sequence b sees.
__device__ __forceinline__ int visible(const mattn_select& p, int b, int q) {
  const int nb = p.lengths ? min((int)(((int64_t)max(p.lengths[b], 0) + p.block_size - 1) / p.block_size), p.nblk) : p.nblk;
  if (!p.causal) return nb;
  const int64_t pos = position(p, b, q);
  return pos < 0 ? 0 : (int)min((int64_t)nb, pos / p.block_size + 1);
}

// Sum over the group's heads of V columns of query q.
template <class Tag, int V>
__device__ __forceinline__ void sum_group(const mattn_select& p, int b, int hk, int q, int col, double (&o)[V]) {
  const int G = p.Hq / p.Hkv;
#pragma unroll
  for (int e = 0; e < V; ++e) o[e] = 0.0;
  for (int g = 0; g < G; ++g) {
    float x[V];
    load_v<Tag, V>(p.q, b * p.q_stride[0] + q * p.q_stride[1] + (int64_t)(hk * G + g) * p.q_stride[2] + col, x);
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] += (double)x[e];
  }
}

// Many rows: float64 matrix cores.  v_mfma_f64_16x16x4: lane l holds A row l % 16 and B
// column l % 16 at k = l / 16, and of the result column l % 16, rows 4 i + l / 16.  A is
// the queries, B the means; product e of step j takes the columns 32 j + 8 (l / 16) + e
// of both, so that each lane reads 8 consecutive ones.  A wave sums 16 queries over their
// heads once and walks 16 blocks at a time, the next ones' means on their way; 64 queries
// by `span` blocks a workgroup.  Bound by the products, 64 cycles each, 32 a step at D = 128.
typedef double f64x4 __attribute__((ext_vector_type(4)));
template <class Tag, int NJ>  // NJ: ceil(D / 32)
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256)))
void scores_mfma(SelArgs a, int span) {
  const mattn_select& p = a.p;
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int b = blockIdx.z / p.Hkv, hk = blockIdx.z % p.Hkv;
  const int q0 = a.row0 + (gridDim.x - 1 - blockIdx.x) * 64 + 16 * (threadIdx.x >> 6);  // late queries see most: first
  const int qend = a.row0 + a.rows;
  if (q0 >= qend) return;
  const int most = visible(p, b, min(q0 + 15, qend - 1));  // of the wave's last query: the most
  const int j0 = blockIdx.y * span, j1 = min(j0 + span, most);
  if (j0 >= j1) return;
  // columns 32 t + 8 g .. + 7 of a row, zeros past D
  const auto load = [&](auto tag, const void* base, int64_t at, float(&x)[NJ][8]) {
#pragma unroll
    for (int t = 0; t < NJ; ++t) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[t][e] = 0.f;
      if (32 * t + 8 * g < p.D) load_v<decltype(tag), 8>(base, at + 32 * t + 8 * g, x[t]);
    }
  };
  float x[NJ][8], y[NJ][8];  // this step's means and the next one's
  const int64_t m = b * p.m_stride[0] + hk * p.m_stride[2];
  const auto fetch = [&](int j) { load(float{}, p.means, m + min(j + l16, p.nblk - 1) * p.m_stride[1], y); };
  double qf[NJ][8];
#pragma unroll
  for (int t = 0; t < NJ; ++t)
#pragma unroll
    for (int e = 0; e < 8; ++e) qf[t][e] = 0.0;
  const int G = p.Hq / p.Hkv;
  const int64_t at = b * p.q_stride[0] + (int64_t)min(q0 + l16, qend - 1) * p.q_stride[1];
  load(Tag{}, p.q, at + (int64_t)hk * G * p.q_stride[2], x);
  fetch(j0);
  for (int h = 0; h < G; ++h) {  // the next head's columns on their way
    float z[NJ][8];
#pragma unroll
    for (int t = 0; t < NJ; ++t)
#pragma unroll
      for (int e = 0; e < 8; ++e) z[t][e] = x[t][e];
    if (h + 1 < G) load(Tag{}, p.q, at + (int64_t)(hk * G + h + 1) * p.q_stride[2], x);
#pragma unroll
    for (int t = 0; t < NJ; ++t)
#pragma unroll
      for (int e = 0; e < 8; ++e) qf[t][e] += (double)z[t][e];
  }
  const int64_t out = ((int64_t)blockIdx.z * a.rows + (q0 - a.row0)) * p.nblk;
  for (int j = j0; j < j1; j += 16) {
#pragma unroll
    for (int t = 0; t < NJ; ++t)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[t][e] = y[t][e];
    if (j + 16 < j1) fetch(j + 16);
    f64x4 c = {0.0, 0.0, 0.0, 0.0}, d = c;  // two chains
#pragma unroll
    for (int t = 0; t < NJ; ++t)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        c = __builtin_amdgcn_mfma_f64_16x16x4f64(qf[t][e], (double)x[t][e], c, 0, 0, 0);
        d = __builtin_amdgcn_mfma_f64_16x16x4f64(qf[t][e + 1], (double)x[t][e + 1], d, 0, 0, 0);
      }
    c += d;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (q0 + 4 * i + g < qend && j + l16 < j1) put_score(a, out + (int64_t)(4 * i + g) * p.nblk + j + l16, c[i]);
  }
}

// Few rows: bound by reading the means once.  16 lanes take a block's mean, 8 columns
// each, for all rows; the summed queries lie in LDS.
constexpr int kFewRows = 8;
constexpr int kMaxD = 128;
template <class Tag>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256)))
void scores_few(SelArgs a, int per_group) {
  __shared__ double qs[kFewRows * kMaxD];
  const mattn_select& p = a.p;
  const int b = blockIdx.y / p.Hkv, hk = blockIdx.y % p.Hkv, l16 = threadIdx.x & 15;
  const int rows = a.rows, most = visible(p, b, a.row0 + rows - 1);
  const int j0 = blockIdx.x * 16 * per_group;
  if (j0 >= most) return;
  for (int i = threadIdx.x; i < rows * (p.D / 4); i += 256) {
    double x[4];
    sum_group<Tag, 4>(p, b, hk, a.row0 + i / (p.D / 4), 4 * (i % (p.D / 4)), x);
#pragma unroll
    for (int e = 0; e < 4; ++e) qs[4 * i + e] = x[e];
  }
  __syncthreads();
  const float* m = p.means + b * p.m_stride[0] + hk * p.m_stride[2];
  constexpr int NB = 4;  // blocks of a group in flight
  for (int t = 0; t < per_group; t += NB) {
    f32x4 x[NB][2];
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      const int j = j0 + 16 * (t + u) + (threadIdx.x >> 4);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int col = 64 * c + 4 * l16;
        x[u][c] = t + u < per_group && j < most && col < p.D ? *(const f32x4*)(m + j * p.m_stride[1] + col) : f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      const int j = j0 + 16 * (t + u) + (threadIdx.x >> 4);
      if (t + u >= per_group || j >= most) break;
      for (int r = 0; r < rows; ++r) {
        double s = 0.0;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int col = 64 * c + 4 * l16;
          if (col < p.D) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s += qs[r * p.D + col + e] * (double)x[u][c][e];
          }
        }
#pragma unroll
        for (int o = 8; o; o >>= 1) s += __shfl_xor(s, o);
        if (l16 == 0) put_score(a, ((int64_t)blockIdx.y * a.rows + r) * p.nblk + j, s);
      }
    }
  }
}

// ---- choice ---------------------------------------------------------------------------

// Unsigned keys in the order of the scores; NaN as -inf, -0 as 0.
__device__ __forceinline__ uint64_t order_key(double x) {
  x = x != x ? -__builtin_inf() : x + 0.0;
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  return (u >> 63) ? ~u : u | 0x8000000000000000ull;
}

// op over the LPR lanes of a row (16: rotations of a row of lanes; 64: the rows, then swaps)
template <int LPR, class F>
__device__ __forceinline__ float row_reduce(float x, F&& op) {
  const auto ror = [](float v, auto n) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + decltype(n)::value, 0xf, 0xf, false));
  };
  x = op(x, ror(x, std::integral_constant<int, 8>{}));
  x = op(x, ror(x, std::integral_constant<int, 4>{}));
  x = op(x, ror(x, std::integral_constant<int, 2>{}));
  x = op(x, ror(x, std::integral_constant<int, 1>{}));
  if constexpr (LPR == 64) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t a0 = a[0], a1 = a[1];
    x = op(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1));
    const uint32_t w = __builtin_bit_cast(uint32_t, x);
    const auto c = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    const uint32_t c0 = c[0], c1 = c[1];
    x = op(__builtin_bit_cast(float, c0), __builtin_bit_cast(float, c1));
  }
  return x;
}

// Candidates of a row: blocks [c0, c1), `need` of them behind the f first ones at `out`.
struct Row {
  int b, hk, q, f, c0, c1, need;
  int32_t* out;
};
__device__ __forceinline__ Row row_of(const SelArgs& a, int bh, int r) {
  const mattn_select& p = a.p;
  Row o;
  o.b = bh / p.Hkv;
  o.hk = bh % p.Hkv;
  o.q = a.row0 + r;
  const int nv = visible(p, o.b, o.q);
  o.f = min(p.first, nv);
  const int l = min(p.last, nv - o.f);  // always: [0, f) and [nv - l, nv)
  o.c0 = o.f;
  o.c1 = nv - l;
  o.need = min(p.count, nv) - o.f - l;
  o.out = p.blocks + (((int64_t)o.b * p.L + o.q) * p.Hkv + o.hk) * p.count;
  return o;
}
// What is taken without a look at the scores; whether anything is left to choose.
__device__ __forceinline__ bool take_given(const mattn_select& p, const Row& o, int lane, int lanes) {
  const int all = o.c1 - o.c0 == o.need ? o.need : 0, l = min(p.last, visible(p, o.b, o.q) - o.f);
  for (int i = lane; i < o.f; i += lanes) o.out[i] = i;
  for (int i = lane; i < all; i += lanes) o.out[o.f + i] = o.c0 + i;
  for (int i = lane; i < l; i += lanes) o.out[o.f + o.need + i] = o.c1 + i;
  for (int i = o.f + o.need + l + lane; i < p.count; i += lanes) o.out[i] = -1;
  return o.need > 0 && !all;
}

// Row r of head bh, where float32 ties at the cut: those above it are taken, the ties scored
// in float64 and the best of them chosen.  All lanes of a wave, 64 NV blocks.
template <int NV>
__device__ __forceinline__ void choose_exactly(const SelArgs& a, int bh, int r, float cut, int lane) {
  const mattn_select& p = a.p;
  const Row o = row_of(a, bh, r);
  const float* s = (const float*)a.s + ((int64_t)bh * a.rows + r) * p.nblk;
  double qs[2];  // the summed query, columns lane + 64 c
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    qs[c] = 0.0;
    const int col = lane + 64 * c, G = p.Hq / p.Hkv;
    if (col < p.D)
      for (int g = 0; g < G; ++g) {
        const int64_t e = o.b * p.q_stride[0] + o.q * p.q_stride[1] + (int64_t)(o.hk * G + g) * p.q_stride[2] + col;
        float x[1];
        if (p.dtype == MATTN_F32) load_v<float, 1>(p.q, e, x);
        else if (p.dtype == MATTN_BF16) load_v<bf16_tag, 1>(p.q, e, x);
        else load_v<f16_tag, 1>(p.q, e, x);
        qs[c] += (double)x[0];
      }
  }
  const float* means = p.means + o.b * p.m_stride[0] + o.hk * p.m_stride[2];
  uint64_t key[NV], in[NV], open[NV];  // keys of the open ones (0: not open); those taken for sure; the open ones
  int left = o.need, n_open = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = lane + 64 * i;
    const bool c = j >= o.c0 && j < o.c1;
    float v = c ? s[j] : 0.f;
    v = v != v ? NEG_INF : v;
    open[i] = __ballot(c && v == cut);
    in[i] = __ballot(c && v > cut);
    left -= __builtin_popcountll(in[i]);
    n_open += __builtin_popcountll(open[i]);
    key[i] = 0;
  }
  const bool few = n_open <= 16;  // one after the other, a lane a column; otherwise a lane a block
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (few) {
      for (uint64_t m = open[i]; m; m &= m - 1) {
        const int l = (int)__builtin_ctzll(m);
        const float* row = means + (int64_t)(l + 64 * i) * p.m_stride[1];
        double x = 0.0;
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (lane + 64 * c < p.D) x += qs[c] * (double)row[lane + 64 * c];
#pragma unroll
        for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
        if (lane == l) key[i] = order_key(x);
      }
    } else if (open[i]) {
      const bool mine = (open[i] >> lane) & 1;
      const float* row = means + (int64_t)(mine ? lane + 64 * i : o.c0) * p.m_stride[1];
      double x = 0.0;
#pragma unroll
      for (int c = 0; c < 2; ++c)
        for (int d = 0; d < 64 && 64 * c + d < p.D; ++d) x += __shfl(qs[c], d) * (double)row[64 * c + d];
      if (mine) key[i] = order_key(x);
    }
  }
  const auto keys_from = [&](uint64_t t) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) n += __builtin_popcountll(__ballot(key[i] >= t));
    return n;
  };
  uint64_t t = 0;  // the largest with at least `left` keys at or above it; an exact cut ends the search
  int above = -1;
  for (int bit = 63; bit >= 0 && above != left; --bit) {
    const int n = keys_from(t | (1ull << bit));
    if (n >= left) {
      t |= 1ull << bit;
      above = n;
    }
  }
  // of those equal to t the lowest indices (after an exact cut: none is left to the comparison)
  int equal = above != left ? left - keys_from(t + 1) : 64 * NV, at = o.f;
  const uint64_t below = (1ull << lane) - 1;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const bool same = key[i] != 0 && key[i] == t;
    const uint64_t m = __ballot(same);
    const bool take = ((in[i] >> lane) & 1) || key[i] > t || (same && __builtin_popcountll(m & below) < equal);
    equal -= min(equal, (int)__builtin_popcountll(m));
    const uint64_t w = __ballot(take);
    if (take) o.out[at + __builtin_popcountll(w & below)] = lane + 64 * i;
    at += __builtin_popcountll(w);
  }
}

// LPR lanes hold a row's scores, lane l those of blocks l + LPR i, i < NV; 64 / LPR rows a wave.
template <int LPR, int NV>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256)))
void choose_blocks(SelArgs a) {
  const mattn_select& p = a.p;
  const int lane = threadIdx.x & 63, l = lane & (LPR - 1), bh = blockIdx.y;
  const int r = blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const bool live = r < a.rows;
  const Row o = row_of(a, bh, min(r, a.rows - 1));
  const float* s = (const float*)a.s + ((int64_t)bh * a.rows + min(r, a.rows - 1)) * p.nblk;
  const bool open = live && take_given(p, o, l, LPR);
  const auto fmin_ = [](float x, float y) { return fminf(x, y); };
  const auto fmax_ = [](float x, float y) { return fmaxf(x, y); };
  const auto add_ = [](float x, float y) { return x + y; };

  float v[NV];  // NaN: no candidate (no comparison holds)
  float lo = __builtin_inff(), hi = NEG_INF;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = l + LPR * i;
    v[i] = __builtin_nanf("");
    if (open && j >= o.c0 && j < o.c1) {
      const float x = s[j];
      v[i] = x == x ? x : NEG_INF;
    }
    lo = fminf(lo, v[i]);  // (of a number and NaN the number)
    hi = fmaxf(hi, v[i]);
  }
  lo = row_reduce<LPR>(lo, fmin_);
  hi = row_reduce<LPR>(hi, fmax_);
  const auto count_from = [&](float t) {
    if constexpr (LPR == 64) {
      int n = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) n += __builtin_popcountll(__ballot(v[i] >= t));
      return (float)n;
    } else {
      float n = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) n += v[i] >= t ? 1.f : 0.f;
      return row_reduce<LPR>(n, add_);
    }
  };
  // count(>= lo) >= need, count(>= hi) < need but where hi is the largest value: trials
  // between, which end at an exact cut or at neighbours
  const float need = (float)o.need;
  float above = open ? (float)(o.c1 - o.c0) : 0.f;
  bool go = open && lo < hi;
  if (go) {
    const float n = count_from(hi);
    if (n >= need) {
      lo = hi;
      above = n;
      go = false;
    }
  }
  while (go && above > need) {
    float mid = 0.5f * lo + 0.5f * hi;
    if (!(mid > lo && mid < hi)) {  // neighbours, or infinite: halve their places in the order instead
      const auto place = [](float x) {
        const int32_t b = __builtin_bit_cast(int32_t, x);
        return b < 0 ? (int64_t)(int32_t)0x80000000 - b : (int64_t)b;
      };
      const int64_t a0 = place(lo), b0 = place(hi), m = (a0 + b0) >> 1;
      if (b0 - a0 <= 1) break;
      mid = __builtin_bit_cast(float, m < 0 ? (int32_t)((int64_t)(int32_t)0x80000000 - m) : (int32_t)m);
    }
    const float k = count_from(mid);
    if (k >= need) {
      lo = mid;
      above = k;
    } else {
      hi = mid;
    }
  }
  const bool sure = open && above == need;

  // taken ones in the order of their blocks
  int at = o.f;
  const uint64_t mine = (LPR == 64 ? ~0ull : (1ull << LPR) - 1) << (lane & ~(LPR - 1)), below = mine & ((1ull << lane) - 1);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const bool take = sure && v[i] >= lo;
    const uint64_t m = __ballot(take);
    if (take) o.out[at + __builtin_popcountll(m & below)] = l + LPR * i;
    at += __builtin_popcountll(m & mine);
  }
  // rows with ties at the cut, one after the other with the whole wave
  uint64_t rest = __ballot(open && !sure);
  while (rest) {
    const int from = (int)__builtin_ctzll(rest) & ~(LPR - 1);
    rest &= LPR == 64 ? 0ull : ~(((1ull << LPR) - 1) << from);
    choose_exactly<LPR * NV / 64>(a, bh, __shfl(r, from), __shfl(lo, from), lane);
  }
}

// Any number of blocks: float64 scores, read again for every trial; a wave a row.
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256)))
void choose_wide(SelArgs a) {
  const mattn_select& p = a.p;
  const int lane = threadIdx.x & 63, bh = blockIdx.y, r = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= a.rows) return;
  const Row o = row_of(a, bh, r);
  if (!take_given(p, o, lane, 64)) return;
  const double* s = (const double*)a.s + ((int64_t)bh * a.rows + r) * p.nblk;
  const int steps = (o.c1 + 63) / 64;
  const auto value = [&](int i) -> uint64_t {  // of block lane + 64 i; 0: no candidate
    const int j = lane + 64 * i;
    return j >= o.c0 && j < o.c1 ? order_key(s[j]) : 0;
  };
  const auto count_from = [&](uint64_t t) {
    int n = 0;
    for (int i = 0; i < steps; ++i) n += __builtin_popcountll(__ballot(value(i) >= t));
    return n;
  };
  // the largest t with at least `need` keys at or above it; an exact cut ends the search
  uint64_t t = 0;
  int above = 0;
  for (int bit = 63; bit >= 0 && above != o.need; --bit) {
    const int n = count_from(t | (1ull << bit));
    if (n >= o.need) {
      t |= 1ull << bit;
      above = n;
    }
  }
  const bool cut = above != o.need;
  int equal = cut ? o.need - count_from(t + 1) : 0, at = o.f;  // of those equal to t the lowest indices
  const uint64_t below = (1ull << lane) - 1;
  for (int i = 0; i < steps; ++i) {
    const uint64_t x = value(i), m = __ballot(cut && x == t);
    const bool take = cut ? x > t || (x == t && __builtin_popcountll(m & below) < equal) : x >= t;
    equal -= min(equal, (int)__builtin_popcountll(m));
    const uint64_t w = __ballot(take);
    if (take) o.out[at + __builtin_popcountll(w & below)] = lane + 64 * i;
    at += __builtin_popcountll(w);
  }
}

// ---- host -----------------------------------------------------------------------------

constexpr size_t kScoreBytes = 256u << 20;  // of the scores at most (one row of each at least)
int score_bytes(const mattn_select* p) { return p->nblk > kWide ? 8 : 4; }

// Queries of a launch.
int64_t select_rows(const mattn_select* p) {
  const int64_t per = (int64_t)p->B * p->Hkv * p->nblk * score_bytes(p);
  int64_t rows = (int64_t)kScoreBytes / per;
  rows = rows < 1 ? 1 : rows > 64 ? rows / 64 * 64 : rows;
  return rows < p->L ? rows : p->L;
}

int select_check(const mattn_select* p) {
  if (!p) return MATTN_ERR_NULL;
  if (p->B <= 0 || p->L <= 0 || p->nblk <= 0 || p->Hq <= 0 || p->Hkv <= 0 || p->Hq % p->Hkv) return MATTN_ERR_SHAPE;
  if (p->D <= 0 || p->D > kMaxD || p->D % 8) return MATTN_ERR_HEAD_DIM;
  if (p->block_size <= 0 || p->count <= 0 || p->first < 0 || p->last < 0 || p->first > p->count - p->last)
    return MATTN_ERR_SHAPE;
  if (p->dtype != MATTN_BF16 && p->dtype != MATTN_F16 && p->dtype != MATTN_F32) return MATTN_ERR_DTYPE;
  if (!p->q || !p->means || !p->blocks) return MATTN_ERR_NULL;
  const int es = p->dtype == MATTN_F32 ? 4 : 2;
  if (((uintptr_t)p->q | (uintptr_t)p->means) & 15) return MATTN_ERR_STRIDE;
  for (int i = 0; i < 3; ++i)
    if (p->q_stride[i] < 0 || p->m_stride[i] < 0 || (p->q_stride[i] * es) % 16 || p->m_stride[i] % 4) return MATTN_ERR_STRIDE;
  if ((int64_t)p->B * p->Hkv > 65535 || (int64_t)p->B * p->Hkv * p->L >= (1ll << 31) || p->nblk > (1 << 24))
    return MATTN_ERR_TOO_LARGE;
  return MATTN_OK;
}

template <class Tag>
void launch_scores(const SelArgs& a, hipStream_t st) {
  const mattn_select& p = a.p;
  const int bh = p.B * p.Hkv;
  if (a.rows > kFewRows) {
    // wide spans sum the queries less often: as wide as leaves the card four workgroups a CU
    const int tiles = (a.rows + 63) / 64;
    int span = 512;
    while (span > 64 && (int64_t)tiles * bh * ((p.nblk + span - 1) / span) < 1024) span /= 2;
    const dim3 grid(tiles, (p.nblk + span - 1) / span, bh);
    if (p.D <= 64) hipLaunchKernelGGL((scores_mfma<Tag, 2>), grid, dim3(256), 0, st, a, span);
    else hipLaunchKernelGGL((scores_mfma<Tag, 4>), grid, dim3(256), 0, st, a, span);
    return;
  }
  // enough workgroups to fill the card, at most 16 blocks a group of 16 lanes
  int per = 1;
  while (per < 16 && (int64_t)bh * ((p.nblk + 32 * per - 1) / (32 * per)) >= 1024) per *= 2;
  hipLaunchKernelGGL(scores_few<Tag>, dim3((p.nblk + 16 * per - 1) / (16 * per), bh), dim3(256), 0, st, a, per);
}

void launch_choice(const SelArgs& a, hipStream_t st) {
  const mattn_select& p = a.p;
  const int bh = p.B * p.Hkv;
  const auto grid = [&](int rows) { return dim3((a.rows + rows - 1) / rows, bh); };
  if (p.nblk <= 128) hipLaunchKernelGGL((choose_blocks<16, 8>), grid(16), dim3(256), 0, st, a);
  else if (p.nblk <= 512) hipLaunchKernelGGL((choose_blocks<64, 8>), grid(4), dim3(256), 0, st, a);
  else if (p.nblk <= kWide) hipLaunchKernelGGL((choose_blocks<64, 32>), grid(4), dim3(256), 0, st, a);
  else hipLaunchKernelGGL(choose_wide, grid(4), dim3(256), 0, st, a);
}

}  // namespace
}  // namespace mattn

using namespace mattn;

extern "C" int mattn_block_means(const mattn_means* p, void* stream) {
  if (!p) return MATTN_ERR_NULL;
  if (p->B <= 0 || p->L <= 0 || p->H <= 0 || p->D <= 0 || p->block_size <= 0 || p->new_keys < 0) return MATTN_ERR_SHAPE;
  if (p->dtype != MATTN_BF16 && p->dtype != MATTN_F16 && p->dtype != MATTN_F32) return MATTN_ERR_DTYPE;
  if (!p->k || !p->means) return MATTN_ERR_NULL;
  if (p->new_keys > 0 && p->new_keys > p->L) return MATTN_ERR_SHAPE;
  const int V = p->dtype == MATTN_F32 ? 4 : 8;
  bool vec = p->D % V == 0 && !((uintptr_t)p->k & 15);
  for (int i = 0; i < 3; ++i) {
    if (p->k_stride[i] < 0) return MATTN_ERR_STRIDE;
    vec = vec && p->k_stride[i] % V == 0;
  }
  const int nblk = (int)(((int64_t)p->L + p->block_size - 1) / p->block_size);
  const int nj = p->new_keys > 0 ? (int)((p->new_keys + (int64_t)p->block_size - 2) / p->block_size) + 1 : nblk;
  const int64_t chunks = (int64_t)p->H * p->D / (vec ? V : 1);
  const int64_t groups = (chunks + 31) / 32;
  if (p->B > 65535 || nj <= 0 || groups * nj >= (1ll << 31)) return MATTN_ERR_TOO_LARGE;
  const dim3 grid((uint32_t)(groups * nj), p->B);
  const auto go = [&](auto tag) {
    if (vec) hipLaunchKernelGGL((block_means<decltype(tag), kChunk<decltype(tag)>>), grid, dim3(256), 0, (hipStream_t)stream, *p, nblk,
                                (uint32_t)groups);
    else hipLaunchKernelGGL((block_means<decltype(tag), 1>), grid, dim3(256), 0, (hipStream_t)stream, *p, nblk,
                                (uint32_t)groups);
  };
  if (p->dtype == MATTN_BF16) go(bf16_tag{});
  else if (p->dtype == MATTN_F16) go(f16_tag{});
  else go(float{});
  return hipGetLastError() == hipSuccess ? MATTN_OK : MATTN_ERR_LAUNCH;
}

extern "C" size_t mattn_select_workspace_bytes(const mattn_select* p) {
  if (select_check(p)) return 0;
  return (size_t)select_rows(p) * p->B * p->Hkv * p->nblk * score_bytes(p);
}

extern "C" int mattn_select_blocks(const mattn_select* p, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = select_check(p)) return rc;
  if (!workspace) return MATTN_ERR_NULL;
  if (workspace_bytes < mattn_select_workspace_bytes(p)) return MATTN_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return MATTN_ERR_STRIDE;
  hipStream_t st = (hipStream_t)stream;
  SelArgs a{*p, workspace, p->nblk > kWide, 0, 0};
  const int64_t step = select_rows(p);
  for (int64_t r = 0; r < p->L; r += step) {
    a.row0 = (int)r;
    a.rows = (int)(p->L - r < step ? p->L - r : step);
    if (p->dtype == MATTN_BF16) launch_scores<bf16_tag>(a, st);
    else if (p->dtype == MATTN_F16) launch_scores<f16_tag>(a, st);
    else launch_scores<float>(a, st);
    launch_choice(a, st);
    if (hipGetLastError() != hipSuccess) return MATTN_ERR_LAUNCH;
  }
  return MATTN_OK;
}
