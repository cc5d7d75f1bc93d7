// Selection of key blocks for each query (mattn_block_means, mattn_select_blocks).
//
//   m_j = mean of the keys of block j (float64 sum, rounded once to float32)
//   s_qj = (sum over the group's query heads of q) . m_j, in float64
//   blocks of q: the `first` first and `last` newest visible ones, and the best by s of
//   the others, ties to the lower index; ascending, -1 behind
//
// A selection is whole numbers: neighbours in the order of s lie closer than float32
// holds apart (of 65536 rows of 128 blocks one or two are cut elsewhere by float32
// scores), so the scores are float64, whose order of additions does not show.  Summing
// the group's queries first makes a score cost 2 D flop whatever the group's size.
//
// Scores go to a workspace, rows at a time, in float64; a wave per row then finds the
// n-th best by a search over the bits of the (order-preserving) keys it holds in
// registers: count by ballot how many are at or above a trial threshold.
#include "elem.hpp"

namespace mattn {
namespace {

typedef double f64x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int held_of(const int32_t* lengths, int b, int most) {
  return lengths ? min(max(lengths[b], 0), most) : most;
}

// ---- means ----------------------------------------------------------------------------

// A workgroup forms 32 chunks of V columns of one block: 8 threads a chunk, each every
// eighth key (32 chunks are 512 bytes of a row).  Bound by HBM: each key is read once.
template <class Tag, int V>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256)))
void block_means(mattn_means p, int nblk) {
  __shared__ double red[8][32 * V];
  const int cc = threadIdx.x & 31, kr = threadIdx.x >> 5;
  const int b = blockIdx.z, held = held_of(p.lengths, b, p.L);
  int j = blockIdx.y;
  if (p.new_keys > 0) {  // only the blocks that hold one of the newest keys
    j += max(held - p.new_keys, 0) / p.block_size;
    if ((int64_t)j * p.block_size >= held) return;
  }
  const int cpr = p.D / V;  // chunks of a head's row
  const int64_t c = (int64_t)blockIdx.x * 32 + cc;
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
    const int64_t ci = (int64_t)blockIdx.x * 32 + i / V;
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
  double* s;        // scores of rows [row0, row0 + rows) of each (b, hk): [B * Hkv][rows][nblk]
  int row0, rows;   // queries of this launch
};

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
// the queries, B the means; product e of step j takes the columns 16 j + 4 (l / 16) + e
// of both, so that each lane reads 4 consecutive ones.  A wave holds 16 queries and
// walks 16 blocks at a time; 64 queries by kTileBlocks blocks a workgroup.
constexpr int kTileBlocks = 128;
template <class Tag, int NJ>  // NJ: ceil(D / 16)
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256)))
void scores_mfma(SelArgs a) {
  const mattn_select& p = a.p;
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int b = blockIdx.z / p.Hkv, hk = blockIdx.z % p.Hkv;
  const int q0 = a.row0 + blockIdx.x * 64 + 16 * (threadIdx.x >> 6);
  const int qend = a.row0 + a.rows;
  if (q0 >= qend) return;
  const int most = visible(p, b, min(q0 + 15, qend - 1));  // of the wave's last query: the most
  const int j0 = blockIdx.y * kTileBlocks, j1 = min(j0 + kTileBlocks, most);
  if (j0 >= j1) return;
  double qf[NJ][4];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int col = 16 * j + 4 * g;
    if (col < p.D) {
      sum_group<Tag, 4>(p, b, hk, min(q0 + l16, qend - 1), col, qf[j]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) qf[j][e] = 0.0;
    }
  }
  const float* m = p.means + b * p.m_stride[0] + hk * p.m_stride[2];
  double* out = a.s + ((int64_t)blockIdx.z * a.rows + (q0 - a.row0)) * p.nblk;
  for (int j = j0; j < j1; j += 16) {
    f64x4 c = {0.0, 0.0, 0.0, 0.0};
    const float* row = m + min(j + l16, p.nblk - 1) * p.m_stride[1] + 4 * g;
#pragma unroll
    for (int t = 0; t < NJ; ++t) {
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
      if (16 * t + 4 * g < p.D) x = *(const f32x4*)(row + 16 * t);
#pragma unroll
      for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f64_16x16x4f64(qf[t][e], (double)x[e], c, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (q0 + 4 * i + g < qend && j + l16 < j1) out[(int64_t)(4 * i + g) * p.nblk + j + l16] = c[i];
  }
}

// Few rows: bound by reading the means once.  16 lanes take a block's mean, 8 columns
// each (two steps at D > 128), for all rows; the summed queries lie in LDS.
constexpr int kFewRows = 8;
constexpr int kMaxD = 256;
template <class Tag>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256)))
void scores_few(SelArgs a, int per_group) {
  __shared__ double qs[kFewRows * kMaxD];
  const mattn_select& p = a.p;
  const int b = blockIdx.y / p.Hkv, hk = blockIdx.y % p.Hkv, l16 = threadIdx.x & 15;
  const int most = visible(p, b, a.row0 + a.rows - 1);
  const int j0 = blockIdx.x * 16 * per_group;
  if (j0 >= most) return;
  for (int i = threadIdx.x; i < a.rows * (p.D / 4); i += 256) {
    double x[4];
    sum_group<Tag, 4>(p, b, hk, a.row0 + i / (p.D / 4), 4 * (i % (p.D / 4)), x);
#pragma unroll
    for (int e = 0; e < 4; ++e) qs[4 * i + e] = x[e];
  }
  __syncthreads();
  const float* m = p.means + b * p.m_stride[0] + hk * p.m_stride[2];
  for (int t = 0; t < per_group; ++t) {
    const int j = j0 + 16 * t + (threadIdx.x >> 4);
    if (j >= most) break;
    const float* row = m + j * p.m_stride[1];
    float x[4][4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int col = 64 * c + 4 * l16;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      if (col < p.D) v = *(const f32x4*)(row + col);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[c][e] = v[e];
    }
    for (int r = 0; r < a.rows; ++r) {
      double s = 0.0;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int col = 64 * c + 4 * l16;
        if (col < p.D) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s += qs[r * p.D + col + e] * (double)x[c][e];
        }
      }
#pragma unroll
      for (int o = 8; o; o >>= 1) s += __shfl_xor(s, o);
      if (l16 == 0) a.s[((int64_t)blockIdx.y * a.rows + r) * p.nblk + j] = s;
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

// A wave per row.  NV > 0: lane l holds the keys of blocks l + 64 i, i < NV; NV = 0: any
// number of blocks, read again for every trial.
template <int NV>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256)))
void choose_blocks(SelArgs a) {
  const mattn_select& p = a.p;
  constexpr int kUnroll = NV > 0 ? NV : 1;
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (int64_t)p.B * p.Hkv * a.rows) return;
  const int r = (int)(row % a.rows), bh = (int)(row / a.rows), q = a.row0 + r;
  const int b = bh / p.Hkv, hk = bh % p.Hkv;
  int32_t* out = p.blocks + (((int64_t)b * p.L + q) * p.Hkv + hk) * p.count;
  const int nv = visible(p, b, q);
  const int f = min(p.first, nv), l = min(p.last, nv - f);  // always: [0, f) and [nv - l, nv)
  const int c0 = f, c1 = nv - l;                            // candidates
  const int need = min(p.count, nv) - f - l;
  const double* s = a.s + row * p.nblk;

  for (int i = lane; i < f; i += 64) out[i] = i;
  for (int i = lane; i < l; i += 64) out[f + need + i] = c1 + i;
  for (int i = f + need + l + lane; i < p.count; i += 64) out[i] = -1;
  if (need <= 0) return;
  if (need == c1 - c0) {
    for (int i = lane; i < need; i += 64) out[f + i] = c0 + i;
    return;
  }

  uint64_t v[NV > 0 ? NV : 1];
  const auto key = [&](int i) -> uint64_t {  // of block lane + 64 i; 0: no candidate
    const int j = lane + 64 * i;
    return j >= c0 && j < c1 ? order_key(s[j]) : 0;
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = key(i);
  }
  const int steps = NV > 0 ? NV : (c1 + 63) / 64;
  const auto value = [&](int i) -> uint64_t {
    if constexpr (NV > 0) return v[i];
    else return key(i);
  };
  const auto count_from = [&](uint64_t t) {
    int n = 0;
#pragma unroll kUnroll
    for (int i = 0; i < steps; ++i) n += __builtin_popcountll(__ballot(value(i) >= t));
    return n;
  };
  // the largest t with at least `need` keys at or above it; an exact cut ends the search
  uint64_t t = 0;
  int above = 0;
  for (int bit = 63; bit >= 0; --bit) {
    const uint64_t trial = t | (1ull << bit);
    const int n = count_from(trial);
    if (n >= need) {
      t = trial;
      above = n;
      if (n == need) break;
    }
  }
  // ties at t: the lowest indices
  int ties = 0;  // how many of those equal to t are taken
  const bool cut = above != need;
  if (cut) ties = need - count_from(t + 1);
  int at = f;
#pragma unroll kUnroll
  for (int i = 0; i < steps; ++i) {
    const uint64_t x = value(i);
    bool take = cut ? x > t : x >= t;
    if (cut) {
      const uint64_t same = __ballot(x == t);
      take = take || (x == t && __builtin_popcountll(same & ((1ull << lane) - 1)) < ties);
      ties -= min(ties, (int)__builtin_popcountll(same));
    }
    const uint64_t m = __ballot(take);
    if (take) out[at + __builtin_popcountll(m & ((1ull << lane) - 1))] = lane + 64 * i;
    at += __builtin_popcountll(m);
  }
}

// ---- host -----------------------------------------------------------------------------

constexpr size_t kScoreBytes = 256u << 20;  // of the scores' workspace at most (one row of each at least)

int64_t select_rows(const mattn_select* p) {
  const int64_t per = (int64_t)p->B * p->Hkv * p->nblk * 8;
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
  if (a.rows <= kFewRows) {
    // enough workgroups to fill the card, at most 8 blocks a group of 16 lanes
    int per = 1;
    while (per < 8 && (int64_t)bh * ((p.nblk + 32 * per - 1) / (32 * per)) >= 1024) per *= 2;
    hipLaunchKernelGGL(scores_few<Tag>, dim3((p.nblk + 16 * per - 1) / (16 * per), bh), dim3(256), 0, st, a, per);
    return;
  }
  const dim3 grid((a.rows + 63) / 64, (p.nblk + kTileBlocks - 1) / kTileBlocks, bh);
  if (p.D <= 64) hipLaunchKernelGGL((scores_mfma<Tag, 4>), grid, dim3(256), 0, st, a);
  else if (p.D <= 128) hipLaunchKernelGGL((scores_mfma<Tag, 8>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((scores_mfma<Tag, 16>), grid, dim3(256), 0, st, a);
}

void launch_choice(const SelArgs& a, hipStream_t st) {
  const int64_t rows = (int64_t)a.p.B * a.p.Hkv * a.rows;
  const dim3 grid((uint32_t)((rows + 3) / 4));
  if (a.p.nblk <= 128) hipLaunchKernelGGL(choose_blocks<2>, grid, dim3(256), 0, st, a);
  else if (a.p.nblk <= 512) hipLaunchKernelGGL(choose_blocks<8>, grid, dim3(256), 0, st, a);
  else if (a.p.nblk <= 2048) hipLaunchKernelGGL(choose_blocks<32>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(choose_blocks<0>, grid, dim3(256), 0, st, a);
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
  if (p->B > 65535 || nj > 65535 || nj <= 0 || (chunks + 31) / 32 >= (1ll << 31)) return MATTN_ERR_TOO_LARGE;
  const dim3 grid((uint32_t)((chunks + 31) / 32), nj, p->B);
  const auto go = [&](auto tag) {
    if (vec) hipLaunchKernelGGL((block_means<decltype(tag), kChunk<decltype(tag)>>), grid, dim3(256), 0, (hipStream_t)stream, *p, nblk);
    else hipLaunchKernelGGL((block_means<decltype(tag), 1>), grid, dim3(256), 0, (hipStream_t)stream, *p, nblk);
  };
  if (p->dtype == MATTN_BF16) go(bf16_tag{});
  else if (p->dtype == MATTN_F16) go(f16_tag{});
  else go(float{});
  return hipGetLastError() == hipSuccess ? MATTN_OK : MATTN_ERR_LAUNCH;
}

extern "C" size_t mattn_select_workspace_bytes(const mattn_select* p) {
  if (select_check(p)) return 0;
  return (size_t)select_rows(p) * p->B * p->Hkv * p->nblk * 8;
}

extern "C" int mattn_select_blocks(const mattn_select* p, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = select_check(p)) return rc;
  if (!workspace) return MATTN_ERR_NULL;
  if (workspace_bytes < mattn_select_workspace_bytes(p)) return MATTN_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return MATTN_ERR_STRIDE;
  SelArgs a{*p, (double*)workspace, 0, 0};
  const int64_t step = select_rows(p);
  for (int64_t r = 0; r < p->L; r += step) {
    a.row0 = (int)r;
    a.rows = (int)(p->L - r < step ? p->L - r : step);
    if (p->dtype == MATTN_BF16) launch_scores<bf16_tag>(a, (hipStream_t)stream);
    else if (p->dtype == MATTN_F16) launch_scores<f16_tag>(a, (hipStream_t)stream);
    else launch_scores<float>(a, (hipStream_t)stream);
    launch_choice(a, (hipStream_t)stream);
    if (hipGetLastError() != hipSuccess) return MATTN_ERR_LAUNCH;
  }
  return MATTN_OK;
}
