// Attention of each query over the key blocks selected for it (mattn_selected_fwd,
// mattn_selected_bwd).
//
//   O_q = sum_k P_qk V_k over the keys k of q's blocks that q sees,
//   P_qk = exp(scale q.k - lse_q); the blocks are shared by the G query heads of a key head
//   delta = dO . O, dS = P (dO . V - delta) scale; dQ = dS K, dK = dS^T Q, dV = P^T dO
//
// Three forms (sel_plan).  By queries (few rows, one token of each sequence): a workgroup takes
// one query and key head, its waves the tiles of 32 keys of its blocks.  By tiles of queries:
// a wave holds 32 neighbouring rows (query, head) and walks the union of their blocks.  By
// blocks: the queries that selected a block are listed once (list_* kernels), and a workgroup
// takes a block's keys and some hundred rows of its list: whole matrix-core tiles whatever the
// group is, K and V read once for all of them; a row's partial results of its blocks (float32,
// with a log-sum-exp each, at [row][slot of the block in the query's selection], so that
// nothing is added in an order of chance) are joined by a second kernel.  dK and dV are always
// formed by blocks, dQ by tiles (from the dS that the dK/dV kernel leaves in memory) or blocks.
//
// Infinite and NaN values: 0 times one is NaN in a matrix product, so a tile with such
// values in rows that some of its queries (keys) must not see would spoil those.  The
// products run with such values as 0 and mark the block, and the joining kernels add what
// they give to the results that do see them, from the formula.
//
// Bound by HBM reads of K and V (by queries), by LDS reads and the exponentials beside the
// matrix products (by tiles, dK/dV), and by the partial rows (by blocks with narrow blocks):
// D * 4 bytes written and read for each (row, block).  Measured in 16 bits at d = 128:
// [1, 8192, 32/8], 16 blocks of 64 keys: forward 0.62 ms (union's products at 0.8 PFLOP/s,
// 3.6 times those of the selections), dK/dV 0.65 ms (0.40 PFLOP/s), dQ 0.42 ms; [1, 16384,
// 16/4], 4 blocks of 512: 0.43 ms and 0.15 ms of joining (4.2 TB/s); one token of each of 32
// sequences, 64 blocks of 64: 105 us (5.1 TB/s).
#include <math.h>

#include <initializer_list>

#include "selected.hpp"

namespace mattn {
namespace {

constexpr int kChunkQ = 256;    // queries a list workgroup takes
constexpr int kRange = 1024;    // blocks a list workgroup takes
constexpr int kSlotBits = 10;   // of a list entry
constexpr int kMaxSel = 1 << kSlotBits;  // blocks of a query
constexpr int kRows = 512;      // rows (query, head) of a block that a forward or dQ workgroup takes at most
constexpr int kRowsKV = 2048;   // rows that a dK/dV workgroup takes at most
constexpr int kMaxDS = 1024;    // keys of a block whose dS is kept in memory

struct Desc {
  int blk, row0;  // block (-1: idle) and first row of its list
};

struct SArgs {
  mattn_selected p;
  int G, nblk, bh_n;
  float scale_log2;
  const void *q, *k, *v, *dO;
  void *o, *dq, *dk, *dv;
  float *o32, *lse, *delta;  // [B * Hkv][Lq][G] rows (o32 [rows][D])
  float *part, *plse;        // [rows][count][D], [rows][count]
  float* kvpart;             // [B * Hkv][max_kv][2][KT][D]
  int *odd, *kvodd;          // [B * Hkv][nblk]: infinite or NaN values were left out (of V or K; of Q or dO)
  // lists
  uint32_t* ok;              // [B * Hkv][Lq][words]: slots that count (visible, first of their block)
  int* cnt;                  // [B * Hkv][nblk][chunks]: entries of a chunk, then their first index in the block's list
  int* off;                  // [B * Hkv][nblk + 1]
  int* kvoff;                // [B * Hkv][nblk + 1]: first dK/dV item of a block
  int* ent;                  // [B * Hkv][Lq * count]: (query << kSlotBits) + slot, by block, in the order of queries
  int* pos;                  // [B * Hkv][Lq * count]: index in ent of each query's slots that count
  void* ds;                  // [B * Hkv][Lq * count (as ent)][G][block_size] dS / scale, the inputs' type (or null)
  Desc *tile, *kvtile;       // [B * Hkv][max_tiles], [B * Hkv][max_kv]
  int words, chunks, max_tiles, max_kv, subs;  // subs: dK/dV key tiles of a block
  int rows_q, rows_kv;                         // rows of a work item
};

__device__ __forceinline__ int keys_held(const mattn_selected& p, int b) {
  return p.lengths ? min(max(p.lengths[b], 0), p.Lk) : p.Lk;
}
__device__ __forceinline__ int64_t first_pos(const mattn_selected& p, int b) { return p.starts ? p.starts[b] : 0; }
// Keys of sequence b that query q sees: those below the result.
__device__ __forceinline__ int key_limit(const mattn_selected& p, int b, int q, int held, int64_t start) {
  if (!p.causal) return held;
  const int64_t e = start + q + 1;
  return e < 0 ? 0 : e < held ? (int)e : held;
}

// ---- lists ----------------------------------------------------------------------------

// The queries of a chunk that selected each block of a range, as bit masks in LDS; the
// selection of query q: slots in order, entries outside [0, blocks seen) and repeated ones
// left out.  FILL: the entries go to their places, otherwise the masks are counted.
template <bool FILL>
__global__ __attribute__((amdgpu_flat_work_group_size(kChunkQ, kChunkQ)))
void list_entries(SArgs a) {
  __shared__ uint32_t bits[kRange][kChunkQ / 32];
  const mattn_selected& p = a.p;
  const int bh = blockIdx.z, b = bh / p.Hkv, hk = bh % p.Hkv, chunk = blockIdx.x;
  const int lo = blockIdx.y * kRange, n = min(kRange, a.nblk - lo);
  const int t = threadIdx.x, q = chunk * kChunkQ + t;
  for (int i = t; i < n * (kChunkQ / 32); i += kChunkQ) (&bits[0][0])[i] = 0u;
  __syncthreads();
  const int32_t* sel = p.blocks + (((int64_t)b * p.Lq + q) * p.Hkv + hk) * p.count;
  const uint32_t mine = 1u << (t & 31);
  int seen = 0;
  if (q < p.Lq) {
    const int lim = key_limit(p, b, q, keys_held(p, b), first_pos(p, b));
    seen = (lim + p.block_size - 1) / p.block_size;
    for (int w = 0; w < a.words; ++w) {
      uint32_t good = 0u;
      for (int c = 32 * w; c < min(32 * w + 32, p.count); ++c) {
        const int j = sel[c] - lo;
        if (j >= 0 && j < n && j + lo < seen && !(atomicOr(&bits[j][t >> 5], mine) & mine)) good |= 1u << (c & 31);
      }
      if constexpr (!FILL) {  // (ranges hold different blocks: their bits are joined in any order)
        uint32_t* o = a.ok + ((int64_t)bh * p.Lq + q) * a.words + w;
        if (gridDim.y == 1) *o = good;
        else if (good) atomicOr(o, good);
      }
    }
  }
  __syncthreads();
  if constexpr (!FILL) {
    for (int j = t; j < n; j += kChunkQ) {
      int s = 0;
#pragma unroll
      for (int w = 0; w < kChunkQ / 32; ++w) s += __popc(bits[j][w]);
      a.cnt[((int64_t)bh * a.nblk + lo + j) * a.chunks + chunk] = s;
    }
  } else if (q < p.Lq) {
    for (int w = 0; w < a.words; ++w) {
      uint32_t good = a.ok[((int64_t)bh * p.Lq + q) * a.words + w];
      for (; good; good &= good - 1) {
        const int c = 32 * w + __ffs(good) - 1, j = sel[c] - lo;
        if (j < 0 || j >= n) continue;
        int r = __popc(bits[j][t >> 5] & (mine - 1));
        for (int x = 0; x < (t >> 5); ++x) r += __popc(bits[j][x]);
        const int64_t head = (int64_t)bh * p.Lq * p.count;
        const int at = a.off[(int64_t)bh * (a.nblk + 1) + lo + j] + a.cnt[((int64_t)bh * a.nblk + lo + j) * a.chunks + chunk] + r;
        a.ent[head + at] = (q << kSlotBits) + c;
        a.pos[head + (int64_t)q * p.count + c] = at;
      }
    }
  }
}

__global__ __attribute__((amdgpu_flat_work_group_size(256, 256)))
void list_clear(uint32_t* x, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) x[i] = 0u;
}

// inclusive sum over the lanes of a wave
__device__ __forceinline__ int wave_scan(int x, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  return x;
}

// Counts of a block's chunks to first indices; the block's total to off (a wave a block).
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256)))
void list_chunks(SArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= (int64_t)a.bh_n * a.nblk) return;
  int* c = a.cnt + i * a.chunks;
  int sum = 0;
  for (int x = 0; x < a.chunks; x += 64) {
    const int v = x + lane < a.chunks ? c[x + lane] : 0, s = wave_scan(v, lane);
    if (x + lane < a.chunks) c[x + lane] = sum + s - v;
    sum += __shfl(s, 63);
  }
  if (lane == 0) a.off[i / a.nblk * (a.nblk + 1) + i % a.nblk] = sum;
}

// Totals to first entries, and the work items of the list kernels (a workgroup a head).
constexpr int kScan = 1024;
__global__ __attribute__((amdgpu_flat_work_group_size(kScan, kScan)))
void list_items(SArgs a) {
  __shared__ int wsum[3][kScan / 64];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  int* off = a.off + (int64_t)blockIdx.x * (a.nblk + 1);
  int* kvoff = a.kvoff + (int64_t)blockIdx.x * (a.nblk + 1);
  Desc* tile = a.tile + (int64_t)blockIdx.x * a.max_tiles;
  Desc* kvtile = a.kvtile + (int64_t)blockIdx.x * a.max_kv;
  int base[3] = {0, 0, 0};  // entries, tiles, dK/dV items before this range
  for (int j0 = 0; j0 < a.nblk; j0 += kScan) {
    const int j = j0 + t, n = j < a.nblk ? off[j] : 0;
    const int rows = n * a.G;
    const int v[3] = {n, (rows + a.rows_q - 1) / a.rows_q, (rows + a.rows_kv - 1) / a.rows_kv * a.subs};
    int s[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      s[i] = wave_scan(v[i], lane);
      if (lane == 63) wsum[i][w] = s[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      int before = base[i], all = 0;
      for (int x = 0; x < kScan / 64; ++x) {
        before += x < w ? wsum[i][x] : 0;
        all += wsum[i][x];
      }
      s[i] += before - v[i];
      base[i] += all;
    }
    __syncthreads();
    if (j < a.nblk) {
      off[j] = s[0];
      kvoff[j] = s[2];
      a.odd[(int64_t)blockIdx.x * a.nblk + j] = 0;
    }
    // the range's items, a wave a block at a time (values of the wave's own 64 blocks)
    for (int x = 0; x < 64 && j0 + 64 * w + x < a.nblk; ++x) {
      const int nt = __shfl(v[1], x), st = __shfl(s[1], x), nk = __shfl(v[2], x), sk = __shfl(s[2], x);
      for (int i = lane; i < nt; i += 64) tile[st + i] = Desc{j0 + 64 * w + x, i * a.rows_q};
      // (key tile, rows): the tiles of a block next to each other
      for (int i = lane; i < nk; i += 64) kvtile[sk + i] = Desc{j0 + 64 * w + x, i};
    }
  }
  if (t == 0) {
    off[a.nblk] = base[0];
    kvoff[a.nblk] = base[2];
  }
  for (int i = base[1] + t; i < a.max_tiles; i += kScan) tile[i] = Desc{-1, 0};
  for (int i = base[2] + t; i < a.max_kv; i += kScan) kvtile[i] = Desc{-1, 0};
}

// ---- by blocks and by tiles: parts of both ----------------------------------------------

// Row r of a block's list: its query, slot and head.
struct RowId {
  int q, slot, g;
};
__device__ __forceinline__ RowId row_id(const SArgs& a, const int* list, int r) {
  const int e = r / a.G, x = list[e];
  return RowId{x >> kSlotBits, x & ((1 << kSlotBits) - 1), r - e * a.G};
}

// Rows k0 .. k0 + N - 1 of a [L, D] slice to LDS, zeros for rows at or past `end` and columns
// at or past d.  Whether this thread's part holds an infinite or NaN value; CLEAN: 0 for those.
template <class Tag, int D, int N, bool CLEAN>
__device__ __forceinline__ bool stage_keys(char* lds, const void* base, int64_t stride, int64_t k0, int end, int d) {
  bool odd = false;
  using T = STile<Tag, D>;
  constexpr int EC = 16 / SOp<Tag>::ES;  // elements of a chunk
#pragma unroll
  for (int i = 0; i < N * T::CPR / 256; ++i) {
    const int x = i * 256 + threadIdx.x, r = x / T::CPR, c = x % T::CPR;
    u32x4 v = {0u, 0u, 0u, 0u};
    if (k0 + r < end && c * EC < d) v = *(const u32x4*)((const char*)base + SOp<Tag>::ES * ((k0 + r) * stride + c * EC));
    if (SOp<Tag>::odd(v)) {
      odd = true;
      if constexpr (CLEAN) v = SOp<Tag>::finite16(v);
    }
    *(u32x4*)(lds + T::at(r, c)) = v;
  }
  return odd;
}

template <class Tag, int D>
__device__ __forceinline__ void load_rows(typename SOp<Tag>::Frag (&f)[D / 16], const void* base, int64_t at, int hi, int d) {
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    const int c = 16 * s + 8 * hi;
    f[s] = c < d ? SOp<Tag>::load((const char*)base + SOp<Tag>::ES * (at + c)) : SOp<Tag>::zero();
  }
}

// O^T (register 4 j + i of tile mt: column 32 mt + 8 j + 4 hi + i of the lane's row) to a row of floats
template <int D>
__device__ __forceinline__ void put_row(float* out, const f32x16 (&acc)[D / 32], float s, int hi, int d) {
#pragma unroll
  for (int mt = 0; mt < D / 32; ++mt)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = 32 * mt + 8 * j + 4 * hi;
      if (c < d)
        *(f32x4*)(out + c) = f32x4{acc[mt][4 * j] * s, acc[mt][4 * j + 1] * s, acc[mt][4 * j + 2] * s, acc[mt][4 * j + 3] * s};
    }
}

// Bits r of rows 8 (r / 4) + 4 hi + r % 4 (from row 0 of a 32-row tile) below `lim`.
__device__ __forceinline__ uint32_t below(int lim, int hi) {
  uint32_t m = 0u;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = min(max(lim - 8 * j - 4 * hi, 0), 4);
    m |= ((1u << n) - 1u) << (4 * j);
  }
  return m;
}

// Bit i of vis as all ones or zero, opaque to the compiler (which would make it a compare
// and a select): masking an element is then one bit operation.
__device__ __forceinline__ uint32_t seen_bit(uint32_t vis, int i) {
  uint32_t m = (uint32_t)__builtin_amdgcn_sbfe((int)vis, i, 1);
  asm("" : "+v"(m));
  return m;
}

constexpr int kKT = 64;  // keys of a staged tile

// One tile of 64 keys for a wave's 32 rows (lane = row, `see` of its keys): scores, the
// running maximum m (of scores before sl, the positive scale in base 2) and sum, and O.  The
// scores are formed transposed (rows of the MFMA result: keys), so that a row's softmax is one
// lane's and its neighbour's, and P^T is the next product's operand as it stands.  The maximum
// moves only when a score passes it by 2^8 (the weights are then below 2^8, in every type's
// range), so that the sums are hardly ever rescaled.  The sum adds the weights as rounded to
// the inputs' type, so that O is a weighted mean of V's rows; its logarithm is the row's lse,
// here and in the backward.  slow: rows are masked element by element; otherwise one that sees
// none of the tile gets weights 0 by an infinite subtrahend (NaN where a score is not finite).
template <class Tag, int D>
__device__ __forceinline__ void attend_tile(const char* kt, const char* vt, const typename SOp<Tag>::Frag (&qf)[D / 16], int see, bool slow,
                                            float sl, int lane, float& m, float& sum, f32x16 (&acc)[D / 32]) {
  using O = SOp<Tag>;
  using T = STile<Tag, D>;
  const int l32 = lane & 31, hi = lane >> 5;
  float s[2][16];  // (single floats: of a 16-register result changed in a branch the compiler has
                   // written back registers of another value)
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    f32x16 r16 = f32x16{};
#pragma unroll
    for (int c = 0; c < D / 16; ++c) r16 = O::mma32(T::row(kt, 32 * u + l32, 2 * c + hi), qf[c], r16);
#pragma unroll
    for (int i = 0; i < 16; ++i) s[u][i] = r16[i];
  }
  if constexpr (O::ES == 2) reads_ahead<2 * D / 16, 6, 1>();
  if (slow) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t vis = below(see - 32 * u, hi);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[u][i] = mask_neg_inf(s[u][i], seen_bit(vis, i));
    }
  }
  float top = NEG_INF;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int i = 0; i < 16; i += 2) top = fmaxf(fmaxf(s[u][i], s[u][i + 1]), top);
  top = see > 0 ? wave_max32(top) : NEG_INF;  // (both halves of a row have one `see`)
  if (__any((top - m) * sl > 8.f)) {          // (the first scores of a row: m is -inf)
    const float to = fmaxf(m, top), keep = to == NEG_INF ? 1.f : fast_exp2((m - to) * sl);
    m = to;
    sum *= keep;
#pragma unroll
    for (int mt = 0; mt < D / 32; ++mt) acc[mt] *= keep;
  }
  const float ref = see > 0 ? (m == NEG_INF ? 0.f : m * sl) : -NEG_INF;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[u][i] = fast_exp2(__builtin_fmaf(s[u][i], sl, -ref));
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = s[u][8 * j + i];
      const auto f = O::pack(y);
      sum = O::total(f, sum);
#pragma unroll
      for (int mt = 0; mt < D / 32; ++mt) acc[mt] = O::mma32(T::tr32(vt, 2 * u + j, mt, lane), f, acc[mt]);
    }
  }
  if constexpr (O::ES == 2) reads_ahead<4 * D / 32, 6, 2>();
}

// Forward and dQ.  Four waves of 32 rows each (lane = row, both halves of a wave), 128 rows
// at a time.  The tile of a block of at most 64 keys stays in LDS for all rows; of a wider one,
// forward in 16 bits, the next tile's loads are on their way while this one's products run.
// P and dS are rounded to the inputs' type (as V and K are), sums are float32.
template <class Tag, int D, bool GRAD>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256), amdgpu_waves_per_eu(SOp<Tag>::ES == 2 && (D == 64 || !GRAD) ? 2 : 1)))
void by_block_q(SArgs a) {
  using O = SOp<Tag>;
  using T = STile<Tag, D>;
  constexpr bool AHEAD = !GRAD && O::ES == 2;
  __shared__ __align__(16) char lds[AHEAD ? 2 : 1][2 * kKT * T::RB];
  const mattn_selected& p = a.p;
  const int bh = blockIdx.x % a.bh_n, b = bh / p.Hkv, hk = bh % p.Hkv;
  const Desc desc = a.tile[(int64_t)bh * a.max_tiles + blockIdx.x / a.bh_n];
  if (desc.blk < 0) return;
  const int* off = a.off + (int64_t)bh * (a.nblk + 1) + desc.blk;
  const int* list = a.ent + (int64_t)bh * p.Lq * p.count + off[0];
  const int rows = min((off[1] - off[0]) * a.G - desc.row0, a.rows_q);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l32 = lane & 31, hi = lane >> 5;
  const int held = keys_held(p, b);
  const int64_t start = first_pos(p, b), k0 = (int64_t)desc.blk * p.block_size;
  const int inside = (int)min((int64_t)p.block_size, held - k0);  // keys of the block
  const int tiles = (inside + kKT - 1) / kKT;
  const char* kb = (const char*)a.k + O::ES * (b * p.k_stride[0] + hk * p.k_stride[2]);
  const char* vb = (const char*)a.v + O::ES * (b * p.v_stride[0] + hk * p.v_stride[2]);
  const bool zero = p.scale == 0.f;
  const float sl = zero ? 1.f : fabsf(a.scale_log2);  // (forward: the scale's sign is Q's)

  // a row's operands; those of the next 128 rows are loaded ahead of the products of these
  struct Rows {
    RowId id;
    typename O::Frag q[D / 16], g[GRAD ? D / 16 : 1];
    float lse, delta;
  };
  const auto load = [&](Rows& x, int r0) {
    x.id = row_id(a, list, desc.row0 + min(r0 + 32 * wave + l32, rows - 1));
    const int h = hk * a.G + x.id.g;
    load_rows<Tag, D>(x.q, a.q, b * p.q_stride[0] + x.id.q * p.q_stride[1] + h * p.q_stride[2], hi, p.D);
    if constexpr (GRAD) {
      const int64_t row = ((int64_t)bh * p.Lq + x.id.q) * a.G + x.id.g;
      load_rows<Tag, D>(x.g, a.dO, b * p.do_stride[0] + x.id.q * p.do_stride[1] + h * p.do_stride[2], hi, p.D);
      x.lse = a.lse[row];
      x.delta = a.delta[row];
    }
  };
  // AHEAD: a tile on its way, this thread's chunks of it
  constexpr int EC = 16 / O::ES, N = AHEAD ? kKT * T::CPR / 256 : 1, RPI = 256 / T::CPR;
  const int my_r = threadIdx.x / T::CPR, my_c = threadIdx.x % T::CPR;
  u32x4 xk[N], xv[N];
  const auto fetch = [&](int t) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = t * kKT + i * RPI + my_r;
      const bool in = r < inside && my_c * EC < p.D;
      xk[i] = in ? *(const u32x4*)(kb + O::ES * ((k0 + r) * p.k_stride[1] + my_c * EC)) : u32x4{0u, 0u, 0u, 0u};
      xv[i] = in ? *(const u32x4*)(vb + O::ES * ((k0 + r) * p.v_stride[1] + my_c * EC)) : u32x4{0u, 0u, 0u, 0u};
    }
  };
  // the tile on its way to LDS; infinite and NaN values of V as 0, and the block marked
  const auto put = [&](char* kt) {
    bool odd = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = i * RPI + my_r;
      if (O::odd(xv[i])) {
        odd = true;
        xv[i] = O::finite16(xv[i]);
      }
      *(u32x4*)(kt + T::at(r, my_c)) = xk[i];
      *(u32x4*)(kt + kKT * T::RB + T::at(r, my_c)) = xv[i];
    }
    if (odd) a.odd[(int64_t)bh * a.nblk + desc.blk] = 1;
  };

  constexpr bool EARLY = O::ES == 2 || !GRAD || D == 64;  // (float32's Q and dO at D = 128: 128 registers, twice would spill)
  Rows next;
  if constexpr (EARLY) load(next, 0);
  if constexpr (AHEAD) fetch(0);
  int buf = 0;
  bool odd = false;  // GRAD: some tile of K holds an infinite or NaN value
  for (int r0 = 0; r0 < rows; r0 += 128) {
    const bool live = r0 + 32 * wave + l32 < rows;
    Rows now;
    if constexpr (EARLY) {
      now = next;
      if (r0 + 128 < rows) load(next, r0 + 128);
    } else {
      load(now, r0);
    }
    const RowId id = now.id;
    const int64_t row = ((int64_t)bh * p.Lq + id.q) * a.G + id.g;
    const int64_t lim = key_limit(p, b, id.q, held, start) - k0;  // keys of the block the row sees
    const int seen = (int)min(lim, (int64_t)inside);
    const int64_t out = row * p.count + id.slot;
    f32x16 acc[D / 32];
    if constexpr (!GRAD) {
#pragma unroll
      for (int c = 0; c < D / 16; ++c) now.q[c] = O::sign(now.q[c], p.scale < 0.f, zero);
#pragma unroll
      for (int mt = 0; mt < D / 32; ++mt) acc[mt] = f32x16{};
      float m = NEG_INF, sum = 0.f;
      for (int t = 0; t < tiles; ++t) {
        char* kt = lds[buf];
        if (tiles > 1 || r0 == 0) {
          if constexpr (AHEAD) {
            // (the tile before lies in the other buffer, and all were done with this one's last before they came to it)
            put(kt);
            barrier_lds();
            if (tiles > 1) {
              buf ^= 1;
              if (t + 1 < tiles || r0 + 128 < rows) fetch(t + 1 < tiles ? t + 1 : 0);
            }
          } else {
            __syncthreads();
            stage_keys<Tag, D, kKT, false>(kt, kb, p.k_stride[1], k0 + t * kKT, (int)(k0 + inside), p.D);
            if (stage_keys<Tag, D, kKT, true>(kt + kKT * T::RB, vb, p.v_stride[1], k0 + t * kKT, (int)(k0 + inside), p.D))
              a.odd[(int64_t)bh * a.nblk + desc.blk] = 1;
            __syncthreads();
          }
        }
        const int see = min(seen - t * kKT, kKT);
        if (__any(see > 0)) attend_tile<Tag, D>(kt, kt + kKT * T::RB, now.q, see, __any(see < kKT), sl, lane, m, sum, acc);
      }
      sum = wave_sum32(sum);
      const bool some = sum > 0.f || sum != sum;
      if (live) {
        put_row<D>(a.part + out * p.D, acc, some ? 1.f / sum : 0.f, hi, p.D);
        if (hi == 0) a.plse[out] = some ? __builtin_fmaf(m, sl, __log2f(sum)) : NEG_INF;
      }
    } else {
      char *kt = lds[0], *vt = kt + kKT * T::RB;
      const auto walk = [&](auto careful) {
#pragma unroll
        for (int mt = 0; mt < D / 32; ++mt) acc[mt] = f32x16{};
        for (int t = 0; t < tiles; ++t) {
          if (tiles > 1 || (r0 == 0 && !decltype(careful)::value)) {
            __syncthreads();
            const bool ko = stage_keys<Tag, D, kKT, false>(kt, kb, p.k_stride[1], k0 + t * kKT, (int)(k0 + inside), p.D);
            stage_keys<Tag, D, kKT, false>(vt, vb, p.v_stride[1], k0 + t * kKT, (int)(k0 + inside), p.D);
            if (ko) a.odd[(int64_t)bh * a.nblk + desc.blk] = 1;
            odd = __syncthreads_or(ko) || odd;
          }
          // (opaque: places in LDS worked out ahead of the loop would take the registers of the operands)
          int tid = threadIdx.x;
          asm("" : "+v"(tid));
          const int lane = tid & 63, l32 = lane & 31, hi = lane >> 5;
          const bool part = __any(seen < (t + 1) * kKT);  // some row of the wave does not see all of the tile
          // S^T of 32 keys, single floats from here on (as in attend_tile)
          const auto scores = [&](const char* tile, const typename O::Frag(&f)[D / 16], int x, float(&s)[16]) {
            f32x16 r16 = f32x16{};
#pragma unroll
            for (int c = 0; c < D / 16; ++c) r16 = O::mma32(T::row(tile, 32 * x + l32, 2 * c + hi), f[c], r16);
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = r16[i];
          };
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float s[16], dp[16];
            scores(kt, now.q, x, s);
            scores(vt, now.g, x, dp);
            const uint32_t vis = part ? below(seen - t * kKT - 32 * x, hi) : 0xffffu;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float w = fast_exp2(s[i] * a.scale_log2 - now.lse) * (dp[i] - now.delta);
              s[i] = !part || ((vis >> i) & 1u) ? w : 0.f;
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float e[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) e[i] = s[8 * j + i];
              const auto f = O::pack(e);
#pragma unroll
              for (int mt = 0; mt < D / 32; ++mt) {
                auto y = T::tr32(kt, 2 * x + j, mt, lane);
                if constexpr (decltype(careful)::value) y = O::finite(y);
                acc[mt] = O::mma32(y, f, acc[mt]);
              }
            }
          }
        }
      };
      walk(std::false_type{});
      if (odd) walk(std::true_type{});
      if (live) put_row<D>(a.part + out * p.D, acc, p.scale, hi, p.D);
    }
  }
}

// dK and dV of a key tile from a.rows_kv rows of its list, float32: KT keys (64, or 128 for
// blocks of at least 128), 64 rows at a time in LDS.  A wave holds 32 keys (lane = key) as
// operands in registers and, with KT = 64, every other 32 rows; the scores' result has the rows
// along its registers, so P and dS are the operands of dV^T = dO^T P and dK^T = Q^T dS as they
// stand.  Partial sums per item; the items of a block are added in order.
template <int D, int KT>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256)))
void by_block_kv(SArgs a) {
  using Tag = float;
  using O = SOp<Tag>;
  using T = STile<Tag, D>;
  constexpr int NR = 64, KG = KT / 32, RG = 4 / KG;
  __shared__ __align__(16) char lds[2 * NR * T::RB];
  __shared__ __align__(16) float s_lse[NR], s_delta[NR];
  __shared__ __align__(16) int s_see[NR];
  __shared__ int64_t s_q[NR], s_g[NR];
  const mattn_selected& p = a.p;
  const int bh = blockIdx.x % a.bh_n, b = bh / p.Hkv, hk = bh % p.Hkv;
  const int64_t item = (int64_t)bh * a.max_kv + blockIdx.x / a.bh_n;
  const Desc desc = a.kvtile[item];
  if (desc.blk < 0) return;
  const int* off = a.off + (int64_t)bh * (a.nblk + 1) + desc.blk;
  const int* list = a.ent + (int64_t)bh * p.Lq * p.count + off[0];
  const int per = ((off[1] - off[0]) * a.G + a.rows_kv - 1) / a.rows_kv;  // items of a key tile
  const int sub = desc.row0 / per, row0 = desc.row0 % per * a.rows_kv;
  const int rows = min((off[1] - off[0]) * a.G - row0, a.rows_kv);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l32 = lane & 31, hi = lane >> 5;
  const int kg = wave % KG, rg = wave / KG;
  const int held = keys_held(p, b);
  const int64_t start = first_pos(p, b), k0 = (int64_t)desc.blk * p.block_size + sub * KT;
  const int inside = (int)max(min((int64_t)min(p.block_size - sub * KT, KT), held - k0), (int64_t)0);  // keys of the tile
  const int key = 32 * kg + l32;
  char *qt = lds, *gt = lds + NR * T::RB;

  typename O::Frag kf[D / 16], vf[D / 16];
  if (key < inside) {
    load_rows<Tag, D>(kf, a.k, b * p.k_stride[0] + hk * p.k_stride[2] + (k0 + key) * p.k_stride[1], hi, p.D);
    load_rows<Tag, D>(vf, a.v, b * p.v_stride[0] + hk * p.v_stride[2] + (k0 + key) * p.v_stride[1], hi, p.D);
  } else {
#pragma unroll
    for (int c = 0; c < D / 16; ++c) kf[c] = vf[c] = O::zero();
  }
  f32x16 dk[D / 32], dv[D / 32];

  // Rows come from all over memory, microseconds away: those of the next stage are on
  // their way while this stage's products run.  Per stage: the list's entries (a stage before),
  // where the rows lie (ids, in LDS), their values (fetch, in registers).
  constexpr int EC = 16 / O::ES, N = NR * T::CPR / 256;  // chunks of a thread
  struct Stage {
    u32x4 q[N], g[N];
    float lse, delta;
    int see;
  };
  int entry = 0;  // thread r < NR: of row r of the stage after the last one with ids
  const auto look = [&](int r0) {
    if (threadIdx.x < NR) entry = list[(row0 + min(r0 + (int)threadIdx.x, rows - 1)) / a.G];
  };
  const auto ids = [&](Stage& w, int r0) {
    if (threadIdx.x < NR) {
      const int r = threadIdx.x, q = entry >> kSlotBits, g = (row0 + min(r0 + r, rows - 1)) % a.G;
      const bool live = r0 + r < rows;
      const int h = hk * a.G + g;
      const int64_t row = ((int64_t)bh * p.Lq + q) * a.G + g;
      s_q[r] = b * p.q_stride[0] + q * p.q_stride[1] + h * p.q_stride[2];
      s_g[r] = b * p.do_stride[0] + q * p.do_stride[1] + h * p.do_stride[2];
      w.lse = a.lse[row];
      w.delta = a.delta[row];
      w.see = live ? (int)min(max((int64_t)key_limit(p, b, q, held, start) - k0, (int64_t)0), (int64_t)inside) : 0;
    }
    look(r0 + NR);
  };
  const auto fetch = [&](Stage& w, int r0) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int x = i * 256 + threadIdx.x, r = x / T::CPR, c = x % T::CPR;
      const bool live = r0 + r < rows && c * EC < p.D;
      w.q[i] = live ? *(const u32x4*)((const char*)a.q + O::ES * (s_q[r] + c * EC)) : u32x4{0u, 0u, 0u, 0u};
      w.g[i] = live ? *(const u32x4*)((const char*)a.dO + O::ES * (s_g[r] + c * EC)) : u32x4{0u, 0u, 0u, 0u};
    }
  };
  const auto stage = [&](Stage& w, int r0, auto careful) {
    // (opaque: places in LDS worked out ahead of the loop would take the registers of the operands)
    int tid = threadIdx.x;
    asm("" : "+v"(tid));
    const int lane = tid & 63, l32 = lane & 31, hi = lane >> 5, key = 32 * kg + l32;
    barrier_lds();  // the stage before is done with the tiles, all have read the ids
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int x = i * 256 + tid, r = x / T::CPR, c = x % T::CPR;
      *(u32x4*)(qt + T::at(r, c)) = w.q[i];
      *(u32x4*)(gt + T::at(r, c)) = w.g[i];
    }
    if (threadIdx.x < NR) {
      s_lse[threadIdx.x] = w.lse;
      s_delta[threadIdx.x] = w.delta;
      s_see[threadIdx.x] = w.see;
    }
    const bool more = r0 + NR < rows;
    if (more) ids(w, r0 + NR);
    barrier_lds();
    if (more) fetch(w, r0 + NR);
#pragma unroll
    for (int i32 = 0; i32 < NR / 32 / RG; ++i32) {
      const int x = rg + i32 * RG;
      if (r0 + 32 * x >= rows) continue;
      float s[16], dp[16];
      {
        f32x16 x16 = f32x16{}, y16 = f32x16{};
#pragma unroll
        for (int c = 0; c < D / 16; ++c) x16 = O::mma32(T::row(qt, 32 * x + l32, 2 * c + hi), kf[c], x16);
#pragma unroll
        for (int c = 0; c < D / 16; ++c) y16 = O::mma32(T::row(gt, 32 * x + l32, 2 * c + hi), vf[c], y16);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[i] = x16[i];
          dp[i] = y16[i];
        }
      }
      const bool part = __any(s_see[32 * x + l32] < KT);  // some row does not see all of the tile
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = 32 * x + 8 * j + 4 * hi;
        const f32x4 l = *(const f32x4*)(s_lse + r), d = *(const f32x4*)(s_delta + r);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float w = fast_exp2(__builtin_fmaf(s[4 * j + i], a.scale_log2, -l[i])), g = w * (dp[4 * j + i] - d[i]);
          s[4 * j + i] = w;
          dp[4 * j + i] = g;
        }
      }
      if (part) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u32x4 n = *(const u32x4*)(s_see + 32 * x + 8 * j + 4 * hi);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t see = key < (int)n[i] ? 0xffffffffu : 0u;
            asm("" : "+v"(see));
            s[4 * j + i] = mask_zero(s[4 * j + i], see);
            dp[4 * j + i] = mask_zero(dp[4 * j + i], see);
          }
        }
      }
      typename O::Frag pf[2], df[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float e[8], y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          e[i] = s[8 * j + i];
          y[i] = dp[8 * j + i];
        }
        pf[j] = O::pack(e);
        df[j] = O::pack(y);
      }
      const auto add = [&](f32x16(&acc)[D / 32], const char* t, const typename O::Frag(&f)[2]) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int mt = 0; mt < D / 32; ++mt) {
            auto y = T::tr32(t, 2 * x + j, mt, lane);
            if constexpr (decltype(careful)::value) y = O::finite(y);
            acc[mt] = O::mma32(y, f[j], acc[mt]);
          }
      };
      add(dv, gt, pf);
      add(dk, qt, df);
    }
  };
  const auto walk = [&](auto careful) {
#pragma unroll
    for (int mt = 0; mt < D / 32; ++mt) dk[mt] = dv[mt] = f32x16{};
    Stage ahead;
    look(0);
    ids(ahead, 0);
    __syncthreads();
    fetch(ahead, 0);
    for (int r0 = 0; r0 < rows; r0 += NR) stage(ahead, r0, careful);
  };
  walk(std::false_type{});
  // An infinite or NaN value of Q or dO spoils the keys that must not see it: the rows once
  // more with such values as 0 in these products, the rest by add_odd_rows.
  float worst = 0.f;  // NaN where some result is not finite
#pragma unroll
  for (int mt = 0; mt < D / 32; ++mt)
#pragma unroll
    for (int i = 0; i < 16; ++i) worst = __builtin_fmaf(dk[mt][i], 0.f, __builtin_fmaf(dv[mt][i], 0.f, worst));
  if (__syncthreads_or(worst != 0.f)) {
    a.kvodd[(int64_t)bh * a.nblk + desc.blk] = 1;
    walk(std::true_type{});
  }
  // the row groups of a key, through LDS (a [32 keys][D] tile of floats for each key group), then to the item
  float* out = a.kvpart + item * 2 * KT * p.D;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    f32x16(&acc)[D / 32] = w ? dv : dk;
    const float sc = w ? 1.f : p.scale;
    if constexpr (RG == 2) {
      static_assert(2 * 32 * D * 4 <= sizeof(lds));
      __syncthreads();
      float* f = (float*)lds + kg * 32 * D;
      if (rg == 1) {
#pragma unroll
        for (int mt = 0; mt < D / 32; ++mt)
#pragma unroll
          for (int i = 0; i < 16; ++i) f[(mt * 16 + i) * 64 + lane] = acc[mt][i];
      }
      __syncthreads();
      if (rg == 0) {
#pragma unroll
        for (int mt = 0; mt < D / 32; ++mt)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[mt][i] += f[(mt * 16 + i) * 64 + lane];
      }
      if (rg == 0) put_row<D>(out + ((int64_t)w * KT + key) * p.D, acc, sc, hi, p.D);
    } else {
      put_row<D>(out + ((int64_t)w * KT + key) * p.D, acc, sc, hi, p.D);
    }
  }
}

// The same for 16-bit inputs: eight waves, 64 keys, 128 rows at a time.  A wave forms P and dS
// of 32 rows and 32 keys and leaves them in LDS as the operands of the second products, of
// which each wave takes 32 columns of dV or dK: the sums of a wave are 32 registers where
// by_block_kv's are 128, so that two waves fit a SIMD and one works while the other waits.  DS:
// dS also goes to memory, rows of block_size keys in the order of the list.  Measured as whole
// steps against by_block_kv's layout in 16 bits: [1, 8192, 32/8, 128], 16 blocks of 64, 1.75 ->
// 1.68 ms; 3 of 512, 1.93 -> 1.86 ms; d = 64, 1.19 -> 1.13 ms.
template <class Tag, int D, bool DS>
__global__ __attribute__((amdgpu_flat_work_group_size(512, 512), amdgpu_waves_per_eu(2)))
void by_block_kv16(SArgs a) {
  using O = SOp<Tag>;
  using T = STile<Tag, D>;
  constexpr int NR = 128, KT = 64, MT = D / 32, NK = MT / 2;  // NK: key groups a wave sums (8 waves: 2 kinds, MT columns, 2 / NK)
  constexpr int DSB = KT * 2 + 16;  // bytes of a staged row of dS (16 more: rows start on other banks)
  __shared__ __align__(16) char lds[2 * NR * T::RB];
  __shared__ u32x4 s_k[2][D / 16][64];         // K's operands (V's are in registers): key group, step, lane
  __shared__ u32x4 s_f[2][NR / 32][2][2][64];  // P, dS: row group, key group, half, lane
  __shared__ __align__(16) char s_ds[DS ? NR * DSB : 16];
  __shared__ __align__(16) float s_lse[NR], s_delta[NR];
  __shared__ __align__(16) int s_see[NR];
  __shared__ int64_t s_q[2][NR], s_g[2][NR];
  const mattn_selected& p = a.p;
  const int bh = blockIdx.x % a.bh_n, b = bh / p.Hkv, hk = bh % p.Hkv;
  const int64_t item = (int64_t)bh * a.max_kv + blockIdx.x / a.bh_n;
  const Desc desc = a.kvtile[item];
  if (desc.blk < 0) return;
  const int* off = a.off + (int64_t)bh * (a.nblk + 1) + desc.blk;
  const int* list = a.ent + (int64_t)bh * p.Lq * p.count + off[0];
  const int per = ((off[1] - off[0]) * a.G + a.rows_kv - 1) / a.rows_kv;  // items of a key tile
  const int sub = desc.row0 / per, row0 = desc.row0 % per * a.rows_kv;
  const int rows = min((off[1] - off[0]) * a.G - row0, a.rows_kv);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l32 = lane & 31, hi = lane >> 5;
  const int held = keys_held(p, b);
  const int64_t start = first_pos(p, b), k0 = (int64_t)desc.blk * p.block_size + sub * KT;
  const int inside = (int)max(min((int64_t)min(p.block_size - sub * KT, KT), held - k0), (int64_t)0);  // keys of the tile
  const int xg = wave >> 1, kg = wave & 1, key = 32 * kg + l32;                                       // first products
  const int kind = wave >> 2, mt = wave % 4 * NK / 2, kg0 = NK == 2 ? 0 : wave & 1;                   // second ones: dV, dK
  char *qt = lds, *gt = lds + NR * T::RB;

  typename O::Frag vf[D / 16];
  {
    typename O::Frag kf[D / 16];
    if (key < inside) load_rows<Tag, D>(kf, a.k, b * p.k_stride[0] + hk * p.k_stride[2] + (k0 + key) * p.k_stride[1], hi, p.D);
    if (xg == 0) {
#pragma unroll
      for (int c = 0; c < D / 16; ++c) s_k[kg][c][lane] = key < inside ? kf[c] : O::zero();
    }
  }
  if (key < inside) {
    load_rows<Tag, D>(vf, a.v, b * p.v_stride[0] + hk * p.v_stride[2] + (k0 + key) * p.v_stride[1], hi, p.D);
  } else {
#pragma unroll
    for (int c = 0; c < D / 16; ++c) vf[c] = O::zero();
  }
  f32x16 acc[NK];

  // rows on their way, as in by_block_kv
  constexpr int N = NR * T::CPR / 512;
  u32x4 xq[N], xg_[N];
  // thread r < NR: list entry and head of row r of the stage whose places (ids) come next, what
  // goes to LDS with the next stage's values, and with those of the stage after it
  struct Side {
    float lse, delta;
    int see;
  } side{}, later{};
  int entry = 0, e_at = 0, g_at = 0, r_at = 0;
  const int last_e = (row0 + rows - 1) / a.G, step_e = NR / a.G, step_g = NR % a.G;
  const auto ids = [&](int buf) {
    if (threadIdx.x < NR) {
      const int r = threadIdx.x, q = entry >> kSlotBits, h = hk * a.G + g_at;
      const int64_t row = ((int64_t)bh * p.Lq + q) * a.G + g_at;
      s_q[buf][r] = b * p.q_stride[0] + q * p.q_stride[1] + h * p.q_stride[2];
      s_g[buf][r] = b * p.do_stride[0] + q * p.do_stride[1] + h * p.do_stride[2];
      later.lse = a.lse[row];
      later.delta = a.delta[row];
      later.see = r_at < rows ? (int)min(max((int64_t)key_limit(p, b, q, held, start) - k0, (int64_t)0), (int64_t)inside) : 0;
      r_at += NR;
      e_at += step_e;
      g_at += step_g;
      if (g_at >= a.G) {
        g_at -= a.G;
        ++e_at;
      }
      entry = list[min(e_at, last_e)];
    }
  };
  const auto fetch = [&](int r0, int buf, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int x = i * 512 + tid, r = x / T::CPR, c = x % T::CPR;
      const bool live = r0 + r < rows && c * 8 < p.D;
      xq[i] = live ? *(const u32x4*)((const char*)a.q + 2 * (s_q[buf][r] + c * 8)) : u32x4{0u, 0u, 0u, 0u};
      xg_[i] = live ? *(const u32x4*)((const char*)a.dO + 2 * (s_g[buf][r] + c * 8)) : u32x4{0u, 0u, 0u, 0u};
    }
  };
  const auto stage = [&](int r0, int buf, bool careful) {  // buf: of the next stage's ids
    // (opaque: places in LDS worked out ahead of the loop would take the registers of the operands)
    int tid = threadIdx.x;
    asm("" : "+v"(tid));
    const int lane = tid & 63, l32 = lane & 31, hi = lane >> 5, key = 32 * kg + l32;
    barrier_lds();  // the stage before is done with the tiles
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int x = i * 512 + tid, r = x / T::CPR, c = x % T::CPR;
      *(u32x4*)(qt + T::at(r, c)) = xq[i];
      *(u32x4*)(gt + T::at(r, c)) = xg_[i];
    }
    if (threadIdx.x < NR) {
      s_lse[threadIdx.x] = side.lse;
      s_delta[threadIdx.x] = side.delta;
      s_see[threadIdx.x] = side.see;
    }
    side = later;
    barrier_lds();
    if (r0 + NR < rows) fetch(r0 + NR, buf, tid);
    const int groups = min(NR / 32, (rows - r0 + 31) / 32);  // of 32 rows
    if (xg < groups) {
      float s[16], dp[16];
      {
        f32x16 x16 = f32x16{}, y16 = f32x16{};
#pragma unroll
        for (int c = 0; c < D / 16; ++c) x16 = O::mma32(T::row(qt, 32 * xg + l32, 2 * c + hi), s_k[kg][c][lane], x16);
#pragma unroll
        for (int c = 0; c < D / 16; ++c) y16 = O::mma32(T::row(gt, 32 * xg + l32, 2 * c + hi), vf[c], y16);
        reads_ahead<D / 16, 3, 2>();
        reads_ahead<D / 16, 4, 1>();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[i] = x16[i];
          dp[i] = y16[i];
        }
      }
      const bool part = __any(s_see[32 * xg + l32] < KT);  // some row does not see all of the tile
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = 32 * xg + 8 * j + 4 * hi;
        const f32x4 l = *(const f32x4*)(s_lse + r), d = *(const f32x4*)(s_delta + r);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float w = fast_exp2(__builtin_fmaf(s[4 * j + i], a.scale_log2, -l[i])), g = w * (dp[4 * j + i] - d[i]);
          s[4 * j + i] = w;
          dp[4 * j + i] = g;
        }
      }
      if (part) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u32x4 n = *(const u32x4*)(s_see + 32 * xg + 8 * j + 4 * hi);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t on = key < (int)n[i] ? 0xffffffffu : 0u;
            asm("" : "+v"(on));
            s[4 * j + i] = mask_zero(s[4 * j + i], on);
            dp[4 * j + i] = mask_zero(dp[4 * j + i], on);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float e[8], y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          e[i] = s[8 * j + i];
          y[i] = dp[8 * j + i];
        }
        const u32x4 df = O::pack(y);
        s_f[0][xg][kg][j][lane] = O::pack(e);
        s_f[1][xg][kg][j][lane] = df;
        if constexpr (DS) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *(uint16_t*)(s_ds + (32 * xg + 16 * j + 8 * (i >> 2) + 4 * hi + (i & 3)) * DSB + key * 2) = (uint16_t)elt16(df, i);
        }
      }
    }
    barrier_lds();
    if (r0 + 2 * NR < rows) ids(buf ^ 1);
    const char* t = kind ? qt : gt;
    for (int x = 0; x < groups; ++x) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        auto y = T::tr32(t, 2 * x + j, mt, lane);
        if (careful) y = O::finite(y);
#pragma unroll
        for (int n = 0; n < NK; ++n) acc[n] = O::mma32(y, s_f[kind][x][kg0 + n][j][lane], acc[n]);
      }
    }
    if constexpr (DS) {  // dS to memory, past the caches: the rows lie in them
      const int keys = min(KT, p.block_size - sub * KT) / 8;  // chunks of a row
      char* o = (char*)a.ds + 2 * ((((int64_t)bh * p.Lq * p.count + off[0]) * a.G + row0 + r0) * p.block_size + sub * KT);
#pragma unroll
      for (int i = 0; i < NR * (KT / 8) / 512; ++i) {
        const int x = i * 512 + tid, r = x / (KT / 8), c = x % (KT / 8);
        if (r0 + r < rows && c < keys) 
          __builtin_nontemporal_store(*(const u32x4*)(s_ds + r * DSB + 16 * c), (u32x4*)(o + (int64_t)r * p.block_size * 2 + 16 * c));
      }
    }
  };
  const auto walk = [&](bool careful) {
#pragma unroll
    for (int n = 0; n < NK; ++n) acc[n] = f32x16{};
    r_at = threadIdx.x;
    const int at = row0 + min((int)threadIdx.x, rows - 1);
    e_at = at / a.G;
    g_at = at % a.G;
    if (threadIdx.x < NR) entry = list[e_at];
    ids(0);
    side = later;
    if (NR < rows) ids(1);
    __syncthreads();
    fetch(0, 0, threadIdx.x);
    for (int r0 = 0, buf = 1; r0 < rows; r0 += NR, buf ^= 1) stage(r0, buf, careful);
  };
  walk(false);
  float worst = 0.f;  // NaN where some result is not finite: as in by_block_kv
#pragma unroll
  for (int n = 0; n < NK; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) worst = __builtin_fmaf(acc[n][i], 0.f, worst);
  if (__syncthreads_or(worst != 0.f)) {
    a.kvodd[(int64_t)bh * a.nblk + desc.blk] = 1;
    walk(true);
  }
  // kvpart holds dK, then dV
  float* out = a.kvpart + (item * 2 + (kind ? 0 : 1)) * KT * p.D;
  const float sc = kind ? p.scale : 1.f;
#pragma unroll
  for (int n = 0; n < NK; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = 32 * mt + 8 * j + 4 * hi;
      if (c < p.D)
        *(f32x4*)(out + (int64_t)(32 * (kg0 + n) + l32) * p.D + c) =
            f32x4{acc[n][4 * j] * sc, acc[n][4 * j + 1] * sc, acc[n][4 * j + 2] * sc, acc[n][4 * j + 3] * sc};
    }
}

// ---- joining --------------------------------------------------------------------------

// whether x holds in some lane of this lane's group of lpr
__device__ __forceinline__ bool group_any(bool x, int lpr) {
  const uint64_t m = __ballot(x);
  const int lane = threadIdx.x & 63, first = lane & ~(lpr - 1);
  return (m >> first) & (lpr == 64 ? ~0ull : (1ull << lpr) - 1);
}

// What the infinite and NaN values of a block's V (GRAD: K) give to a row's O (dQ), which
// lpr lanes hold 4 columns each: weights from the formula, the row's lse known.
template <class Tag, bool GRAD>
__device__ __forceinline__ void add_odd_keys(const SArgs& a, f32x4& o, float lse, int64_t row, int b, int hk, int h, int q, int blk,
                                          int col, int lpr) {
  const mattn_selected& p = a.p;
  const int held = keys_held(p, b), lim = key_limit(p, b, q, held, first_pos(p, b));
  const int64_t k0 = (int64_t)blk * p.block_size, k1 = min(k0 + p.block_size, (int64_t)lim);
  const auto load = [&](const void* base, int64_t at, float(&x)[4]) {
    if (col < p.D) load_v<Tag, 4>(base, at + col, x);
    else x[0] = x[1] = x[2] = x[3] = 0.f;
  };
  const auto dot = [&](const float(&x)[4], const float(&y)[4]) {
    float s = x[0] * y[0] + x[1] * y[1] + x[2] * y[2] + x[3] * y[3];
    for (int d = lpr >> 1; d; d >>= 1) s += __shfl_xor(s, d);
    return s;
  };
  float qx[4];
  load(a.q, b * p.q_stride[0] + q * p.q_stride[1] + h * p.q_stride[2], qx);
  const auto nan = [](const auto& x) { return x[0] != x[0] && x[1] != x[1] && x[2] != x[2] && x[3] != x[3]; };
  for (int64_t k = k0; k < k1; ++k) {
    if (!group_any(!nan(o), lpr)) return;  // all NaN already
    float kx[4], vx[4];
    load(a.k, b * p.k_stride[0] + k * p.k_stride[1] + hk * p.k_stride[2], kx);
    load(a.v, b * p.v_stride[0] + k * p.v_stride[1] + hk * p.v_stride[2], vx);
    const float(&x)[4] = GRAD ? kx : vx;
    bool odd[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) odd[i] = !__builtin_isfinite(x[i]);
    if (!group_any(odd[0] || odd[1] || odd[2] || odd[3], lpr)) continue;
    float w = fast_exp2(dot(qx, kx) * a.scale_log2 - lse);
    if constexpr (GRAD) {
      float gx[4];
      load(a.dO, b * p.do_stride[0] + q * p.do_stride[1] + h * p.do_stride[2], gx);
      w *= (dot(gx, vx) - a.delta[row]) * p.scale;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += odd[i] ? w * x[i] : 0.f;
  }
}

// The same of the rows of a block's list for 4 columns of a key's dK (W = 0) or dV (W = 1).
template <class Tag, int W>
__device__ __forceinline__ void add_odd_rows(const SArgs& a, float (&o)[4], int bh, int key, int blk, int col) {
  const mattn_selected& p = a.p;
  const int b = bh / p.Hkv, hk = bh % p.Hkv, held = keys_held(p, b);
  const int* off = a.off + (int64_t)bh * (a.nblk + 1) + blk;
  const int* list = a.ent + (int64_t)bh * p.Lq * p.count + off[0];
  const int64_t ka = b * p.k_stride[0] + key * p.k_stride[1] + hk * p.k_stride[2];
  const int64_t va = b * p.v_stride[0] + key * p.v_stride[1] + hk * p.v_stride[2];
  for (int r = 0; r < (off[1] - off[0]) * a.G; ++r) {
    if (o[0] != o[0] && o[1] != o[1] && o[2] != o[2] && o[3] != o[3]) return;  // all NaN already
    const RowId id = row_id(a, list, r);
    if (key >= key_limit(p, b, id.q, held, first_pos(p, b))) continue;
    const int h = hk * a.G + id.g;
    const int64_t qa = b * p.q_stride[0] + id.q * p.q_stride[1] + h * p.q_stride[2];
    const int64_t ga = b * p.do_stride[0] + id.q * p.do_stride[1] + h * p.do_stride[2];
    float x[4];
    load_v<Tag, 4>(W ? a.dO : a.q, (W ? ga : qa) + col, x);
    if (__builtin_isfinite(x[0]) && __builtin_isfinite(x[1]) && __builtin_isfinite(x[2]) && __builtin_isfinite(x[3])) continue;
    const auto dot = [&](const void* u, int64_t ua, const void* w, int64_t wa) {
      float s = 0.f;
      for (int c = 0; c < p.D; c += 4) {
        float y[4], z[4];
        load_v<Tag, 4>(u, ua + c, y);
        load_v<Tag, 4>(w, wa + c, z);
        s += y[0] * z[0] + y[1] * z[1] + y[2] * z[2] + y[3] * z[3];
      }
      return s;
    };
    const int64_t row = ((int64_t)bh * p.Lq + id.q) * a.G + id.g;
    float w = fast_exp2(dot(a.q, qa, a.k, ka) * a.scale_log2 - a.lse[row]);
    if constexpr (W == 0) w *= (dot(a.dO, ga, a.v, va) - a.delta[row]) * p.scale;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += __builtin_isfinite(x[i]) ? 0.f : w * x[i];
  }
}

// A row's partial results, 4 columns a lane: weighted by their log-sum-exp (forward), or
// added (dQ).  Slots outside the selection's valid ones hold nothing and are not read.
template <class Tag, bool GRAD>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256)))
void join_rows(SArgs a, int lpr_log2, int slots, bool all) {
  const mattn_selected& p = a.p;
  const int lpr = 1 << lpr_log2, lane = threadIdx.x & (lpr - 1), col = 4 * lane;
  const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> lpr_log2;
  if (row >= (int64_t)a.bh_n * p.Lq * a.G) return;
  const int g = (int)(row % a.G), q = (int)(row / a.G % p.Lq), bh = (int)(row / a.G / p.Lq);
  const uint32_t* ok = a.ok + ((int64_t)bh * p.Lq + q) * a.words;
  const float* part = a.part + row * slots * p.D;
  const float* plse = a.plse + row * slots;
  const auto valid = [&](int s) { return all || ((ok[s >> 5] >> (s & 31)) & 1u); };
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  float lse = GRAD ? a.lse[row] : NEG_INF, sum = 0.f, m = NEG_INF;
  // weights of the slots, lpr at a time, a lane each
  if constexpr (!GRAD) {
    bool nan = false;
    for (int s = lane; s < slots; s += lpr)
      if (valid(s)) {
        m = fmaxf(m, plse[s]);
        nan = nan || plse[s] != plse[s];
      }
    for (int d = lpr >> 1; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    if (group_any(nan, lpr)) m = __builtin_nanf("");
  }
  if (GRAD || m != NEG_INF) {
    for (int s0 = 0; s0 < slots; s0 += lpr) {
      const int s = s0 + lane;
      float w = 0.f;
      if (s < slots && valid(s)) w = GRAD ? 1.f : fast_exp2(plse[s] - m);
      sum += w;
      const int n = min(lpr, slots - s0);
      for (int i = 0; i < n; i += 8) {  // 8 rows in flight; unused slots are read, not added
        f32x4 x[8];
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          y[e] = __shfl(w, (threadIdx.x & 63 & ~(lpr - 1)) + min(i + e, lpr - 1));
          if (i + e >= n) y[e] = 0.f;
          x[e] = *(const f32x4*)(part + (int64_t)min(s0 + i + e, slots - 1) * p.D + min(col, p.D - 4));
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[c] += y[e] != 0.f ? y[e] * x[e][c] : 0.f;
      }
    }
  }
  if constexpr (!GRAD) {
    for (int d = lpr >> 1; d; d >>= 1) sum += __shfl_xor(sum, d);
    if (m != NEG_INF) {
      const float r = 1.f / sum;
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] *= r;
      lse = m + __log2f(sum);
    }
  }
  const int b = bh / p.Hkv, h = bh % p.Hkv * a.G + g;
  if (!all) {
    const int32_t* sel = p.blocks + (((int64_t)b * p.Lq + q) * p.Hkv + bh % p.Hkv) * p.count;
    bool any = false;
    for (int s = lane; s < slots; s += lpr) any = any || (valid(s) && a.odd[(int64_t)bh * a.nblk + sel[s]]);
    if (group_any(any, lpr))
      for (int s = 0; s < slots; ++s)
        if (valid(s) && a.odd[(int64_t)bh * a.nblk + sel[s]]) add_odd_keys<Tag, GRAD>(a, o, lse, row, b, bh % p.Hkv, h, q, sel[s], col, lpr);
  }
  if (col < p.D) {
    const int64_t* st = GRAD ? p.dq_stride : p.o_stride;
    const float x[4] = {o[0], o[1], o[2], o[3]};
    store_v<Tag, 4>(GRAD ? a.dq : a.o, b * st[0] + q * st[1] + h * st[2] + col, x);
    if (!GRAD && a.o32) *(f32x4*)(a.o32 + row * p.D + col) = o;
  }
  if (!GRAD && lane == 0 && a.lse) a.lse[row] = lse;
}

// delta = dO . O of each row, 4 columns a lane; no block marked yet
template <class Tag>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256)))
void row_delta(SArgs a, int lpr_log2) {
  const mattn_selected& p = a.p;
  const int lpr = 1 << lpr_log2, lane = threadIdx.x & (lpr - 1), col = 4 * lane;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)a.bh_n * a.nblk; i += (int64_t)gridDim.x * 256)
    a.odd[i] = a.kvodd[i] = 0;
  const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> lpr_log2;
  if (row >= (int64_t)a.bh_n * p.Lq * a.G) return;
  const int g = (int)(row % a.G), q = (int)(row / a.G % p.Lq), bh = (int)(row / a.G / p.Lq);
  const int b = bh / p.Hkv, h = bh % p.Hkv * a.G + g;
  float s = 0.f;
  if (col < p.D) {
    float x[4];
    load_v<Tag, 4>(a.dO, b * p.do_stride[0] + q * p.do_stride[1] + h * p.do_stride[2] + col, x);
    const f32x4 o = *(const f32x4*)(a.o32 + row * p.D + col);
#pragma unroll
    for (int i = 0; i < 4; ++i) s += x[i] * o[i];
  }
  for (int o = lpr >> 1; o; o >>= 1) s += __shfl_xor(s, o);
  if (lane == 0) a.delta[row] = s;
}

// dK and dV of each key: the items of its block in order, 4 columns a thread; zeros for keys no query saw.
template <class Tag>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256)))
void join_keys(SArgs a, int KT) {
  const mattn_selected& p = a.p;
  const int cpr = p.D / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int col = 4 * (int)(i % cpr);
  const int64_t kk = i / cpr;
  if (kk >= p.Lk) return;
  const int key = (int)kk, w = blockIdx.y & 1, bh = blockIdx.y >> 1, b = bh / p.Hkv, hk = bh % p.Hkv;
  const int blk = key / p.block_size, in = key % p.block_size, sub = in / KT;
  const int* kvoff = a.kvoff + (int64_t)bh * (a.nblk + 1) + blk;
  const int per = (kvoff[1] - kvoff[0]) / a.subs;
  const float* part = a.kvpart + (((int64_t)bh * a.max_kv + kvoff[0] + sub * per) * 2 + w) * KT * p.D + (int64_t)(in % KT) * p.D + col;
  float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int x = 0; x < per; ++x) {
    const f32x4 v = *(const f32x4*)(part + (int64_t)x * 2 * KT * p.D);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += v[e];
  }
  if (a.kvodd[(int64_t)bh * a.nblk + blk]) {
    if (w) add_odd_rows<Tag, 1>(a, o, bh, key, blk, col);
    else add_odd_rows<Tag, 0>(a, o, bh, key, blk, col);
  }
  const int64_t* st = w ? p.dv_stride : p.dk_stride;
  store_v<Tag, 4>(w ? a.dv : a.dk, b * st[0] + kk * st[1] + hk * st[2] + col, o);
}

// ---- by tiles of queries --------------------------------------------------------------

// Forward without partial rows: a wave holds 32 rows (32 / G neighbouring queries of a
// key head with all their heads), a workgroup four such; it walks the blocks that any of its
// queries selected, each row masked to its own.  The union grows with the queries of a tile,
// but no faster than their selections together, and each block costs products (and one read
// of K and V from the cache) where the form by blocks costs 8 D bytes of memory a row.  K and
// V of the next tile are loaded while this tile's products run.
//
// A negative or zero scale is folded into Q.  A row that did not select a block gets weights 0
// (attend_tile); where infinite or NaN values make that NaN, or spoil a product (0 times them),
// the result is not finite, and the workgroup walks its blocks once more with every element
// masked and such values as 0 (add_odd_keys then gives them to the rows that see them).
//
// GRAD: dQ = scale dS K the same way, from the dS that the dK/dV kernel has left in memory:
// 2 bytes a pair, where a partial row of dQ takes 8 D for each row and block.
//
// Per wave and tile of 64 keys at D = 128: 1024 (dQ: 512) cycles of matrix products, 1280 of
// LDS traffic a workgroup, some 850 of vector instructions (32 exponentials of 16 cycles).
constexpr int kSpan = 512;  // blocks whose selections lie in LDS at a time
template <class Tag, int D, bool GRAD>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256), amdgpu_waves_per_eu(SOp<Tag>::ES == 2 ? 2 : 1)))
void by_tile(SArgs a, int hgroups, int tiles_q) {
  using O = SOp<Tag>;
  using T = STile<Tag, D>;
  constexpr int NBUF = SOp<Tag>::ES == 2 ? 2 : 1;  // K and V tiles in LDS
  __shared__ __align__(16) char lds[NBUF][(GRAD ? 1 : 2) * kKT * T::RB];
  __shared__ uint32_t s_sel[kSpan][4];  // block, wave: the wave's queries that selected it
  constexpr int kPos = 8192;
  __shared__ int s_pos[GRAD ? kPos : 1];  // GRAD: block, query: where the query's dS of the block lies
  __shared__ int s_list[kSpan], s_n, s_odd[2];
  const mattn_selected& p = a.p;
  int x = blockIdx.x;
  const int bh = x % a.bh_n, b = bh / p.Hkv, hk = bh % p.Hkv;
  x /= a.bh_n;
  const int h0 = 32 * (x % hgroups), G = min(a.G - h0, 32), R = 32 / min(a.G, 32);  // heads, queries of a wave
  const int q0 = (tiles_q - 1 - x / hgroups) * 4 * R;                              // late queries see most: first
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l32 = lane & 31, hi = lane >> 5;
  const int held = keys_held(p, b);
  const int64_t start = first_pos(p, b);
  const int qi = l32 / G, q = q0 + wave * R + qi, h = hk * a.G + h0 + l32 % G;
  const bool live = qi < R && q < p.Lq;
  const int qc = live ? q : p.Lq - 1;
  const int64_t row = ((int64_t)bh * p.Lq + qc) * a.G + h0 + l32 % G;
  const int lim = live ? key_limit(p, b, qc, held, start) : 0;
  const bool zero = p.scale == 0.f;
  const float sl = zero ? 1.f : fabsf(a.scale_log2);
  typename O::Frag qf[GRAD ? 1 : D / 16];
  if constexpr (!GRAD) {
    load_rows<Tag, D>(qf, a.q, b * p.q_stride[0] + qc * p.q_stride[1] + h * p.q_stride[2], hi, p.D);
#pragma unroll
    for (int c = 0; c < D / 16; ++c) qf[c] = O::sign(qf[c], p.scale < 0.f, zero);
  }
  float lse = GRAD ? a.lse[row] : 0.f;
  const char* kb = (const char*)a.k + O::ES * (b * p.k_stride[0] + hk * p.k_stride[2]);
  const char* vb = (const char*)a.v + O::ES * (b * p.v_stride[0] + hk * p.v_stride[2]);
  // K and V of a tile, as buffers that end behind its last key: this thread's chunks lie at
  // fixed offsets (past the end where the head is narrower than D), what is past the end is 0
  constexpr int EC = 16 / O::ES, N = kKT * T::CPR / 256, RPI = 256 / T::CPR;
  const int my_r = threadIdx.x / T::CPR, my_c = threadIdx.x % T::CPR;
  const bool in_d = my_c * EC < p.D;
  const int ksb = (int)p.k_stride[1] * O::ES, vsb = (int)p.v_stride[1] * O::ES;  // bytes of a row
  const uint32_t k_at = in_d ? my_r * ksb + 16 * my_c : 0x80000000u, v_at = in_d ? my_r * vsb + 16 * my_c : 0x80000000u;
  u32x4 xk[N], xv[GRAD ? 1 : N];
  typename O::Frag xs[GRAD ? kKT / 16 : 1], cs[GRAD ? kKT / 16 : 1];  // GRAD: dS of the tile in flight, of this one
  int64_t key0 = 0;  // first key of the tile in flight, and its keys
  int key_n = 0;
  int ds_at = -1, ds_key = 0;
  const auto fetch = [&]() {
    const auto kr = make_rsrc(kb + key0 * ksb, (uint32_t)((key_n - 1) * ksb + p.D * O::ES));
#pragma unroll
    for (int i = 0; i < N; ++i)
      xk[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(kr, (int)k_at, i * RPI * ksb, 0));
    if constexpr (!GRAD) {
      const auto vr = make_rsrc(vb + key0 * vsb, (uint32_t)((key_n - 1) * vsb + p.D * O::ES));
#pragma unroll
      for (int i = 0; i < N; ++i)
        xv[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(vr, (int)v_at, i * RPI * vsb, 0));
    } else {
      const char* d = (const char*)a.ds + O::ES * ((((int64_t)bh * p.Lq * p.count + ds_at) * a.G + h0 + l32 % G) * p.block_size + ds_key);
#pragma unroll
      for (int i = 0; i < kKT / 16; ++i)
        xs[i] = ds_at >= 0 && ds_key + 16 * i < p.block_size ? O::load(d + O::ES * (16 * i + 8 * hi)) : O::zero();
    }
  };
  if (threadIdx.x < 2) s_odd[threadIdx.x] = 0;
  const int last = key_limit(p, b, min(q0 + 4 * R, p.Lq) - 1, held, start);
  const int blocks = (last + p.block_size - 1) / p.block_size;
  f32x16 acc[D / 32];
  float m, sum;
  int seq = 0;
  bool careful = false, spoilt = false;  // spoilt: some tile held an infinite or NaN value
  for (;; careful = true) {
#pragma unroll
    for (int mt = 0; mt < D / 32; ++mt) acc[mt] = f32x16{};
    m = NEG_INF, sum = 0.f;
    const int full = GRAD ? min(kSpan, kPos / (4 * R)) : kSpan;
    for (int lo = 0; lo < blocks; lo += full) {
      const int span = min(full, blocks - lo);
      __syncthreads();
      for (int i = threadIdx.x; i < span * 4; i += 256) (&s_sel[0][0])[i] = 0u;
      if constexpr (GRAD)
        for (int i = threadIdx.x; i < span * 4 * R; i += 256) s_pos[i] = -1;
      __syncthreads();
      for (int i = threadIdx.x; i < 4 * R * p.count; i += 256) {
        const int t = i / p.count, qq = q0 + t;
        if (qq >= p.Lq) break;
        const int c = i % p.count, j = p.blocks[(((int64_t)b * p.Lq + qq) * p.Hkv + hk) * p.count + c] - lo;
        if (j >= 0 && j < span && (int64_t)(j + lo) * p.block_size < key_limit(p, b, qq, held, start)) {
          if constexpr (GRAD) {  // (of a repeated block the slot that counts)
            if (!((a.ok[((int64_t)bh * p.Lq + qq) * a.words + (c >> 5)] >> (c & 31)) & 1u)) continue;
            s_pos[j * 4 * R + t] = a.pos[((int64_t)bh * p.Lq + qq) * p.count + c];
          }
          atomicOr(&s_sel[j][t / R], 1u << (t % R));
        }
      }
      __syncthreads();
      if (wave == 0) {
        int n = 0;
        for (int j = 0; j < span; j += 64) {
          const bool any = j + lane < span && (s_sel[j + lane][0] | s_sel[j + lane][1] | s_sel[j + lane][2] | s_sel[j + lane][3]);
          const uint64_t bm = __ballot(any);
          if (any) s_list[n + __builtin_popcountll(bm & ((1ull << lane) - 1))] = j + lane;
          n += __builtin_popcountll(bm);
        }
        if (lane == 0) s_n = n;
      }
      __syncthreads();
      const int n = __builtin_amdgcn_readfirstlane(s_n);
      if (n == 0) continue;
      int e = 0, t = 0;  // tile in flight: entry, tile of its block
      bool further = false;  // the block has a tile behind it
      uint32_t bits = 0u;    // the wave's queries that selected the block
      const auto place = [&]() {
        const int j = __builtin_amdgcn_readfirstlane(s_list[e]);
        bits = __builtin_amdgcn_readfirstlane(s_sel[j][wave]);
        const int64_t k0 = (int64_t)(lo + j) * p.block_size;
        const int inside = (int)min((int64_t)p.block_size, held - k0);
        key0 = k0 + t * kKT;
        key_n = min(inside - t * kKT, kKT);
        further = t * kKT + kKT < inside;
        if constexpr (GRAD) {
          ds_at = live ? s_pos[j * 4 * R + wave * R + qi] : -1;
          ds_key = t * kKT;
        }
      };
      const auto put = [&](char* kt) {  // the tile in flight to LDS
        ++seq;
        char* vt = kt + kKT * T::RB;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int r = i * RPI + my_r;
          u32x4 last = GRAD ? xk[i] : xv[GRAD ? 0 : i];
          if (careful && O::odd(last)) {
            s_odd[seq & 1] = seq;  // (the other place may still be read for the tile before)
            last = O::finite16(last);
          }
          if constexpr (!GRAD) *(u32x4*)(kt + T::at(r, my_c)) = xk[i];
          *(u32x4*)((GRAD ? kt : vt) + T::at(r, my_c)) = last;
        }
        if constexpr (GRAD) {
#pragma unroll
          for (int i = 0; i < kKT / 16; ++i) cs[i] = xs[i];
        }
      };
      place();
      fetch();
      put(lds[0]);
      barrier_lds();
      int buf = 0;
      while (e < n) {
        const char *kt = lds[buf], *vt = kt + kKT * T::RB;
        const int see = live && ((bits >> qi) & 1u) ? (int)min((int64_t)key_n, lim - key0) : 0;
        spoilt = spoilt || (careful && s_odd[seq & 1] == seq);
        if (further) {
          ++t;
        } else {
          ++e;
          t = 0;
        }
        if (e < n) {
          place();
          fetch();
        }
        if (__any(see > 0)) {
          if constexpr (!GRAD) {
            const bool slow = careful || __any(see > 0 && see < kKT);  // some row sees a part of the tile
            attend_tile<Tag, D>(kt, vt, qf, see, slow, sl, lane, m, sum, acc);
          } else {
#pragma unroll
            for (int i = 0; i < kKT / 16; ++i)
#pragma unroll
              for (int mt = 0; mt < D / 32; ++mt) acc[mt] = O::mma32(T::tr32n(kt, i, mt, lane), cs[i], acc[mt]);
            if constexpr (O::ES == 2) reads_ahead<kKT / 16 * D / 32, 6, 2>();
          }
        }
        if constexpr (NBUF == 2) buf ^= 1;
        else barrier_lds();  // all are done with the one buffer
        if (e < n) put(lds[buf]);
        barrier_lds();
      }
    }
    if (careful) break;
    float worst = 0.f;  // NaN where some result is not finite
#pragma unroll
    for (int mt = 0; mt < D / 32; ++mt)
#pragma unroll
      for (int i = 0; i < 16; ++i) worst = __builtin_fmaf(acc[mt][i], 0.f, worst);
    if (!__syncthreads_or(live && worst != 0.f)) break;
  }

  const int64_t* os = GRAD ? p.dq_stride : p.o_stride;
  char* out = (char*)(GRAD ? a.dq : a.o);
  float r = p.scale;
  if constexpr (!GRAD) {
    sum = wave_sum32(sum);
    r = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    lse = sum > 0.f || sum != sum ? __builtin_fmaf(m, sl, __log2f(sum)) : NEG_INF;
  }
  if (live) {
    const int64_t at = b * os[0] + qc * os[1] + h * os[2];
#pragma unroll
    for (int mt = 0; mt < D / 32; ++mt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = 32 * mt + 8 * j + 4 * hi;
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = acc[mt][4 * j + i] * r;
        if (c < p.D) {
          store_v<Tag, 4>(out, at + c, y);
          if (!GRAD && a.o32) *(f32x4*)(a.o32 + row * p.D + c) = f32x4{y[0], y[1], y[2], y[3]};
        }
      }
    if (!GRAD && a.lse && hi == 0) a.lse[row] = lse;
  }
  if (!spoilt) return;
  // what the infinite and NaN values give to the rows that see them
  float* s_lse = (float*)lds[0];
  __syncthreads();
  if (live && hi == 0) s_lse[32 * wave + l32] = lse;
  __syncthreads();
  int lpr = 2;
  while (4 * lpr < p.D) lpr *= 2;
  const int col = 4 * (threadIdx.x & (lpr - 1));
  for (int y = threadIdx.x / lpr; y < 128; y += 256 / lpr) {
    const int wi = y >> 5, ri = y & 31, yq = q0 + wi * R + ri / G, yg = h0 + ri % G;
    if (ri / G >= R || yq >= p.Lq) continue;
    const int64_t yrow = ((int64_t)bh * p.Lq + yq) * a.G + yg, at = b * os[0] + yq * os[1] + (int64_t)(hk * a.G + yg) * os[2] + col;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int c = 0; c < p.count; ++c) {
      const int j = p.blocks[(((int64_t)b * p.Lq + yq) * p.Hkv + hk) * p.count + c];
      if (j >= 0 && j < a.nblk) add_odd_keys<Tag, GRAD>(a, o, s_lse[y], yrow, b, hk, hk * a.G + yg, yq, j, col, lpr);
    }
    if (col < p.D && (o[0] != 0.f || o[1] != 0.f || o[2] != 0.f || o[3] != 0.f)) {
      float z[4];
      load_v<Tag, 4>(out, at, z);
#pragma unroll
      for (int i = 0; i < 4; ++i) z[i] += o[i];
      store_v<Tag, 4>(out, at, z);
      if (!GRAD && a.o32) {
        f32x4 w = *(const f32x4*)(a.o32 + yrow * p.D + col);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] += o[i];
        *(f32x4*)(a.o32 + yrow * p.D + col) = w;
      }
    }
  }
}

// ---- by queries -----------------------------------------------------------------------

// One query, key head, 16 of its query heads and a part of its keys: the workgroup's four
// waves take tiles of 32 keys in turn.  Keys go straight from memory to operands (16 rows
// of 64 bytes a load), values through LDS for the transposed reads.  All rows of a tile
// see the same keys, so values past them are set to zero.  Bound by HBM.
// LDS written by the wave's lanes is read by its other lanes after this
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <class Tag, int D>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256)))
void by_query(SArgs a, int splits, int hgroups) {
  using O = SOp<Tag>;
  using T = STile<Tag, D>;
  constexpr int VB = 32 * T::RB, JB = 16 * D * 4;  // a wave's values; its heads' sums
  __shared__ __align__(16) char lds[4 * (VB > JB ? VB : JB)];
  __shared__ int list[kMaxSel];
  __shared__ int n_list;
  __shared__ float s_m[4][16], s_l[4][16], s_e[4][16];
  const mattn_selected& p = a.p;
  int x = blockIdx.x;
  const int split = x % splits;
  x /= splits;
  const int hg = x % hgroups;
  x /= hgroups;
  const int bh = x % a.bh_n, q = x / a.bh_n, b = bh / p.Hkv, hk = bh % p.Hkv;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int held = keys_held(p, b);
  const int lim = key_limit(p, b, q, held, first_pos(p, b));
  const int seen = (lim + p.block_size - 1) / p.block_size;
  const int32_t* sel = p.blocks + (((int64_t)b * p.Lq + q) * p.Hkv + hk) * p.count;
  if (wave == 0) {  // the valid blocks, in their order; repeated ones left out
    int n = 0;
    bool rising = true;
    for (int c = 0; c < p.count; c += 64) {
      const int j = c + lane < p.count ? sel[c + lane] : -1;
      const bool good = j >= 0 && j < seen;
      const uint64_t m = __ballot(good);
      const int at = n + __builtin_popcountll(m & ((1ull << lane) - 1));
      if (good) list[at] = j;
      n += __builtin_popcountll(m);
    }
    wave_sync();
    for (int c = 0; c < n; c += 64) {
      const int j = c + lane < n ? list[c + lane] : 0x7fffffff;
      const int before = c + lane == 0 ? -1 : c + lane < n ? list[c + lane - 1] : -1;
      if (!__all(j > before)) rising = false;
    }
    if (!rising) {  // compact what occurs for the first time
      int kept = 0;
      for (int c = 0; c < n; ++c) {
        const int j = list[c];
        bool dup = false;
        for (int i = lane; i < kept; i += 64) dup = dup || list[i] == j;
        if (!__any(dup)) {
          if (lane == 0) list[kept] = j;
          ++kept;
        }
        wave_sync();
      }
      n = kept;
    }
    if (lane == 0) n_list = n;
  }
  const int h0 = 16 * hg, nh = min(16, a.G - h0);
  typename O::Frag qf[D / 32];
  {
    const int64_t at = b * p.q_stride[0] + q * p.q_stride[1] + (int64_t)(hk * a.G + h0 + min(l16, nh - 1)) * p.q_stride[2];
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      const int c = 32 * s + 8 * g;
      qf[s] = c < p.D ? O::load((const char*)a.q + O::ES * (at + c)) : O::zero();
    }
  }
  __syncthreads();
  const int bs = p.block_size, nk = n_list * bs;  // keys in the list's order
  const int tiles = (nk + 31) / 32, per = (tiles + splits - 1) / splits;
  const int t1 = min((split + 1) * per, tiles);
  const char* kb = (const char*)a.k + O::ES * (b * p.k_stride[0] + hk * p.k_stride[2]);
  const char* vb = (const char*)a.v + O::ES * (b * p.v_stride[0] + hk * p.v_stride[2]);
  char* vt = lds + wave * VB;
  f32x4 acc[D / 16];
#pragma unroll
  for (int d = 0; d < D / 16; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = NEG_INF, sum = 0.f, exact = 0.f;
  for (int t = split * per + wave; t < t1; t += 4) {
    // key of each of the tile's 32 places (lane % 32), -1 where there is none
    const int at = 32 * t + (lane & 31);
    const int j = at < nk ? list[at / bs] : 0;
    const int kl = at < nk && j * (int64_t)bs + at % bs < lim ? j * bs + at % bs : -1;
    typename O::Frag kf[2][D / 32];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int key = __shfl(kl, 16 * u + l16);
#pragma unroll
      for (int s = 0; s < D / 32; ++s) {
        const int c = 32 * s + 8 * g;
        kf[u][s] = key >= 0 && c < p.D ? O::load(kb + O::ES * (key * p.k_stride[1] + c)) : O::zero();
      }
    }
    constexpr int EC = 16 / O::ES;
    u32x4 vx[VB / 1024];
#pragma unroll
    for (int i = 0; i < VB / 1024; ++i) {
      const int y = 64 * i + lane, key = __shfl(kl, y / T::CPR), c = y % T::CPR;
      vx[i] = key >= 0 && c * EC < p.D ? *(const u32x4*)(vb + O::ES * (key * p.v_stride[1]) + 16 * c) : u32x4{0u, 0u, 0u, 0u};
    }
    f32x4 s2[2];
    float top = NEG_INF;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      s2[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < D / 32; ++s) s2[u] = O::mma16(kf[u][s], qf[s], s2[u]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = __shfl(kl, 16 * u + 4 * g + i);
        s2[u][i] = key >= 0 ? s2[u][i] * a.scale_log2 : NEG_INF;
        top = fmaxf(top, s2[u][i]);
      }
    }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(m, fmaxf(top, __shfl_xor(top, 32)));
    const float ref = top == NEG_INF ? 0.f : top, keep = fast_exp2(m - ref);
    m = top;
    sum *= keep;
    exact *= keep;
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[d][i] *= keep;
    float e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      e[i] = fast_exp2(s2[i >> 2][i & 3] - ref);
      exact += e[i];
    }
    const typename O::Frag pf = O::pack(e);
    if constexpr (O::ES == 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += Elt<std::conditional_t<O::ES == 2, Tag, bf16_tag>>::to_f32(elt16(__builtin_bit_cast(u32x4, pf), i));
    }
#pragma unroll
    for (int i = 0; i < VB / 1024; ++i) {
      const int y = 64 * i + lane;
      *(u32x4*)(vt + T::at(y / T::CPR, y % T::CPR)) = vx[i];
    }
    wave_sync();
#pragma unroll
    for (int d = 0; d < D / 16; ++d) acc[d] = O::mma16(T::tr16(vt, d, lane), pf, acc[d]);
    wave_sync();
  }
  exact += __shfl_xor(exact, 16);
  exact += __shfl_xor(exact, 32);
  if constexpr (O::ES == 2) {
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
  } else {
    sum = exact;
  }
  // the waves' results: [column][head] sums of each in LDS
  __syncthreads();
  float* f = (float*)lds + wave * 16 * D;
#pragma unroll
  for (int d = 0; d < D / 16; ++d) *(f32x4*)(f + l16 * D + 16 * d + 4 * g) = acc[d];
  if (g == 0) {
    s_m[wave][l16] = m;
    s_l[wave][l16] = sum;
    s_e[wave][l16] = exact;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nh * (D / 4); i += 256) {
    const int h = i / (D / 4), c = 4 * (i % (D / 4));
    float top = fmaxf(fmaxf(s_m[0][h], s_m[1][h]), fmaxf(s_m[2][h], s_m[3][h]));
    const float ref = top == NEG_INF ? 0.f : top;
    float o[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f, ex = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float y = fast_exp2(s_m[w][h] - ref);
      l += y * s_l[w][h];
      ex += y * s_e[w][h];
      const f32x4 v = *(const f32x4*)((float*)lds + (w * 16 + h) * D + c);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += y * v[e];
    }
    const float r = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= r;
    if (c >= p.D) continue;
    const int64_t row = ((int64_t)bh * p.Lq + q) * a.G + h0 + h;
    const float lse = ex > 0.f || ex != ex ? ref + __log2f(ex) : NEG_INF;
    if (splits > 1) {
      *(f32x4*)(a.part + (row * splits + split) * p.D + c) = f32x4{o[0], o[1], o[2], o[3]};
      if (c == 0) a.plse[row * splits + split] = lse;
    } else {
      store_v<Tag, 4>(a.o, b * p.o_stride[0] + q * p.o_stride[1] + (int64_t)(hk * a.G + h0 + h) * p.o_stride[2] + c, o);
      if (a.o32) *(f32x4*)(a.o32 + row * p.D + c) = f32x4{o[0], o[1], o[2], o[3]};
      if (c == 0 && a.lse) a.lse[row] = lse;
    }
  }
}

// ---- host -----------------------------------------------------------------------------

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }
int key_tile(const mattn_selected* p) { return p->block_size >= 128 && p->dtype == MATTN_F32 ? 128 : 64; }

int sel_check(const mattn_selected* p) {
  if (!p) return MATTN_ERR_NULL;
  if (p->B <= 0 || p->Lq <= 0 || p->Lk <= 0 || p->Hq <= 0 || p->Hkv <= 0 || p->Hq % p->Hkv) return MATTN_ERR_SHAPE;
  if (p->D <= 0 || p->D > 128 || p->D % 8) return MATTN_ERR_HEAD_DIM;
  if (p->block_size <= 0 || p->block_size % 16 || p->count <= 0 || p->count > kMaxSel) return MATTN_ERR_SHAPE;
  if (p->dtype != MATTN_BF16 && p->dtype != MATTN_F16 && p->dtype != MATTN_F32) return MATTN_ERR_DTYPE;
  if (!isfinite(p->scale * 1.4426950408889634f)) return MATTN_ERR_SHAPE;
  if (!p->blocks) return MATTN_ERR_NULL;
  const int es = p->dtype == MATTN_F32 ? 4 : 2;
  for (const int64_t* s : {p->q_stride, p->k_stride, p->v_stride, p->o_stride, p->do_stride, p->dq_stride, p->dk_stride, p->dv_stride})
    for (int i = 0; i < 3; ++i)
      if (s[i] < 0 || (s[i] * es) % 16) return MATTN_ERR_STRIDE;
  const int64_t lim = 1ll << 31, bh = (int64_t)p->B * p->Hkv, G = p->Hq / p->Hkv;
  if (p->Lk + (int64_t)p->block_size >= lim || p->Lq >= lim >> kSlotBits || (int64_t)p->Lq * p->count * G >= lim || bh > 32767 || bh * p->Lq * G >= lim / 64)
    return MATTN_ERR_TOO_LARGE;
  return MATTN_OK;
}

struct SPlan {
  bool by_query, tile_fwd, tile_bwd;
  int splits, hgroups;
};

// Which form serves the forward, and its splits.
SPlan sel_plan(const mattn_selected* p) {
  const int64_t G = p->Hq / p->Hkv, bh = (int64_t)p->B * p->Hkv;
  SPlan s;
  s.hgroups = (int)cdiv(G, 16);
  const int64_t wgs = bh * p->Lq * s.hgroups, tiles = cdiv((int64_t)p->count * p->block_size, 32);
  s.by_query = p->Lq <= 16;
  // By tiles or by blocks, by their times in ns.  A wave's tile holds R queries; where their
  // selections are independent its union has U = v (1 - (1 - n / v)^R) of the v blocks they see
  // on average, E of all blocks (neighbouring queries share more, which favours tiles).  Measured
  // at D = 128 in 16 bits: by tiles 1.4 a wave and 64 keys (dQ 1.0, and 0.03 a row for writing
  // dS), but no less than a workgroup's walk of E blocks alone takes, 1900 (dQ 1400) for each
  // 64 keys; by blocks 0.28 + 0.05 a row and 64 keys (dQ 0.26 + 0.11), and some 25 us (dQ 10)
  // of lists, joining and launches.  At D = 64 0.6 (dQ 0.7) of all that.  Float32 takes 11 and
  // 0.64; its dQ goes by blocks.  Forward by tiles and by blocks, then both with their gradients:
  // [1, 8192, 32/8, 128], 16 blocks of 64: 0.62 and 1.38 ms, 1.76 and 3.66; [1, 6000, 1, 64], 16 of
  // 64: 116 and 73 us, 291 and 133; [1, 8192, 2, 128], 4 of 64: 200 and 74 us; [1, 300, 8/2, 128],
  // 4 of 64: 21 and 37 us; float32 [1, 1000, 4/1, 128], 9 of 64: 153 and 62 us.
  const bool f32 = p->dtype == MATTN_F32, narrow = p->D <= 64;
  const double R = G < 32 ? 32 / G : 1, T = (double)cdiv(p->block_size, 64), n = p->count;
  const double blocks = fmax(n, (double)cdiv(p->Lk, p->block_size)), v = fmax(n, p->causal && !p->starts ? 0.5 * blocks : blocks);
  const double U = v * (1.0 - pow(1.0 - n / v, R)), E = blocks * (1.0 - pow(1.0 - n / blocks, R));
  const double rows = (double)bh * p->Lq * G, waves = (double)bh * cdiv(G, 32) * p->Lq / R;
  const double c = narrow ? 0.6 : 1.0, cb = narrow ? 0.7 : 1.0;
  const bool tile_fwd = fmax((f32 ? 11.0 : 1.4) * waves * U, (f32 ? 9000.0 : 1900.0) * E) * T * c <
                        25000.0 + rows * n * (0.28 + (f32 ? 0.64 : 0.05) * T) * c;
  const bool tile_bwd = fmax(waves * U, 1400.0 * E) * T * cb + 0.03 * rows * n * T < 10000.0 + rows * n * (0.26 + 0.11 * T) * cb;
  const int es = f32 ? 4 : 2;
  // (a tile's keys are read through buffers with 32-bit offsets)
  const bool fits = p->k_stride[1] < (1 << 30) / (64 * es) && p->v_stride[1] < (1 << 30) / (64 * es);
  s.tile_fwd = !s.by_query && fits && tile_fwd;
  // (dS takes 2 block_size bytes a row and block in memory, partial rows 4 D: wide blocks keep to those)
  s.tile_bwd = fits && !f32 && p->block_size <= kMaxDS && tile_bwd;
  s.splits = 1;
  while (s.splits < 32 && wgs * s.splits < 512 && tiles / (2 * s.splits) >= 4) s.splits *= 2;
  return s;
}

struct SLayout {
  // lists: kept for the backward
  size_t ok, off, kvoff, ent, pos, tile, kvtile, lists;
  // workspace
  size_t cnt, odd, part, plse, fwd;                   // forward
  size_t delta, dqpart, ds, kvpart, bodd, kvodd, bwd;  // backward
  int words, chunks, nblk, max_tiles, max_kv, subs, rows_q, rows_kv;
};

SLayout sel_layout(const mattn_selected* p) {
  SLayout l{};
  const int64_t bh = (int64_t)p->B * p->Hkv, G = p->Hq / p->Hkv, rows = bh * p->Lq * G;
  l.nblk = (int)cdiv(p->Lk, p->block_size);
  l.words = (p->count + 31) / 32;
  l.chunks = (int)cdiv(p->Lq, kChunkQ);
  l.subs = (int)cdiv(p->block_size, key_tile(p));
  const int64_t most = (int64_t)p->Lq * p->count;  // entries of a head
  const int64_t used = l.nblk < most ? l.nblk : most;
  // fewer rows an item where there would be too few items for the card: at [1, 543, 8, 96] in
  // float32 over 3 blocks of 256 the step takes 0.28 ms against 0.9
  const auto share = [&](int64_t of, int64_t unit, int64_t most) {
    const int64_t x = cdiv(cdiv(of, 1024), unit) * unit;
    return (int)(x < most ? x : most);
  };
  l.rows_q = share(bh * most * G, 128, kRows);
  l.rows_kv = share(bh * most * G * l.subs, 256, kRowsKV);
  l.max_tiles = (int)(most * G / l.rows_q + used);
  l.max_kv = (int)((most * G / l.rows_kv + used) * l.subs);
  size_t x = 0;
  const auto take = [&](size_t bytes) {
    const size_t at = x;
    x += align256(bytes);
    return at;
  };
  l.ok = take(bh * p->Lq * l.words * 4);
  l.off = take(bh * (l.nblk + 1) * 4);
  l.kvoff = take(bh * (l.nblk + 1) * 4);
  l.ent = take(bh * most * 4);
  l.pos = take(bh * most * 4);
  l.tile = take(bh * l.max_tiles * sizeof(Desc));
  l.kvtile = take(bh * l.max_kv * sizeof(Desc));
  l.lists = x;
  x = 0;
  const SPlan s = sel_plan(p);
  const int64_t slots = s.by_query ? (s.splits > 1 ? s.splits : 0) : s.tile_fwd ? 0 : p->count;
  l.cnt = take(bh * l.nblk * l.chunks * 4);
  l.odd = take(bh * l.nblk * 4);
  l.part = take(rows * slots * p->D * 4);
  l.plse = take(rows * slots * 4);
  l.fwd = x;
  x = 0;
  l.delta = take(rows * 4);
  if (s.tile_bwd) l.ds = take(rows * p->count * p->block_size * (p->dtype == MATTN_F32 ? 4 : 2));
  else l.dqpart = take(rows * p->count * p->D * 4);
  l.kvpart = take(bh * l.max_kv * 2 * key_tile(p) * p->D * 4);
  l.bodd = take(bh * l.nblk * 4);
  l.kvodd = take(bh * l.nblk * 4);
  l.bwd = x;
  return l;
}

SArgs sel_args(const mattn_selected* p, const SLayout& l, void* lists) {
  SArgs a{};
  a.p = *p;
  a.G = p->Hq / p->Hkv;
  a.nblk = l.nblk;
  a.bh_n = p->B * p->Hkv;
  a.scale_log2 = p->scale * 1.4426950408889634f;
  a.words = l.words;
  a.chunks = l.chunks;
  a.max_tiles = l.max_tiles;
  a.max_kv = l.max_kv;
  a.subs = l.subs;
  a.rows_q = l.rows_q;
  a.rows_kv = l.rows_kv;
  char* c = (char*)lists;
  if (c) {
    a.ok = (uint32_t*)(c + l.ok);
    a.off = (int*)(c + l.off);
    a.kvoff = (int*)(c + l.kvoff);
    a.ent = (int*)(c + l.ent);
    a.pos = (int*)(c + l.pos);
    a.tile = (Desc*)(c + l.tile);
    a.kvtile = (Desc*)(c + l.kvtile);
  }
  return a;
}

void make_lists(const SArgs& a, hipStream_t st) {
  const dim3 grid(a.chunks, (uint32_t)cdiv(a.nblk, kRange), a.bh_n);
  if (grid.y > 1) {
    const int64_t n = (int64_t)a.bh_n * a.p.Lq * a.words;
    hipLaunchKernelGGL(list_clear, dim3((uint32_t)(cdiv(n, 256) < 1024 ? cdiv(n, 256) : 1024)), dim3(256), 0, st, a.ok, n);
  }
  hipLaunchKernelGGL((list_entries<false>), grid, dim3(kChunkQ), 0, st, a);
  hipLaunchKernelGGL(list_chunks, dim3((uint32_t)cdiv((int64_t)a.bh_n * a.nblk, 4)), dim3(256), 0, st, a);
  hipLaunchKernelGGL(list_items, dim3(a.bh_n), dim3(kScan), 0, st, a);
  hipLaunchKernelGGL((list_entries<true>), grid, dim3(kChunkQ), 0, st, a);
}

int lanes_log2(int D) {  // lanes of 4 columns that hold a row
  int l = 1;
  while ((4 << l) < D) ++l;
  return l;
}

template <class F>
void with_type(int dtype, F&& f) {
  if (dtype == MATTN_BF16) f(bf16_tag{});
  else if (dtype == MATTN_F16) f(f16_tag{});
  else f(float{});
}
template <class F>
void with_dim(int D, F&& f) {
  if (D <= 64) f(std::integral_constant<int, 64>{});
  else f(std::integral_constant<int, 128>{});
}

bool misaligned(std::initializer_list<const void*> ps, unsigned mask) {
  for (const void* x : ps)
    if ((uintptr_t)x & mask) return true;
  return false;
}

}  // namespace
}  // namespace mattn

using namespace mattn;

extern "C" int mattn_selected_validate(const mattn_selected* p) { return sel_check(p); }

extern "C" size_t mattn_selected_lists_bytes(const mattn_selected* p) { return sel_check(p) ? 0 : sel_layout(p).lists; }

extern "C" size_t mattn_selected_fwd_workspace_bytes(const mattn_selected* p) {
  if (sel_check(p)) return 0;
  const SLayout l = sel_layout(p);
  return l.fwd + (sel_plan(p).by_query || sel_plan(p).tile_fwd ? 0 : l.lists);
}

extern "C" size_t mattn_selected_bwd_workspace_bytes(const mattn_selected* p) { return sel_check(p) ? 0 : sel_layout(p).bwd; }

extern "C" int mattn_selected_fwd(const mattn_selected* p, const void* q, const void* k, const void* v, void* o, float* o32,
                                  float* lse, void* lists, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = sel_check(p)) return rc;
  if (!q || !k || !v || !o) return MATTN_ERR_NULL;
  const bool grads = lists != nullptr;
  if (grads && (!o32 || !lse)) return MATTN_ERR_NULL;
  const size_t need = mattn_selected_fwd_workspace_bytes(p);
  if (need > 0 && !workspace) return MATTN_ERR_NULL;
  if (workspace_bytes < need) return MATTN_ERR_WORKSPACE;
  if (misaligned({q, k, v, o, o32}, 15) || misaligned({lists, workspace}, 255)) return MATTN_ERR_STRIDE;
  const SLayout l = sel_layout(p);
  const SPlan s = sel_plan(p);
  hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)workspace;
  SArgs a = sel_args(p, l, lists ? lists : ws ? ws + l.fwd : nullptr);
  a.q = q;
  a.k = k;
  a.v = v;
  a.o = o;
  a.o32 = grads ? o32 : nullptr;
  a.lse = grads ? lse : nullptr;
  a.cnt = (int*)(ws + l.cnt);
  a.odd = (int*)(ws + l.odd);
  a.part = (float*)(ws + l.part);
  a.plse = (float*)(ws + l.plse);
  if (grads || !(s.by_query || s.tile_fwd)) make_lists(a, st);
  const int ll = lanes_log2(p->D);
  const int64_t rows = (int64_t)a.bh_n * p->Lq * a.G;
  const dim3 join((uint32_t)cdiv(rows << ll, 256));
  const int hg32 = (a.G + 31) / 32, tiles_q = (int)cdiv(p->Lq, 4 * (32 / (a.G < 32 ? a.G : 32)));
  const dim3 tiles((uint32_t)((int64_t)a.bh_n * hg32 * tiles_q));
  with_type(p->dtype, [&](auto tag) {
    using Tag = decltype(tag);
    with_dim(p->D, [&](auto dim) {
      constexpr int D = decltype(dim)::value;
      if (s.by_query)
        hipLaunchKernelGGL((by_query<Tag, D>), dim3((uint32_t)(a.bh_n * p->Lq * s.hgroups * s.splits)), dim3(256), 0, st, a, s.splits, s.hgroups);
      else if (s.tile_fwd)
        hipLaunchKernelGGL((by_tile<Tag, D, false>), tiles, dim3(256), 0, st, a, hg32, tiles_q);
      else
        hipLaunchKernelGGL((by_block_q<Tag, D, false>), dim3((uint32_t)(a.bh_n * l.max_tiles)), dim3(256), 0, st, a);
    });
    if (!s.by_query && !s.tile_fwd) hipLaunchKernelGGL((join_rows<Tag, false>), join, dim3(256), 0, st, a, ll, p->count, false);
    else if (s.by_query && s.splits > 1) hipLaunchKernelGGL((join_rows<Tag, false>), join, dim3(256), 0, st, a, ll, s.splits, true);
  });
  return hipGetLastError() == hipSuccess ? MATTN_OK : MATTN_ERR_LAUNCH;
}

extern "C" int mattn_selected_bwd(const mattn_selected* p, const void* q, const void* k, const void* v, const float* o32,
                                  const void* do_, const float* lse, const void* lists, void* workspace,
                                  size_t workspace_bytes, void* dq, void* dk, void* dv, void* stream) {
  if (const int rc = sel_check(p)) return rc;
  if (!q || !k || !v || !o32 || !do_ || !lse || !lists || !workspace || !dq || !dk || !dv) return MATTN_ERR_NULL;
  const SLayout l = sel_layout(p);
  if (workspace_bytes < l.bwd) return MATTN_ERR_WORKSPACE;
  if (misaligned({q, k, v, o32, do_, dq, dk, dv}, 15) || misaligned({lists, workspace}, 255)) return MATTN_ERR_STRIDE;
  hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)workspace;
  SArgs a = sel_args(p, l, const_cast<void*>(lists));
  a.q = q;
  a.k = k;
  a.v = v;
  a.dO = do_;
  a.o32 = const_cast<float*>(o32);
  a.lse = const_cast<float*>(lse);
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  a.delta = (float*)(ws + l.delta);
  a.part = (float*)(ws + l.dqpart);
  const SPlan s = sel_plan(p);
  a.kvpart = (float*)(ws + l.kvpart);
  a.ds = s.tile_bwd ? ws + l.ds : nullptr;
  a.odd = (int*)(ws + l.bodd);
  a.kvodd = (int*)(ws + l.kvodd);
  const int ll = lanes_log2(p->D);
  const int64_t rows = (int64_t)a.bh_n * p->Lq * a.G;
  const dim3 join((uint32_t)cdiv(rows << ll, 256));
  const int KT = key_tile(p);
  const dim3 keys((uint32_t)cdiv((int64_t)p->Lk * (p->D / 4), 256), 2 * a.bh_n);
  const int hg32 = (a.G + 31) / 32, tiles_q = (int)cdiv(p->Lq, 4 * (32 / (a.G < 32 ? a.G : 32)));
  const dim3 tiles((uint32_t)((int64_t)a.bh_n * hg32 * tiles_q));
  with_type(p->dtype, [&](auto tag) {
    using Tag = decltype(tag);
    hipLaunchKernelGGL((row_delta<Tag>), join, dim3(256), 0, st, a, ll);
    with_dim(p->D, [&](auto dim) {
      constexpr int D = decltype(dim)::value;
      if (!s.tile_bwd) hipLaunchKernelGGL((by_block_q<Tag, D, true>), dim3((uint32_t)(a.bh_n * l.max_tiles)), dim3(256), 0, st, a);
      const dim3 items((uint32_t)(a.bh_n * l.max_kv));
      if constexpr (std::is_same_v<Tag, float>) {
        if (KT == 128) hipLaunchKernelGGL((by_block_kv<D, 128>), items, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((by_block_kv<D, 64>), items, dim3(256), 0, st, a);
      } else if (s.tile_bwd) {
        hipLaunchKernelGGL((by_block_kv16<Tag, D, true>), items, dim3(512), 0, st, a);
        hipLaunchKernelGGL((by_tile<Tag, D, true>), tiles, dim3(256), 0, st, a, hg32, tiles_q);
      } else {
        hipLaunchKernelGGL((by_block_kv16<Tag, D, false>), items, dim3(512), 0, st, a);
      }
    });
    if (!s.tile_bwd) hipLaunchKernelGGL((join_rows<Tag, true>), join, dim3(256), 0, st, a, ll, p->count, false);
    hipLaunchKernelGGL((join_keys<Tag>), keys, dim3(256), 0, st, a, KT);
  });
  return hipGetLastError() == hipSuccess ? MATTN_OK : MATTN_ERR_LAUNCH;
}
