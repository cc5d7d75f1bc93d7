// Rotary positions, with or without the RMS norm of each head before them (mattn_rotary,
// mattn_norm_rotary_bwd).
//
//   y = x r w,  r = (mean x^2 + eps)^-1/2   (with NORM; y = x without)
//   z = s R(p f) y: columns (i, i + dim / 2) ("half") or (2 i, 2 i + 1) ("interleaved")
//       of the first dim turned by the angle p f_i, the others as they are
//   backward: dy = s R(-p f) dz, g = dy w, dx = r (g - x r mean(g x r)),
//             dw = sum over rows of dy x r
//
// Bound by HBM: a row is read and written once, the norm's sum stays in registers.  A
// row is held by the LPR lanes (a power of two) of one group, each two chunks of 16
// bytes: with "half" the chunks V i and dim / 2 + V i, otherwise two neighbours, so that
// both columns of a pair are always one lane's.  All heads of a position share its
// angles: a workgroup takes PW positions, forms their cosines and sines once in LDS and
// each lane reads its V pairs once for all the heads it walks.
//
// Angles are formed in float64 and reduced to half turns there: at position 10^6 a
// float32 product is off by 0.06 rad.  Sums, statistics and weight gradients are float32
// (a thread's rows, then the groups of a workgroup, then the workgroups in a fixed
// order: no atomics).
//
// Waiting for a row before asking for the next left half the bandwidth unused: a lane now
// asks for its next head's row before it works on the one at hand.  The backward gives
// each tensor its own workgroups, whose weight gradients then fit the registers (both
// tensors' spilled: 148 us against 121).  Measured, bf16, d = 128: 16384 positions of 32 + 8
// heads forward 63 us (5.3 TB/s); 8192 of 32 + 32 heads forward 51 us (5.3 TB/s), backward
// 121 us (3.3 TB/s; a copy reaches 4.8 TB/s) and 7 us of weights.  A one-token call is 5 us of
// kernel.
#include "elem.hpp"

namespace mattn {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPW = 8;        // positions a workgroup forms angles of at a time
constexpr int kMaxHalf = 256;    // dim / 2 at most
constexpr int kMaxGrid = 2048;   // 8 workgroups a CU; more positions are walked

struct RotArgs {
  mattn_rotary p;
  float* part;   // backward: [grid][2][D] partial weight gradients
  int lpr_log2;  // lanes of a row
  int pw_log2;   // positions of a workgroup
  int slots;     // lane slots of a row that hold columns
};

// The columns of lane slot s: a chunk of V at `a` and, where b >= 0, one at `b`;
// rot: they hold V pairs, first pair V s.
struct Slot {
  int a, b;
  bool any, rot;
};
template <int V>
__device__ __forceinline__ Slot slot_of(const RotArgs& A, int s) {
  const int nrot = A.p.dim / (2 * V);
  Slot t;
  t.any = s < A.slots;
  t.rot = s < nrot;
  if (t.rot) {
    const bool half = A.p.layout == MATTN_ROTARY_HALF;
    t.a = half ? V * s : 2 * V * s;
    t.b = half ? A.p.dim / 2 + V * s : t.a + V;
  } else {
    t.a = A.p.dim + 2 * V * (s - nrot);
    t.b = t.a + V < A.p.D ? t.a + V : -1;
  }
  return t;
}

// pairs (first, second): with "half" (a[i], b[i]); interleaved, 2 V consecutive values
template <int V>
__device__ __forceinline__ void turn(float (&a)[V], float (&b)[V], const float (&c)[V], const float (&s)[V], bool half) {
  if (half) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float x = a[i], y = b[i];
      a[i] = x * c[i] - y * s[i];
      b[i] = y * c[i] + x * s[i];
    }
  } else if constexpr (V == 1) {
    const float x = a[0], y = b[0];
    a[0] = x * c[0] - y * s[0];
    b[0] = y * c[0] + x * s[0];
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      float x = a[2 * i], y = a[2 * i + 1];
      a[2 * i] = x * c[i] - y * s[i];
      a[2 * i + 1] = y * c[i] + x * s[i];
      x = b[2 * i], y = b[2 * i + 1];
      b[2 * i] = x * c[V / 2 + i] - y * s[V / 2 + i];
      b[2 * i + 1] = y * c[V / 2 + i] + x * s[V / 2 + i];
    }
  }
}

// Sine and cosine of `turns` turns, each to a few float32 steps of its own value: the
// nearest quarter is taken off in float64, so that neither loses its leading digits
// where it is small.
__device__ __forceinline__ void turn_angle(double turns, float& s, float& c) {
  const double t = 4.0 * (turns - rint(turns)), q = rint(t);
  float x, y;
  sincospif((float)(0.5 * (t - q)), &y, &x);
  const int k = (int)q & 3;
  s = k == 0 ? y : k == 1 ? x : k == 2 ? -y : -x;
  c = k == 0 ? x : k == 1 ? -y : k == 2 ? -x : y;
}

__device__ __forceinline__ float group_sum(float x, int lpr) {
  for (int o = lpr >> 1; o; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// Tag: element type; V: elements of a chunk (16 bytes, or 1 where lengths or addresses
// do not allow those); NIT: lane slots a lane walks (more than 64 only with V = 1).
// MODE 0: rotation, 1: norm and rotation, 2: their backward.
template <class Tag, int V, int NIT, int MODE>
__global__ __attribute__((amdgpu_flat_work_group_size(kThreads, kThreads), amdgpu_waves_per_eu(MODE == 2 ? (NIT == 1 ? 3 : 2) : 4)))
void rotary_kernel(RotArgs A) {
  __shared__ __align__(16) float cs[kMaxPW * kMaxHalf], sn[kMaxPW * kMaxHalf];
  const mattn_rotary& P = A.p;
  const int lpr = 1 << A.lpr_log2, pw = 1 << A.pw_log2, nh = P.dim >> 1;
  const int lane = threadIdx.x & (lpr - 1), grp = threadIdx.x >> A.lpr_log2;  // row group
  const int gpp_log2 = 8 - A.lpr_log2 - A.pw_log2;                          // row groups of a position
  const int pi = grp >> gpp_log2, hg = grp & ((1 << gpp_log2) - 1), gpp = 1 << gpp_log2;
  const bool half = P.layout == MATTN_ROTARY_HALF;
  const int64_t n = (int64_t)P.B * P.L;

  Slot sl[NIT];
#pragma unroll
  for (int i = 0; i < NIT; ++i) sl[i] = slot_of<V>(A, lane + 64 * i);
  // backward: a tensor a workgroup (its weights' gradients stay in registers)
  const int t0 = MODE == 2 ? blockIdx.y : 0, t1 = MODE == 2 ? t0 + 1 : P.n;
  float dw[MODE == 2 ? NIT : 1][2][V];
  if constexpr (MODE == 2) {
#pragma unroll
    for (int i = 0; i < NIT; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) dw[i][0][e] = dw[i][1][e] = 0.f;
  }

  for (int64_t p0 = (int64_t)blockIdx.x << A.pw_log2; p0 < n; p0 += (int64_t)gridDim.x << A.pw_log2) {
    __syncthreads();  // the angles of the positions before are read
    for (int i = threadIdx.x; i < pw * nh; i += kThreads) {
      const int64_t at = p0 + i / nh;
      if (at < n) {
        const int64_t b = at / P.L, l = at % P.L;
        const int64_t e = b * P.pos_stride[0] + l * P.pos_stride[1];
        const double pos = P.pos_bytes == 0 ? (double)l
                           : P.pos_bytes == 4 ? (double)((const int32_t*)P.positions)[e]
                                              : (double)((const int64_t*)P.positions)[e];
        const double turns = pos * P.inv_freq[i % nh] * 0.15915494309189533577;
        float s, c;
        turn_angle(turns, s, c);
        cs[i] = c * P.scale;
        sn[i] = (MODE == 2 || P.inverse ? -s : s) * P.scale;
      }
    }
    __syncthreads();
    const int64_t at = p0 + pi;
    if (at >= n) continue;
    const int64_t b = at / P.L, l = at % P.L;
    float c[NIT][V], s[NIT][V];
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
#pragma unroll
      for (int e = 0; e < V; ++e) c[i][e] = s[i][e] = 0.f;
      if (sl[i].rot) {
        load_v<float, V>(cs, pi * nh + V * (lane + 64 * i), c[i]);
        load_v<float, V>(sn, pi * nh + V * (lane + 64 * i), s[i]);
      }
    }
    for (int t = t0; t < t1; ++t) {
      const int64_t xo = b * P.x_stride[t][0] + l * P.x_stride[t][1];
      const int64_t yo = b * P.y_stride[t][0] + l * P.y_stride[t][1];
      const int64_t go = MODE == 2 ? b * P.g_stride[t][0] + l * P.g_stride[t][1] : 0;
      float w[NIT][2][V];
      if constexpr (MODE != 0) {
#pragma unroll
        for (int i = 0; i < NIT; ++i) {
#pragma unroll
          for (int e = 0; e < V; ++e) w[i][0][e] = w[i][1][e] = 1.f;
          if (P.w[t] && sl[i].any) {
            load_v<float, V>(P.w[t], sl[i].a, w[i][0]);
            if (sl[i].b >= 0) load_v<float, V>(P.w[t], sl[i].b, w[i][1]);
          }
        }
      }
      // a row's columns as they lie in memory (a slot without columns: zeros); the next
      // head's are on their way while this one's are worked on
      using R = Raw<Tag, V>;
      R nx[NIT][2], ng[MODE == 2 ? NIT : 1][2];
      const auto load = [&](int h) {
#pragma unroll
        for (int i = 0; i < NIT; ++i) {
          nx[i][0] = nx[i][1] = R{};
          if constexpr (MODE == 2) ng[i][0] = ng[i][1] = R{};
          if (sl[i].any) {
            const int64_t r = xo + h * P.x_stride[t][2], q = go + h * P.g_stride[t][2];
            nx[i][0] = load_raw<Tag, V>(P.x[t], r + sl[i].a);
            if constexpr (MODE == 2) ng[i][0] = load_raw<Tag, V>(P.g[t], q + sl[i].a);
            if (sl[i].b >= 0) {
              nx[i][1] = load_raw<Tag, V>(P.x[t], r + sl[i].b);
              if constexpr (MODE == 2) ng[i][1] = load_raw<Tag, V>(P.g[t], q + sl[i].b);
            }
          }
        }
      };
      if (hg < P.H[t]) load(hg);
      for (int h = hg; h < P.H[t]; h += gpp) {
        float x[NIT][2][V], g[MODE == 2 ? NIT : 1][2][V];
#pragma unroll
        for (int i = 0; i < NIT; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            from_raw<Tag, V>(nx[i][j], x[i][j]);
            if constexpr (MODE == 2) from_raw<Tag, V>(ng[i][j], g[i][j]);
          }
        if (h + gpp < P.H[t]) load(h + gpp);
        float r = 1.f;
        if constexpr (MODE != 0) {
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < NIT; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) ss += x[i][0][e] * x[i][0][e] + x[i][1][e] * x[i][1][e];
          r = 1.f / sqrtf(group_sum(ss, lpr) / (float)P.D + P.eps);
        }
        if constexpr (MODE == 1) {
#pragma unroll
          for (int i = 0; i < NIT; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
              x[i][0][e] *= r * w[i][0][e];
              x[i][1][e] *= r * w[i][1][e];
            }
        }
        if constexpr (MODE == 2) {
          float m = 0.f;
#pragma unroll
          for (int i = 0; i < NIT; ++i) {
            if (sl[i].rot) turn<V>(g[i][0], g[i][1], c[i], s[i], half);
#pragma unroll
            for (int e = 0; e < V; ++e)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                x[i][j][e] *= r;
                dw[i][j][e] += g[i][j][e] * x[i][j][e];
                g[i][j][e] *= w[i][j][e];
                m += g[i][j][e] * x[i][j][e];
              }
          }
          m = group_sum(m, lpr) / (float)P.D;
#pragma unroll
          for (int i = 0; i < NIT; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e)
#pragma unroll
              for (int j = 0; j < 2; ++j) x[i][j][e] = r * (g[i][j][e] - x[i][j][e] * m);
        } else {
#pragma unroll
          for (int i = 0; i < NIT; ++i)
            if (sl[i].rot) turn<V>(x[i][0], x[i][1], c[i], s[i], half);
        }
        const int64_t q = yo + h * P.y_stride[t][2];
#pragma unroll
        for (int i = 0; i < NIT; ++i)
          if (sl[i].any) {
            store_v<Tag, V>(P.y[t], q + sl[i].a, x[i][0]);
            if (sl[i].b >= 0) store_v<Tag, V>(P.y[t], q + sl[i].b, x[i][1]);
          }
      }
    }
  }

  if constexpr (MODE == 2) {  // the row groups' weight gradients, a chunk at a time
    const int ng = kThreads >> A.lpr_log2;
#pragma unroll
    for (int i = 0; i < NIT; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) cs[threadIdx.x + kThreads * e] = dw[i][j][e];
        __syncthreads();
        const int o = j == 0 ? sl[i].a : sl[i].b;
        if (grp == 0 && sl[i].any && o >= 0) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            float sum = 0.f;
            for (int k = 0; k < ng; ++k) sum += cs[(k << A.lpr_log2) + lane + kThreads * e];
            A.part[((int64_t)blockIdx.x * 2 + t0) * P.D + o + e] = sum;
          }
        }
      }
  }
}

// dw[t][c] = sum over the workgroups' partial gradients, in a fixed order: 16 columns by 64
// interleaved runs of workgroups, then the runs.
__global__ __attribute__((amdgpu_flat_work_group_size(1024, 1024)))
void rotary_dw(const float* part, int n, int D, float* dw0, float* dw1) {
  __shared__ float red[1024];
  const int c = blockIdx.x * 16 + (threadIdx.x & 15), t = blockIdx.y, run = threadIdx.x >> 4;
  float sum = 0.f;
  if (c < D) {
#pragma unroll 8
    for (int i = run; i < n; i += 64) sum += part[((int64_t)i * 2 + t) * D + c];
  }
  red[threadIdx.x] = sum;
  __syncthreads();
  float* dw = t == 0 ? dw0 : dw1;
  if (run == 0 && c < D && dw) {
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < 64; ++i) sum += red[i * 16 + threadIdx.x];
    dw[c] = sum;
  }
}

// Lanes, positions and grid of a problem.  vec: 16-byte chunks.
struct RotPlan {
  int lpr_log2, pw_log2, slots, grid;
};
bool rot_vec(const mattn_rotary* p, bool bwd) {
  const int es = p->dtype == MATTN_F32 ? 4 : 2, V = 16 / es;
  if ((p->dim / 2) % V || (p->D - p->dim) % V) return false;
  for (int t = 0; t < p->n; ++t) {
    if (((uintptr_t)p->x[t] | (uintptr_t)p->y[t] | (bwd ? (uintptr_t)p->g[t] : 0) | (p->norm ? (uintptr_t)p->w[t] : 0)) & 15)
      return false;
    for (int i = 0; i < 3; ++i)
      if ((p->x_stride[t][i] | p->y_stride[t][i] | (bwd ? p->g_stride[t][i] : 0)) % V) return false;
  }
  return true;
}
RotPlan rot_plan(const mattn_rotary* p, bool vec) {
  const int V = vec ? (p->dtype == MATTN_F32 ? 4 : 8) : 1;
  RotPlan r;
  r.slots = p->dim / (2 * V) + ((p->D - p->dim) / V + 1) / 2;
  r.lpr_log2 = 0;
  while ((1 << r.lpr_log2) < r.slots && r.lpr_log2 < 6) ++r.lpr_log2;
  // as many positions as leave a row group at least 4 heads, and the card its workgroups
  const int64_t n = (int64_t)p->B * p->L;
  const int heads = p->H[0] + (p->n > 1 ? p->H[1] : 0);
  r.pw_log2 = 0;
  while (r.pw_log2 < 3 && r.pw_log2 + r.lpr_log2 < 8 && ((int64_t)heads << (r.pw_log2 + r.lpr_log2)) < 4 * kThreads &&
         (n >> (r.pw_log2 + 1)) >= 512)
    ++r.pw_log2;
  const int64_t wgs = (n + (1 << r.pw_log2) - 1) >> r.pw_log2;
  r.grid = (int)(wgs < kMaxGrid ? wgs : kMaxGrid);
  return r;
}

int rot_check(const mattn_rotary* p, bool norm, bool bwd) {
  if (!p) return MATTN_ERR_NULL;
  if (p->n != 1 && p->n != 2) return MATTN_ERR_SHAPE;
  if (p->B <= 0 || p->L <= 0 || p->D <= 0 || p->D > 512 || p->dim < 0 || p->dim > p->D || p->dim % 2) return MATTN_ERR_SHAPE;
  if (p->dtype != MATTN_BF16 && p->dtype != MATTN_F16 && p->dtype != MATTN_F32) return MATTN_ERR_DTYPE;
  if (p->layout != MATTN_ROTARY_HALF && p->layout != MATTN_ROTARY_INTERLEAVED) return MATTN_ERR_SHAPE;
  if (p->pos_bytes != 0 && p->pos_bytes != 4 && p->pos_bytes != 8) return MATTN_ERR_DTYPE;
  if ((p->dim > 0 && !p->inv_freq) || (p->pos_bytes && !p->positions)) return MATTN_ERR_NULL;
  for (int t = 0; t < p->n; ++t) {
    if (p->H[t] <= 0) return MATTN_ERR_SHAPE;
    if (!p->x[t] || !p->y[t] || (bwd && !p->g[t])) return MATTN_ERR_NULL;
    for (int i = 0; i < 3; ++i)
      if (p->x_stride[t][i] < 0 || p->y_stride[t][i] < 0 || (bwd && p->g_stride[t][i] < 0)) return MATTN_ERR_STRIDE;
  }
  if (norm && !(p->eps >= 0.f)) return MATTN_ERR_SHAPE;
  return MATTN_OK;
}

template <int MODE>
int rot_launch(const mattn_rotary* p, float* part, hipStream_t st) {
  const bool vec = rot_vec(p, MODE == 2);
  const RotPlan r = rot_plan(p, vec);
  const RotArgs a{*p, part, r.lpr_log2, r.pw_log2, r.slots};
  const auto go = [&](auto tag, auto v, auto nit) {
    hipLaunchKernelGGL((rotary_kernel<decltype(tag), decltype(v)::value, decltype(nit)::value, MODE>), dim3(r.grid, MODE == 2 ? p->n : 1),
                       dim3(kThreads), 0, st, a);
  };
  using one = std::integral_constant<int, 1>;
  const auto pick = [&](auto tag) {
    constexpr int V = kChunk<decltype(tag)>;
    if (vec) go(tag, std::integral_constant<int, V>{}, one{});
    else if (r.slots <= 64) go(tag, one{}, one{});
    else go(tag, one{}, std::integral_constant<int, 4>{});
  };
  if (p->dtype == MATTN_BF16) pick(bf16_tag{});
  else if (p->dtype == MATTN_F16) pick(f16_tag{});
  else pick(float{});
  return hipGetLastError() == hipSuccess ? MATTN_OK : MATTN_ERR_LAUNCH;
}

}  // namespace
}  // namespace mattn

using namespace mattn;

extern "C" int mattn_rotary_fwd(const mattn_rotary* p, void* stream) {
  const bool norm = p && p->norm;
  if (const int rc = rot_check(p, norm, false)) return rc;
  if (norm && p->inverse) return MATTN_ERR_SHAPE;
  return norm ? rot_launch<1>(p, nullptr, (hipStream_t)stream) : rot_launch<0>(p, nullptr, (hipStream_t)stream);
}

extern "C" size_t mattn_norm_rotary_bwd_workspace_bytes(const mattn_rotary* p) {
  if (rot_check(p, true, true)) return 0;
  return (size_t)rot_plan(p, rot_vec(p, true)).grid * 2 * p->D * sizeof(float);
}

extern "C" int mattn_norm_rotary_bwd(const mattn_rotary* p, float* dw0, float* dw1, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  if (const int rc = rot_check(p, true, true)) return rc;
  if (!workspace) return MATTN_ERR_NULL;
  if (workspace_bytes < mattn_norm_rotary_bwd_workspace_bytes(p)) return MATTN_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 3) return MATTN_ERR_STRIDE;
  if (const int rc = rot_launch<2>(p, (float*)workspace, (hipStream_t)stream)) return rc;
  if (!dw0 && !dw1) return MATTN_OK;
  hipLaunchKernelGGL(rotary_dw, dim3((p->D + 15) / 16, p->n), dim3(1024), 0, (hipStream_t)stream, (const float*)workspace,
                     rot_plan(p, rot_vec(p, true)).grid, p->D, dw0, dw1);
  return hipGetLastError() == hipSuccess ? MATTN_OK : MATTN_ERR_LAUNCH;
}
