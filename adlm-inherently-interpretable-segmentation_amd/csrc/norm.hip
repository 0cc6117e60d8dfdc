// norm.hip — group norm with an activation on channels-last maps (gfx950), forward and backward.
//
// For sample b and group g (M = HW * C / G values: the group's channels at every pixel)
//   mean = p + sum (x - p) / M,  rstd = 1 / sqrt(sum (x - p)^2 / M - (mean - p)^2 + eps)
// with the pivot p, the group's first value, and sums in f64
//   xh = (x - mean) rstd,  z = xh w[c] + beta[c],  y = act(z)
// and with gz = gy act'(z), per channel S1 = sum_pixels gz, S2 = sum_pixels gz xh,
//   g_w[c] = sum_b S2,  g_beta[c] = sum_b S1
//   g_x = rstd (w gz - (c1 + xh c2)),  c1 = sum_{c in g} w S1 / M,  c2 = sum_{c in g} w S2 / M
// Nothing here is a matrix product: every kernel is bound by the bytes it moves. A map is read as
// rows of C channels: a thread owns one vector of V channels (16 B where C, the strides and the
// addresses allow it, else 4 B or one element) and walks down the pixels, so a wave's loads are
// contiguous over the row and its per-channel constants stay in registers. Pixels are cut into
// chunks over workgroups; their partial sums are joined in a fixed order (no atomics: the same
// bits on every run).
#include <type_traits>

#include "protoseg_device.h"
#include "protoseg_host.h"

namespace protoseg {

namespace {

constexpr int kGnThreads = 256;
constexpr long long kGnTarget = 512, kGnLeast = 4096, kGnEnough = 16384, kGnMost = 1 << 18;  // gn_chunks
constexpr long long kGnJoinInside = 4096;  // gn_apply_kernel

enum GnAct { kGnIdentity = 0, kGnRelu = 1, kGnSigmoid = 2, kGnSilu = 3 };

// V consecutive elements as f32 (one 16-B / 4-B / element load), and back (round to nearest even).
template <typename T, int V>
struct Raw {
  typedef T type __attribute__((ext_vector_type(V)));
};
template <typename T>
struct Raw<T, 1> {
  typedef T type;
};
template <typename T, int V>
__device__ __forceinline__ void unpack(const typename Raw<T, V>::type& r, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = static_cast<float>(r);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = static_cast<float>(r[i]);
  }
}
template <typename T, int V>
__device__ __forceinline__ typename Raw<T, V>::type pack(const float (&v)[V]) {
  typename Raw<T, V>::type r;
  if constexpr (V == 1) {
    r = static_cast<T>(v[0]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = static_cast<T>(v[i]);
  }
  return r;
}

struct GnMap {  // element (b, pixel, c) at p[b * sb + pixel * sp + c]
  const void* p;
  long long sb, sp;
};

struct GnShape {
  int B, HW, C, G, cpg;
  int ppc, nchunk;  // pixels per chunk, chunks per sample
  bool stream;      // NT of put_map, where vectors are 16 B
};

// A result beyond the L2s (8 x 4 MiB) is stored past the caches: kept there it would push out the map that the
// second pass reads again (1 x 2048 x 129 x 257 bf16, three maps in turn: 80.8 us for 91.8, and 125 for 135 with
// a reader behind it). A smaller one is left to the operation that reads it (3 x 150 x 33 x 47 f16 with a
// reader: 24.7 us for 26.0).
constexpr long long kGnStream = 32 << 20;
template <bool NT, typename V>
__device__ __forceinline__ void put_map(V* p, const V& v) {
  if constexpr (NT) __builtin_nontemporal_store(v, p);
  else *p = v;
}

// 1 / (1 + exp(-z)) by v_exp_f32 and v_rcp_f32 (1 ulp each; the exponent's argument is rounded
// once, so the relative error is |z| 2^-24 + 2^-22): exact division and exp would make the 16-bit
// kernels wait for the vector unit instead of the memory.
__device__ __forceinline__ float sigmoid_of(float z) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504f));
}
template <int ACT>
__device__ __forceinline__ float act_of(float z) {
  if constexpr (ACT == kGnRelu) return z < 0.f ? 0.f : z;  // NaN stays NaN
  if constexpr (ACT == kGnSigmoid) return sigmoid_of(z);
  if constexpr (ACT == kGnSilu) return z * sigmoid_of(z);
  return z;
}

// What a thread keeps of its V channels: V / S runs of S channels, each inside one group.
template <int V, int S>
struct GnCoef {
  float mh[V / S], ml[V / S];  // mean as a pair: x - mh is exact near the mean, so a mean far larger than the spread costs nothing
  float a[V], beta[V];         // rstd * w, bias
};

// Column layout of a workgroup: `cb` vectors of V channels per pixel row, R pixel rows per step.
struct GnLane {
  int cb, R, col, row;
  bool on;
};
template <int V>
__device__ __forceinline__ GnLane gn_lane(int C) {
  GnLane l;
  const int ncol = C / V, left = ncol - static_cast<int>(blockIdx.y) * kGnThreads;
  l.cb = left < kGnThreads ? left : kGnThreads;
  l.R = kGnThreads / l.cb;
  l.row = static_cast<int>(threadIdx.x) / l.cb;
  l.col = static_cast<int>(threadIdx.x) - l.row * l.cb;
  l.on = l.row < l.R;
  return l;
}

// The groups that a workgroup's channels [c0, c1) meet: at most one per run, and a broken one at either end.
constexpr int gn_most_groups(int V, int S) { return kGnThreads * V / S + 2; }
struct GnGroups {
  int c0, c1, g0, ng;
};
template <int V>
__device__ __forceinline__ GnGroups gn_groups(const GnLane& l, const GnShape& s) {
  GnGroups g;
  g.c0 = static_cast<int>(blockIdx.y) * kGnThreads * V;
  g.c1 = g.c0 + l.cb * V;
  g.g0 = g.c0 / s.cpg;
  g.ng = (g.c1 - 1) / s.cpg - g.g0 + 1;
  return g;
}

template <typename T>
__device__ __forceinline__ T wave_part_sum(T v, int lanes) {  // over aligned runs of `lanes` (a power of two)
  for (int m = 1; m < lanes; m <<= 1) v += __shfl_xor(v, m);
  return v;
}
// Lanes given to each of n items by a 256-thread workgroup: the largest power of two up to a wave.
__host__ __device__ __forceinline__ int lanes_per(int n) {
  int l = 64;
  while (l > 1 && n * l > kGnThreads) l >>= 1;
  return l;
}

// Partial pairs of the chunks: a workgroup (chunk, block of channels) leaves one pair for each group
// that it meets, part[(b * nchunk + chunk) * gy + block][ngb]. pair_total joins those of one group,
// `lanes` lanes a group, each result in every lane. A group that lies in two blocks of channels is joined by the
// workgroups of both: `lanes`, and with it the order of the sum, is the same for all of them.
struct GnParts {
  int gy, ngb, block_c;  // blocks of channels, pairs per block, channels per block
  int lanes;
};
template <typename P2>
__device__ __forceinline__ void pair_total(const P2* __restrict__ part, const GnParts& pt, const GnShape& s, int b, int g,
                                           int sub, int lanes, double& a, double& q) {
  const int y0 = g * s.cpg / pt.block_c, ny = ((g + 1) * s.cpg - 1) / pt.block_c - y0 + 1;
  a = q = 0.0;
#pragma unroll 4
  for (int e = sub; e < s.nchunk * ny; e += lanes) {
    const int chunk = ny == 1 ? e : e / ny, y = y0 + e - chunk * ny;
    const P2 v = part[((static_cast<long long>(b) * s.nchunk + chunk) * pt.gy + y) * pt.ngb + g - y * pt.block_c / s.cpg];
    a += static_cast<double>(v.x);
    q += static_cast<double>(v.y);
  }
  a = wave_part_sum(a, lanes);
  q = wave_part_sum(q, lanes);
}

// The first value of a group: what its sums are taken from. The variance is a difference of two sums, and a rounding
// of one of them is as large as the mean's square: from 0 they lose the variance's f32 digits at means of 2^13
// spreads and 8e-4 of it at 2^20. From a value of the group itself both sums are of the spread's size, or the
// value lies so far out that it makes the variance.
template <typename T>
__device__ __forceinline__ double gn_pivot(const GnMap& x, const GnShape& s, int b, int g) {
  return static_cast<double>(static_cast<float>(static_cast<const T*>(x.p)[b * x.sb + g * s.cpg]));
}

// Partial sums of one chunk: (sum x - p, sum (x - p)^2) of each group that the workgroup's channels meet.
// f64 from the first subtraction on: three f64 operations an element are far below
// the rate that would bound the kernel. 1 x 2048 x 129 x 257 bf16: 22.2 us, 6.1 TB/s. Maps of a few MB
// (2 x 256 x 65 x 65 bf16: 4.6 us) are a launch and the latency of two rounds of loads.
template <typename T, int V, int S>
__global__ __launch_bounds__(kGnThreads) void gn_stats_kernel(GnMap x, GnShape s, GnParts pt, double2* __restrict__ part) {
  constexpr int kN = V / S, kU = 8;
  __shared__ double red[2][kGnThreads * kN];
  const int b = static_cast<int>(blockIdx.x) / s.nchunk, chunk = static_cast<int>(blockIdx.x) - b * s.nchunk;
  const GnLane l = gn_lane<V>(s.C);
  const GnGroups gr = gn_groups<V>(l, s);
  typedef typename Raw<T, V>::type vec;
  double sum[kN], sq[kN], pivot[kN];
#pragma unroll
  for (int n = 0; n < kN; ++n) sum[n] = sq[n] = 0.0;
  if (l.on) {
    const int c = gr.c0 + l.col * V;
    int g = c / s.cpg;
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      if (c + n * S >= (g + 1) * s.cpg) ++g;  // a run lies in one group, the next run in the same or the next one
      pivot[n] = gn_pivot<T>(x, s, b, g);
    }
    const int p1 = min(s.HW, (chunk + 1) * s.ppc);
    const T* src = static_cast<const T*>(x.p) + b * x.sb + gr.c0 + l.col * V;
    int p = chunk * s.ppc + l.row;
    auto add = [&](const vec& r) {
      float v[V];
      unpack<T, V>(r, v);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const double d = static_cast<double>(v[i]) - pivot[i / S];
        sum[i / S] += d;
        sq[i / S] = fma(d, d, sq[i / S]);
      }
    };
    for (; p + (kU - 1) * l.R < p1; p += kU * l.R) {
      vec r[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) r[u] = *reinterpret_cast<const vec*>(src + (p + u * l.R) * x.sp);
#pragma unroll
      for (int u = 0; u < kU; ++u) add(r[u]);
    }
    for (; p < p1; p += l.R) add(*reinterpret_cast<const vec*>(src + p * x.sp));
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      red[0][(l.row * l.cb + l.col) * kN + n] = sum[n];
      red[1][(l.row * l.cb + l.col) * kN + n] = sq[n];
    }
  }
  __syncthreads();
  const int nrun = l.cb * kN;  // rows first, then the runs of each group
  for (int i = threadIdx.x; i < nrun; i += kGnThreads) {
    double a = red[0][i], q = red[1][i];
    for (int r = 1; r < l.R; ++r) {
      a += red[0][r * nrun + i];
      q += red[1][r * nrun + i];
    }
    red[0][i] = a;
    red[1][i] = q;
  }
  __syncthreads();
  const int lanes = lanes_per(gr.ng), sub = static_cast<int>(threadIdx.x) & (lanes - 1);
  double2* out = part + (static_cast<long long>(blockIdx.x) * pt.gy + blockIdx.y) * pt.ngb;
  for (int gi = static_cast<int>(threadIdx.x) / lanes; gi < gr.ng; gi += kGnThreads / lanes) {
    const int lo = max((gr.g0 + gi) * s.cpg, gr.c0), hi = min((gr.g0 + gi + 1) * s.cpg, gr.c1);
    double a = 0.0, q = 0.0;
    for (int i = (lo - gr.c0) / S + sub; i < (hi - gr.c0) / S; i += lanes) {
      a += red[0][i];
      q += red[1][i];
    }
    a = wave_part_sum(a, lanes);
    q = wave_part_sum(q, lanes);
    if (sub == 0) out[gi] = make_double2(a, q);
  }
}

__device__ __forceinline__ double2 stat_of(double sum, double sq, double M, double eps, double pivot) {
  const double d = sum / M;
  double var = sq / M - d * d;
  var = var < 0.0 ? 0.0 : var;  // NaN stays NaN
  return make_double2(pivot + d, 1.0 / sqrt(var + eps));
}

// One workgroup per (group, sample): the chunks' partials joined. STATS: to mean and rstd of a map of T. 3.8 to 4.8 us,
// a launch and one chain of loads.
template <typename P2, bool STATS, typename T>
__global__ __launch_bounds__(kGnThreads) void gn_join_kernel(GnMap x, const P2* __restrict__ part, GnShape s, GnParts pt,
                                                             double eps, double2* __restrict__ out) {
  __shared__ double red[2][kGnThreads / 64];
  const int g = blockIdx.x, b = blockIdx.y, wave = static_cast<int>(threadIdx.x) >> 6;
  const int y0 = g * s.cpg / pt.block_c, ny = ((g + 1) * s.cpg - 1) / pt.block_c - y0 + 1;
  double a = 0.0, q = 0.0;
#pragma unroll 4
  for (int e = threadIdx.x; e < s.nchunk * ny; e += kGnThreads) {
    const int chunk = ny == 1 ? e : e / ny, y = y0 + e - chunk * ny;
    const P2 v = part[((static_cast<long long>(b) * s.nchunk + chunk) * pt.gy + y) * pt.ngb + g - y * pt.block_c / s.cpg];
    a += static_cast<double>(v.x);
    q += static_cast<double>(v.y);
  }
  a = wave_part_sum(a, 64);
  q = wave_part_sum(q, 64);
  if ((threadIdx.x & 63) == 0) red[0][wave] = a, red[1][wave] = q;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kGnThreads / 64; ++w) a += red[0][w], q += red[1][w];
    const long long i = static_cast<long long>(b) * s.G + g;
    if constexpr (STATS) out[i] = stat_of(a, q, static_cast<double>(s.HW) * s.cpg, eps, gn_pivot<T>(x, s, b, g));
    else out[i] = make_double2(a, q);
  }
}

// (mean as a pair, rstd) of the workgroup's groups in LDS, then a thread's constants from it.
__device__ __forceinline__ float4 lds_stat(double2 st) {
  const float mh = static_cast<float>(st.x);
  return make_float4(mh, static_cast<float>(st.x - static_cast<double>(mh)), static_cast<float>(st.y), 0.f);
}
template <int V, int S>
__device__ __forceinline__ void load_coef(GnCoef<V, S>& k, const float4* cg, const float* w, const float* beta, int c0, int g0,
                                          const GnShape& s) {
  float wc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    wc[i] = w ? w[c0 + i] : 1.f;
    k.beta[i] = beta ? beta[c0 + i] : 0.f;
  }
#pragma unroll
  for (int n = 0; n < V / S; ++n) {
    const float4 st = cg[(c0 + n * S) / s.cpg - g0];
    k.mh[n] = st.x;
    k.ml[n] = st.y;
#pragma unroll
    for (int i = 0; i < S; ++i) k.a[n * S + i] = st.z * wc[n * S + i];
  }
}

// y = act(z). part: the statistics' partials, joined here by every workgroup (the first chunk's
// leave them in `stat`), or null where gn_join_kernel has joined them: a launch less costs more
// than a few thousand pairs read from L2 by each workgroup, many more than that do not.
// 1 x 2048 x 129 x 257 bf16: 44.2 us, 6.1 TB/s read and written (56.7 without the next rows' loads in
// flight while these are computed); 2 x 256 x 65 x 65 bf16: 9.3 us.
template <typename T, int V, int S, int ACT, bool NT>
__global__ __launch_bounds__(kGnThreads) void gn_apply_kernel(GnMap x, GnShape s, GnParts pt, const double2* __restrict__ part,
                                                              double eps, double2* __restrict__ stat,
                                                              const float* __restrict__ w, const float* __restrict__ beta,
                                                              T* __restrict__ y) {
  constexpr int kU = 4;
  __shared__ float4 cg[gn_most_groups(V, S)];
  const int b = static_cast<int>(blockIdx.x) / s.nchunk, chunk = static_cast<int>(blockIdx.x) - b * s.nchunk;
  const GnLane l = gn_lane<V>(s.C);
  const GnGroups gr = gn_groups<V>(l, s);
  typedef typename Raw<T, V>::type vec;
  const int c0 = gr.c0 + (l.on ? l.col : 0) * V;
  const int p1 = min(s.HW, (chunk + 1) * s.ppc);
  const T* src = static_cast<const T*>(x.p) + b * x.sb + c0;
  int p = chunk * s.ppc + l.row;
  vec r[kU];  // the first rows are on their way while the statistics are joined
#pragma unroll
  for (int u = 0; u < kU; ++u) r[u] = *reinterpret_cast<const vec*>(src + min(p + u * l.R, p1 - 1) * x.sp);
  if (part) {
    const int lanes = pt.lanes, sub = static_cast<int>(threadIdx.x) & (lanes - 1);
    for (int gi = static_cast<int>(threadIdx.x) / lanes; gi < gr.ng; gi += kGnThreads / lanes) {
      double a, q;
      pair_total(part, pt, s, b, gr.g0 + gi, sub, lanes, a, q);
      if (sub == 0) {
        const double2 st = stat_of(a, q, static_cast<double>(s.HW) * s.cpg, eps, gn_pivot<T>(x, s, b, gr.g0 + gi));
        cg[gi] = lds_stat(st);
        // by the block of its first channel alone
        if (chunk == 0 && (gr.g0 + gi) * s.cpg >= gr.c0) stat[static_cast<long long>(b) * s.G + gr.g0 + gi] = st;
      }
    }
  } else {
    for (int gi = threadIdx.x; gi < gr.ng; gi += kGnThreads) cg[gi] = lds_stat(stat[static_cast<long long>(b) * s.G + gr.g0 + gi]);
  }
  __syncthreads();
  if (!l.on) return;
  T* dst = y + static_cast<long long>(b) * s.HW * s.C + c0;
  GnCoef<V, S> k;
  load_coef<V, S>(k, cg, w, beta, c0, gr.g0, s);
  auto put = [&](const vec& rx, int pp) {
    float v[V];
    unpack<T, V>(rx, v);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = act_of<ACT>(fmaf((v[i] - k.mh[i / S]) - k.ml[i / S], k.a[i], k.beta[i]));
    put_map<NT>(reinterpret_cast<vec*>(dst + static_cast<long long>(pp) * s.C), pack<T, V>(v));
  };
  while (p < p1) {
    vec n[kU];
    const int pn = p + kU * l.R;
    if (pn < p1) {
#pragma unroll
      for (int u = 0; u < kU; ++u) n[u] = *reinterpret_cast<const vec*>(src + min(pn + u * l.R, p1 - 1) * x.sp);
    }
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (p + u * l.R < p1) put(r[u], p + u * l.R);
#pragma unroll
    for (int u = 0; u < kU; ++u) r[u] = n[u];
    p = pn;
  }
}

// gz = gy act'(z). The side of relu's border is decided as in 64 bits: where the f32 z is within
// its own rounding of 0 (four roundings of the product, one of the sum), z is formed again in f64.
template <int ACT>
__device__ __forceinline__ float grad_z(float gy, float x, float d, float a, float beta, const double2* stat, const float* w,
                                        int b, int c, const GnShape& s) {
  if constexpr (ACT == kGnIdentity) return gy;
  const float t = d * a, z = fmaf(d, a, beta);
  if constexpr (ACT == kGnRelu) {
    bool on = z > 0.f;
    if (fabsf(z) <= 4.76837158e-7f * (fabsf(t) + fabsf(beta))) {
      const double2 st = stat[static_cast<long long>(b) * s.G + c / s.cpg];
      on = fma(static_cast<double>(x) - st.x, st.y * static_cast<double>(w ? w[c] : 1.f), static_cast<double>(beta)) > 0.0;
    }
    return on ? gy : 0.f;
  }
  const float sg = sigmoid_of(z);
  if constexpr (ACT == kGnSigmoid) return gy * (sg * (1.f - sg));
  return gy * (sg * fmaf(z, 1.f - sg, 1.f));
}

// Partial sums of one chunk, S1 = sum gz and S2 = sum gz xh: per channel (part, f32 rows [2][C] of
// each workgroup), and weighted by w over each group (gpart). Sums in f64, rounded to f32
// once a chunk: the values have mixed signs, and f32 chains left a gradient of few channels 3 times the error of
// a tree of f32 sums (19 x 2 x 16 x 11). That costs the training calls' kernels 0.2 to 1.3 us of 35 to 55.
// 32 x 64 x 65 x 65 f32: 15.4 us, 4.5 TB/s.
template <typename T, int V, int S, int ACT>
__global__ __launch_bounds__(kGnThreads) void gn_bwd_sums_kernel(GnMap x, GnMap gy, GnShape s, GnParts pt,
                                                                 const double2* __restrict__ stat,
                                                                 const float* __restrict__ w, const float* __restrict__ beta,
                                                                 float* __restrict__ part, float2* __restrict__ gpart) {
  constexpr int kU = 2;
  __shared__ double red[2][kGnThreads * V];
  __shared__ float4 cg[gn_most_groups(V, S)];
  const int b = static_cast<int>(blockIdx.x) / s.nchunk, chunk = static_cast<int>(blockIdx.x) - b * s.nchunk;
  const GnLane l = gn_lane<V>(s.C);
  const GnGroups gr = gn_groups<V>(l, s);
  typedef typename Raw<T, V>::type vec;
  const int c0 = gr.c0 + (l.on ? l.col : 0) * V;
  const int p1 = min(s.HW, (chunk + 1) * s.ppc);
  const T* src = static_cast<const T*>(x.p) + b * x.sb + c0;
  const T* grd = static_cast<const T*>(gy.p) + b * gy.sb + c0;
  int p = chunk * s.ppc + l.row;
  vec rx[kU], rg[kU];
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    rx[u] = *reinterpret_cast<const vec*>(src + min(p + u * l.R, p1 - 1) * x.sp);
    rg[u] = *reinterpret_cast<const vec*>(grd + min(p + u * l.R, p1 - 1) * gy.sp);
  }
  for (int gi = threadIdx.x; gi < gr.ng; gi += kGnThreads) cg[gi] = lds_stat(stat[static_cast<long long>(b) * s.G + gr.g0 + gi]);
  __syncthreads();
  if (l.on) {
    GnCoef<V, S> k;
    load_coef<V, S>(k, cg, w, beta, c0, gr.g0, s);
    double s1[V], s2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.0;
    auto add = [&](const vec& vx, const vec& vg) {
      float v[V], g[V];
      unpack<T, V>(vx, v);
      unpack<T, V>(vg, g);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = (v[i] - k.mh[i / S]) - k.ml[i / S];
        const float gz = grad_z<ACT>(g[i], v[i], d, k.a[i], k.beta[i], stat, w, b, c0 + i, s);
        s1[i] += static_cast<double>(gz);
        s2[i] = fma(static_cast<double>(gz), static_cast<double>(d), s2[i]);
      }
    };
    while (p < p1) {
      vec nx[kU], ng[kU];
      const int pn = p + kU * l.R;
      if (pn < p1) {
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          nx[u] = *reinterpret_cast<const vec*>(src + min(pn + u * l.R, p1 - 1) * x.sp);
          ng[u] = *reinterpret_cast<const vec*>(grd + min(pn + u * l.R, p1 - 1) * gy.sp);
        }
      }
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (p + u * l.R < p1) add(rx[u], rg[u]);
#pragma unroll
      for (int u = 0; u < kU; ++u) rx[u] = nx[u], rg[u] = ng[u];
      p = pn;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      red[0][(l.row * l.cb + l.col) * V + i] = s1[i];
      red[1][(l.row * l.cb + l.col) * V + i] = s2[i];
    }
  }
  __syncthreads();
  const int n = l.cb * V;
  float* out = part + static_cast<long long>(blockIdx.x) * 2 * s.C + gr.c0;
  for (int i = threadIdx.x; i < n; i += kGnThreads) {
    double a = red[0][i], q = red[1][i];
    for (int r = 1; r < l.R; ++r) {
      a += red[0][r * n + i];
      q += red[1][r * n + i];
    }
    q *= static_cast<double>(cg[(gr.c0 + i) / s.cpg - gr.g0].z);
    out[i] = static_cast<float>(a);
    out[s.C + i] = static_cast<float>(q);
    const double wc = w ? static_cast<double>(w[gr.c0 + i]) : 1.0;
    red[0][i] = wc * a;
    red[1][i] = wc * q;
  }
  __syncthreads();
  const int lanes = lanes_per(gr.ng), sub = static_cast<int>(threadIdx.x) & (lanes - 1);
  float2* gout = gpart + (static_cast<long long>(blockIdx.x) * pt.gy + blockIdx.y) * pt.ngb;
  for (int gi = static_cast<int>(threadIdx.x) / lanes; gi < gr.ng; gi += kGnThreads / lanes) {
    const int lo = max((gr.g0 + gi) * s.cpg, gr.c0) - gr.c0, hi = min((gr.g0 + gi + 1) * s.cpg, gr.c1) - gr.c0;
    double a = 0.0, q = 0.0;
    for (int i = lo + sub; i < hi; i += lanes) {
      a += red[0][i];
      q += red[1][i];
    }
    a = wave_part_sum(a, lanes);
    q = wave_part_sum(q, lanes);
    if (sub == 0) gout[gi] = make_float2(static_cast<float>(a), static_cast<float>(q));
  }
}

// g_x; and in the first `nsum` workgroups the sums of the channels' partials over chunks and
// samples (g_w, g_beta), 16 channels x 16 lanes each, so that their chain of loads runs beside the
// map's. Either part may be absent. gpart / gsum: the groups' partials, or joined (gn_join_kernel).
// 32 x 64 x 65 x 65 f32: 18.1 us, 5.7 TB/s.
template <typename T, int V, int S, int ACT, bool NT>
__global__ __launch_bounds__(kGnThreads) void gn_bwd_apply_kernel(GnMap x, GnMap gy, GnShape s, GnParts pt, int nsum,
                                                                  const double2* __restrict__ stat,
                                                                  const float* __restrict__ w, const float* __restrict__ beta,
                                                                  const float* __restrict__ part,
                                                                  const float2* __restrict__ gpart,
                                                                  const double2* __restrict__ gsum, T* __restrict__ gx,
                                                                  float* __restrict__ gw, float* __restrict__ gb) {
  constexpr int kU = 2;
  __shared__ float4 cg[gn_most_groups(V, S)];
  __shared__ float2 kg[gn_most_groups(V, S)];
  if (static_cast<int>(blockIdx.x) < nsum) {
    if (blockIdx.y) return;
    double* red = reinterpret_cast<double*>(cg);  // [2][16][16]
    const int ch = threadIdx.x & 15, lane = threadIdx.x >> 4, c = static_cast<int>(blockIdx.x) * 16 + ch;
    double s1 = 0.0, s2 = 0.0;
    if (c < s.C) {
      const int rows = s.B * s.nchunk;
#pragma unroll 8
      for (int r = lane; r < rows; r += 16) {
        s1 += static_cast<double>(part[static_cast<long long>(r) * 2 * s.C + c]);
        s2 += static_cast<double>(part[static_cast<long long>(r) * 2 * s.C + s.C + c]);
      }
    }
    red[lane * 16 + ch] = s1;
    red[256 + lane * 16 + ch] = s2;
    __syncthreads();
    if (threadIdx.x < 32) {
      const int which = threadIdx.x >> 4;
      double v = 0.0;
      for (int r = 0; r < 16; ++r) v += red[which * 256 + r * 16 + ch];
      float* out = which ? gw : gb;
      if (out && c < s.C) out[c] = static_cast<float>(v);
    }
    return;
  }
  const int blk = static_cast<int>(blockIdx.x) - nsum;
  const int b = blk / s.nchunk, chunk = blk - b * s.nchunk;
  const GnLane l = gn_lane<V>(s.C);
  const GnGroups gr = gn_groups<V>(l, s);
  typedef typename Raw<T, V>::type vec;
  const int c0 = gr.c0 + (l.on ? l.col : 0) * V;
  const int p1 = min(s.HW, (chunk + 1) * s.ppc);
  const T* src = static_cast<const T*>(x.p) + b * x.sb + c0;
  const T* grd = static_cast<const T*>(gy.p) + b * gy.sb + c0;
  int p = chunk * s.ppc + l.row;
  vec rx[kU], rg[kU];
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    rx[u] = *reinterpret_cast<const vec*>(src + min(p + u * l.R, p1 - 1) * x.sp);
    rg[u] = *reinterpret_cast<const vec*>(grd + min(p + u * l.R, p1 - 1) * gy.sp);
  }
  // g_x = a gz - rstd c1 - d rstd^2 c2, d = x - mean
  auto keep = [&](int gi, double a, double q) {
    const double2 st = stat[static_cast<long long>(b) * s.G + gr.g0 + gi];
    const double over = 1.0 / (static_cast<double>(s.HW) * s.cpg);
    cg[gi] = lds_stat(st);
    kg[gi] = make_float2(static_cast<float>(st.y * a * over), static_cast<float>(st.y * st.y * q * over));
  };
  if (gsum) {
    for (int gi = threadIdx.x; gi < gr.ng; gi += kGnThreads) {
      const double2 v = gsum[static_cast<long long>(b) * s.G + gr.g0 + gi];
      keep(gi, v.x, v.y);
    }
  } else {
    const int lanes = pt.lanes, sub = static_cast<int>(threadIdx.x) & (lanes - 1);
    for (int gi = static_cast<int>(threadIdx.x) / lanes; gi < gr.ng; gi += kGnThreads / lanes) {
      double a, q;
      pair_total(gpart, pt, s, b, gr.g0 + gi, sub, lanes, a, q);
      if (sub == 0) keep(gi, a, q);
    }
  }
  __syncthreads();
  if (!l.on) return;
  T* dst = gx + static_cast<long long>(b) * s.HW * s.C + c0;
  GnCoef<V, S> k;
  load_coef<V, S>(k, cg, w, beta, c0, gr.g0, s);
  float2 kk[V / S];
#pragma unroll
  for (int n = 0; n < V / S; ++n) kk[n] = kg[(c0 + n * S) / s.cpg - gr.g0];
  auto put = [&](const vec& vx, const vec& vg, int pp) {
    float v[V], g[V];
    unpack<T, V>(vx, v);
    unpack<T, V>(vg, g);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float d = (v[i] - k.mh[i / S]) - k.ml[i / S];
      const float gz = grad_z<ACT>(g[i], v[i], d, k.a[i], k.beta[i], stat, w, b, c0 + i, s);
      v[i] = fmaf(k.a[i], gz, -fmaf(d, kk[i / S].y, kk[i / S].x));
    }
    put_map<NT>(reinterpret_cast<vec*>(dst + static_cast<long long>(pp) * s.C), pack<T, V>(v));
  };
  while (p < p1) {
    vec nx[kU], ng[kU];
    const int pn = p + kU * l.R;
    if (pn < p1) {
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        nx[u] = *reinterpret_cast<const vec*>(src + min(pn + u * l.R, p1 - 1) * x.sp);
        ng[u] = *reinterpret_cast<const vec*>(grd + min(pn + u * l.R, p1 - 1) * gy.sp);
      }
    }
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (p + u * l.R < p1) put(rx[u], rg[u], p + u * l.R);
#pragma unroll
    for (int u = 0; u < kU; ++u) rx[u] = nx[u], rg[u] = ng[u];
    p = pn;
  }
}

__global__ void gn_zero_kernel(float* a, float* b, int n) {
  const int i = static_cast<int>(blockIdx.x) * 256 + static_cast<int>(threadIdx.x);
  if (i < n) {
    if (a) a[i] = 0.f;
    if (b) b[i] = 0.f;
  }
}

// Chunks per sample, the same in both passes over a map. About 512 workgroups over the samples (1024: 1 x 2048 x
// 129 x 257 bf16 93.3 us for 91.5, forward and backward of 32 x 64 x 65 x 65 f32 63.0 us for 58.8; 256: 2 x 64 x
// 257 x 257 bf16 50.2 us for 45.5), none below 4096 elements (3 x 150 x 33 x 47 f16: 20.4 us, with 16384
// 29.7). Where every workgroup of the second pass would join more than 2048 pairs of a sample, shorter chunks cost
// as much as they save: 16384 elements then (2 x 256 x 65 x 65 bf16: 34.2 us, with 4096 37.1).
// None above 2^18 elements: forward and backward of 600 x 8 x 256 x 256 bf16 991 us for 1075, of 1 x 64 x 2930 x 2930
// 1700 for 1725.
void gn_chunks(GnShape& s) {
  long long want = ceil_div(kGnTarget, s.B);
  const long long all = static_cast<long long>(s.HW) * s.C, inside = kGnJoinInside / 2 / s.G, enough = ceil_div(all, kGnEnough);
  if (want > ceil_div(all, kGnLeast)) want = ceil_div(all, kGnLeast);
  if (want > inside && want > enough) want = inside > enough ? inside : enough;
  if (want < ceil_div(all, kGnMost)) want = ceil_div(all, kGnMost);
  if (want > s.HW) want = s.HW;
  if (want < 1) want = 1;
  s.ppc = static_cast<int>(ceil_div(s.HW, want));
  s.nchunk = static_cast<int>(ceil_div(s.HW, s.ppc));
}

// Elements per vector: 16 B, two elements, or one, by what divides C, the strides and the addresses.
int gn_vec(int elem, int C, std::initializer_list<GnMap> maps, std::initializer_list<const void*> outs) {
  for (int v : {16 / elem, 2, 1}) {
    bool ok = C % v == 0;
    for (const GnMap& m : maps)
      ok = ok && m.sb % v == 0 && m.sp % v == 0 && reinterpret_cast<uintptr_t>(m.p) % (static_cast<size_t>(v) * elem) == 0;
    for (const void* o : outs) ok = ok && reinterpret_cast<uintptr_t>(o) % (static_cast<size_t>(v) * elem) == 0;
    if (ok) return v;
  }
  return 1;
}

template <int N>
using Int = std::integral_constant<int, N>;

// f(type tag, V, S): V is 16 bytes of the type, 2 or 1; S the longest of V, 2 and 1 channels that
// every vector holds runs of inside one group.
template <typename F>
int gn_dispatch(int dtype, int V, int cpg, F f) {
  auto go = [&](auto tag) {
    using T = decltype(tag);
    constexpr int kV = 16 / sizeof(T);
    if (V == 1) return f(tag, Int<1>(), Int<1>());
    if (V == 2) return f(tag, Int<2>(), Int<1>());
    if (cpg % kV == 0) return f(tag, Int<kV>(), Int<kV>());
    if (cpg % 2 == 0) return f(tag, Int<kV>(), Int<2>());
    return f(tag, Int<kV>(), Int<1>());
  };
  if (dtype == PROTOSEG_F32) return go(float{});
  if (dtype == PROTOSEG_BF16) return go(__bf16{});
  return go(_Float16{});
}
template <typename F>
int gn_act(int act, F f) {
  if (act == kGnRelu) return f(Int<kGnRelu>());
  if (act == kGnSigmoid) return f(Int<kGnSigmoid>());
  if (act == kGnSilu) return f(Int<kGnSilu>());
  return f(Int<kGnIdentity>());
}

int gn_shape(GnShape& s, int dtype, int B, int HW, int C, int G, double eps, int act) {
  if (dtype != PROTOSEG_F32 && dtype != PROTOSEG_BF16 && dtype != PROTOSEG_F16)
    return fail(PROTOSEG_ERR_UNSUPPORTED, "group norm dtype %d (f32, bf16 or f16)", dtype);
  if (B < 0 || HW < 0 || C < 1 || G < 1 || C % G != 0)
    return fail(PROTOSEG_ERR_INVALID, "group norm B %d, HW %d, C %d, groups %d (C a multiple of groups)", B, HW, C, G);
  if (!(eps >= 0.0)) return fail(PROTOSEG_ERR_INVALID, "group norm eps %g", eps);
  if (act < kGnIdentity || act > kGnSilu) return fail(PROTOSEG_ERR_INVALID, "group norm activation %d (0..3)", act);
  if (C > (1 << 20) || B > 65535 || HW > (1 << 30))
    return fail(PROTOSEG_ERR_UNSUPPORTED, "group norm B %d, HW %d, C %d (at most 65535, 2^30, 2^20)", B, HW, C);
  s = GnShape{B, HW, C, G, C / G, 0, 0, static_cast<long long>(B) * HW * C * (dtype == PROTOSEG_F32 ? 4 : 2) > kGnStream};
  if (B > 0 && HW > 0) gn_chunks(s);
  return PROTOSEG_OK;
}
int gn_map(const char* name, const GnMap& m, const GnShape& s) {
  if (!m.p) return fail(PROTOSEG_ERR_INVALID, "group norm: %s must be non-null", name);
  if (m.sp < s.C || (s.B > 1 && m.sb < m.sp * (s.HW - 1) + s.C))
    return fail(PROTOSEG_ERR_INVALID, "group norm: %s strides (%lld, %lld) overlap a row of %d channels", name, m.sb, m.sp,
                s.C);
  return PROTOSEG_OK;
}
GnParts gn_parts(const GnShape& s, int V) {
  GnParts pt;
  pt.block_c = kGnThreads * V;
  pt.gy = static_cast<int>(ceil_div(s.C, pt.block_c));
  const long long n = static_cast<long long>(pt.block_c) / s.cpg + 2;
  pt.ngb = static_cast<int>(n < s.G ? n : s.G);
  pt.lanes = lanes_per(pt.ngb);
  return pt;
}
size_t gn_pairs(const GnShape& s, const GnParts& pt) { return static_cast<size_t>(s.B) * s.nchunk * pt.gy * pt.ngb; }
size_t gn_pairs_most(const GnShape& s) {  // of every vector width that a call may choose
  size_t most = 0;
  for (int V : {8, 4, 2, 1}) {
    const size_t n = gn_pairs(s, gn_parts(s, V));
    most = n > most ? n : most;
  }
  return most;
}
bool gn_join_inside(const GnShape& s, const GnParts& pt) { return static_cast<long long>(s.nchunk) * pt.ngb <= kGnJoinInside; }

}  // namespace

}  // namespace protoseg

using namespace protoseg;

extern "C" size_t protoseg_group_norm_workspace_size(int x_dtype, int B, int HW, int C, int groups, int backward) {
  GnShape s;
  if (gn_shape(s, x_dtype, B, HW, C, groups, 0.0, 0) != PROTOSEG_OK || B == 0 || HW == 0) return 0;
  size_t n = gn_pairs_most(s) * (backward ? sizeof(float2) : sizeof(double2));
  if (backward) n += static_cast<size_t>(B) * (groups * sizeof(double2) + static_cast<size_t>(s.nchunk) * 2 * C * sizeof(float));
  return (n + 255) & ~static_cast<size_t>(255);
}

extern "C" int protoseg_group_norm_fwd(const void* x, int x_dtype, int B, int HW, int C, int64_t stride_b,
                                       int64_t stride_pixel, int groups, const float* weight, const float* bias, double eps,
                                       int act_kind, void* y, double* stats, void* workspace, size_t workspace_bytes,
                                       protoseg_stream_t stream) {
  GnShape s;
  if (int e = gn_shape(s, x_dtype, B, HW, C, groups, eps, act_kind)) return e;
  if (B == 0 || HW == 0) return PROTOSEG_OK;
  const GnMap m{x, stride_b, stride_pixel};
  if (int e = gn_map("x", m, s)) return e;
  if (!y || !stats) return fail(PROTOSEG_ERR_INVALID, "group norm: y and stats must be non-null");
  const size_t need = protoseg_group_norm_workspace_size(x_dtype, B, HW, C, groups, 0);
  if (!workspace || workspace_bytes < need)
    return fail(PROTOSEG_ERR_INVALID, "group norm workspace %zu bytes, needs %zu", workspace ? workspace_bytes : 0, need);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int V = gn_vec(x_dtype == PROTOSEG_F32 ? 4 : 2, C, {m}, {y});
  const GnParts pt = gn_parts(s, V);
  double2* part = static_cast<double2*>(workspace);
  double2* stat = reinterpret_cast<double2*>(stats);
  const bool inside = gn_join_inside(s, pt);
  return gn_dispatch(x_dtype, V, s.cpg, [&](auto tag, auto v, auto run) -> int {
    using T = decltype(tag);
    constexpr int kV = decltype(v)::value, kS = decltype(run)::value;
    const dim3 grid(static_cast<unsigned>(B * s.nchunk), static_cast<unsigned>(pt.gy));
    {
      KernelTimer t("gn_stats_kernel", st);
      hipLaunchKernelGGL((gn_stats_kernel<T, kV, kS>), grid, dim3(kGnThreads), 0, st, m, s, pt, part);
    }
    if (!inside)
      hipLaunchKernelGGL((gn_join_kernel<double2, true, T>), dim3(static_cast<unsigned>(groups), static_cast<unsigned>(B)),
                         dim3(kGnThreads), 0, st, m, part, s, pt, eps, stat);
    return gn_act(act_kind, [&](auto act) -> int {
      KernelTimer t("gn_apply_kernel", st);
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(kGnThreads), 0, st, m, s, pt, inside ? part : nullptr, eps, stat, weight, bias,
                           static_cast<T*>(y));
      };
      constexpr bool kMay = kV * sizeof(T) == 16;
      if (kMay && s.stream) go(gn_apply_kernel<T, kV, kS, decltype(act)::value, kMay>);
      else go(gn_apply_kernel<T, kV, kS, decltype(act)::value, false>);
      return check_launch("group norm forward");
    });
  });
}

extern "C" int protoseg_group_norm_bwd(const void* x, const void* g_y, int x_dtype, int B, int HW, int C, int64_t stride_b,
                                       int64_t stride_pixel, int64_t g_stride_b, int64_t g_stride_pixel, int groups,
                                       const float* weight, const float* bias, int act_kind, const double* stats, void* g_x,
                                       float* g_weight, float* g_bias, void* workspace, size_t workspace_bytes,
                                       protoseg_stream_t stream) {
  GnShape s;
  if (int e = gn_shape(s, x_dtype, B, HW, C, groups, 0.0, act_kind)) return e;
  if (!g_x && !g_weight && !g_bias) return PROTOSEG_OK;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (B == 0 || HW == 0) {
    if (!g_weight && !g_bias) return PROTOSEG_OK;
    hipLaunchKernelGGL(gn_zero_kernel, dim3(static_cast<unsigned>(ceil_div(C, 256))), dim3(256), 0, st, g_weight, g_bias, C);
    return check_launch("gn_zero_kernel");
  }
  const GnMap m{x, stride_b, stride_pixel}, mg{g_y, g_stride_b, g_stride_pixel};
  if (int e = gn_map("x", m, s)) return e;
  if (int e = gn_map("g_y", mg, s)) return e;
  if (!stats) return fail(PROTOSEG_ERR_INVALID, "group norm: stats (the forward's) must be non-null");
  const size_t need = protoseg_group_norm_workspace_size(x_dtype, B, HW, C, groups, 1);
  if (!workspace || workspace_bytes < need)
    return fail(PROTOSEG_ERR_INVALID, "group norm workspace %zu bytes, needs %zu", workspace ? workspace_bytes : 0, need);
  const int V = gn_vec(x_dtype == PROTOSEG_F32 ? 4 : 2, C, {m, mg}, {g_x});
  const GnParts pt = gn_parts(s, V);
  double2* gsum = static_cast<double2*>(workspace);
  float2* gpart = reinterpret_cast<float2*>(gsum + static_cast<size_t>(B) * groups);
  float* part = reinterpret_cast<float*>(gpart + gn_pairs(s, pt));
  const double2* stat = reinterpret_cast<const double2*>(stats);
  const bool inside = gn_join_inside(s, pt);
  return gn_dispatch(x_dtype, V, s.cpg, [&](auto tag, auto v, auto run) -> int {
    return gn_act(act_kind, [&](auto act) -> int {
      using T = decltype(tag);
      constexpr int kV = decltype(v)::value, kS = decltype(run)::value, kAct = decltype(act)::value;
      const unsigned nmap = static_cast<unsigned>(B * s.nchunk);
      {
        KernelTimer t("gn_bwd_sums_kernel", st);
        hipLaunchKernelGGL((gn_bwd_sums_kernel<T, kV, kS, kAct>), dim3(nmap, static_cast<unsigned>(pt.gy)), dim3(kGnThreads), 0,
                           st, m, mg, s, pt, stat, weight, bias, part, gpart);
      }
      if (!inside && g_x)
        hipLaunchKernelGGL((gn_join_kernel<float2, false, T>), dim3(static_cast<unsigned>(groups), static_cast<unsigned>(B)),
                           dim3(kGnThreads), 0, st, m, gpart, s, pt, 0.0, gsum);
      const unsigned nsum = g_weight || g_bias ? static_cast<unsigned>(ceil_div(C, 16)) : 0u;
      KernelTimer t("gn_bwd_apply_kernel", st);
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((g_x ? nmap : 0u) + nsum, static_cast<unsigned>(pt.gy)), dim3(kGnThreads), 0, st, m, mg,
                           s, pt, static_cast<int>(nsum), stat, weight, bias, part, gpart, inside ? nullptr : gsum,
                           static_cast<T*>(g_x), g_weight, g_bias);
      };
      constexpr bool kMay = kV * sizeof(T) == 16;
      if (kMay && s.stream) go(gn_bwd_apply_kernel<T, kV, kS, kAct, kMay>);
      else go(gn_bwd_apply_kernel<T, kV, kS, kAct, false>);
      return check_launch("group norm backward");
    });
  });
}
