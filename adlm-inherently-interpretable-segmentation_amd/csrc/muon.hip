// muon.hip — orthogonalising a matrix by Newton-Schulz products, and the optimizer step around it.
//
// X0 = G / (|G|_F + eps), transposed where G is tall, so that X is m x n with m <= n; then `steps` times
//   X <- a X + b (X X^T) X + c (X X^T)^2 X,
// which maps every singular value s of X to a s + b s^3 + c s^5 and keeps its vectors. Each step is a
// polynomial of the m x m Gram matrix A = X X^T, and all of these commute, so a run of steps (a phase)
// works on m x m matrices alone and touches X twice:
//   A = X X^T;   per step  P = a I + b A + c A A,  Q <- P Q,  A <- P A P;   X <- Q X.
// For an m x n matrix that is 3 m^2 n + O(m^3) multiply-adds a phase against 4 m^2 n a step. A's rounding
// (2^-22 of its norm) can leave a zero eigenvalue slightly negative, and every step multiplies it by a^2:
// a phase is cut where that could reach 2^-13 (3 steps at a = 3.4445), and the next one starts from a new
// X X^T, which has no negative eigenvalues. The default five steps run as 3 + 2.
//
// Products run on v_mfma_f32_32x32x16_f16 with every operand held as a pair of f16 values, hi + lo of the
// value times a power of two (22 bits, no overflow: singular values are bounded by the scalar map, checked
// on the host), as lo hi + hi lo + hi hi with f32 accumulation: the error of an f32 product at 1/3 of the
// f16 rate, against 1/16 of it for the f32 MFMA. Steps amplify what a rounding leaves in the small singular
// directions by up to a^steps (485), so a single f16 or bf16 term would lose the result's last 5 to 8 bits.
//
// Kernels: sums of squares (and the momentum update) -> X in pairs -> the products -> the last product's
// epilogue writes the result or updates the parameters. Matrices of one shape form a group; every launch
// covers all groups. Matrices are padded to 64 rows and columns with zeros, so the products have no edges.
#include <math.h>

#include <algorithm>
#include <type_traits>
#include <utility>
#include <vector>

#include "bf16_split.h"
#include "l2_bf16_common.h"
#include "protoseg_device.h"
#include "protoseg_host.h"

namespace protoseg {

namespace {

using bf16l::dma16;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kPad = 64;
constexpr int kMaxGroups = 24, kMaxItems = 32, kMaxSteps = 32;
constexpr float kScale = 1024.f;  // of X, A and T: entries below 16 (checked) stay below 2^14
constexpr long long kBigTiles = 192;
constexpr int kNormThreads = 256, kMaxChunks = 256;
constexpr long long kNormLeast = 16384;  // elements per workgroup of the sums of squares

enum NsOut { kOutF32 = 0, kOutBF16 = 1, kOutF16 = 2, kOutStep = 3 };

// Per matrix, written by ns_load_kernel for the last product: where the result goes.
struct NsTarget {
  void* out;
  float rate, keep;  // kOutStep: p <- keep p - rate O
  int small;         // X0's norm is at most 2^-small (above 0 where eps outweighs |G|)
};

// One shape. Buffers (byte offsets from the workspace; every matrix a hi plane and a lo plane, row-major):
// X0, X1 [count][2][mp][np] f16 at x; A, P, T, Q0, Q1 [count][2][mp][mp] f16 at sq; Gram partials
// [count][split][mp][mp] f32 at part.
struct NsGroup {
  int m, n, mp, np, count, tall;
  int split, first;  // workgroups along the Gram contraction; first workgroup of the group in this launch
  int chunks, target;  // chunks of the sums of squares; index of the first matrix's NsTarget and sums
  long long x, sq, part;
};
struct NsGroups {
  NsGroup g[kMaxGroups];
  int n;
  unsigned char* ws;
  long long targets, sums;  // byte offsets: NsTarget[matrices], double[matrices][kMaxChunks]
};
enum NsBuf { kX0 = 0, kX1 = 1, kA = 2, kP = 3, kT = 4, kQ0 = 5, kQ1 = 6 };

// Equal-shaped matrices at a constant distance: the call's own arrays, or one parameter.
struct NsItem {
  const void* src;
  float *p, *buf;     // kOutStep: parameters and momentum; else p is the output
  long long sb, ob;   // elements from matrix to matrix
  int count, group, index;  // the item's first matrix is the group's `index`
  int first;
  float rate, keep;
};
struct NsItems {
  NsItem it[kMaxItems];
  int n;
};

__device__ __forceinline__ long long x_bytes(const NsGroup& g) { return 4LL * g.mp * g.np; }
__device__ __forceinline__ long long sq_bytes(const NsGroup& g) { return 4LL * g.mp * g.mp; }
__device__ __forceinline__ _Float16* plane_of(const NsGroups& gs, const NsGroup& g, int buf, int mat) {
  const long long o = buf <= kX1 ? g.x + (static_cast<long long>(buf) * g.count + mat) * x_bytes(g)
                                 : g.sq + (static_cast<long long>(buf - kA) * g.count + mat) * sq_bytes(g);
  return reinterpret_cast<_Float16*>(gs.ws + o);
}

struct Pair {
  _Float16 hi, lo;
};
__device__ __forceinline__ Pair split_pair(float v) {
  Pair p;
  p.hi = static_cast<_Float16>(v);
  p.lo = static_cast<_Float16>(v - static_cast<float>(p.hi));
  return p;
}

template <typename T>
__device__ __forceinline__ float src_at(const void* p, long long i) {
  return static_cast<float>(static_cast<const T*>(p)[i]);
}

__device__ __forceinline__ int item_of(const NsItems& its, int blk) {
  int k = 0;
  while (k + 1 < its.n && blk >= its.it[k + 1].first) ++k;
  return k;
}
__device__ __forceinline__ int group_of(const NsGroups& gs, int blk) {
  int k = 0;
  while (k + 1 < gs.n && blk >= gs.g[k + 1].first) ++k;
  return k;
}

// Sum of squares of one chunk of a matrix, in f64 (squares of every f32 stay in range). STEP: the momentum
// B <- mu B + g is written here, and the squares are those of the update U = g + mu B (nesterov) or B.
template <typename T, bool STEP>
__global__ __launch_bounds__(kNormThreads) void ns_norm_kernel(NsGroups gs, NsItems its, float mu, int nesterov) {
  __shared__ double red[kNormThreads / 64];
  const int k = item_of(its, blockIdx.x);
  const NsItem& it = its.it[k];
  const NsGroup& g = gs.g[it.group];
  const int local = static_cast<int>(blockIdx.x) - it.first, mat = local / g.chunks, chunk = local - mat * g.chunks;
  const long long total = static_cast<long long>(g.m) * g.n;
  const long long per = ((total + g.chunks - 1) / g.chunks + 3) & ~3LL;
  const long long e1 = min(total, per * (chunk + 1));
  const T* src = static_cast<const T*>(it.src) + mat * it.sb;
  float* buf = STEP ? it.buf + mat * it.sb : nullptr;
  double s = 0.0;
  constexpr int kU = 4;
  for (long long e = per * chunk + threadIdx.x; e < e1; e += kU * kNormThreads) {
    float v[kU], o[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const long long i = min(e + u * kNormThreads, e1 - 1);
      v[u] = src_at<T>(src, i);
      if constexpr (STEP) o[u] = buf[i];
    }
    pin_batch(v);
    if constexpr (STEP) pin_batch(o);
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (e + u * kNormThreads >= e1) continue;
      float w = v[u];
      if constexpr (STEP) {
        const float nb = fmaf(mu, o[u], v[u]);
        buf[e + u * kNormThreads] = nb;
        w = nesterov ? fmaf(mu, nb, v[u]) : nb;
      }
      s = fma(static_cast<double>(w), static_cast<double>(w), s);
    }
  }
  for (int m = 1; m < 64; m <<= 1) s += __shfl_xor(s, m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double* sums = reinterpret_cast<double*>(gs.ws + gs.sums) + (g.target + it.index + mat) * static_cast<long long>(kMaxChunks);
    sums[chunk] = ((red[0] + red[1]) + red[2]) + red[3];
  }
}

// X0 of one 64 x 64 tile: the (update's) values over their norm, transposed where the matrix is tall, as
// f16 pairs, zeros in the padding.
template <typename T, bool STEP>
__global__ __launch_bounds__(256) void ns_load_kernel(NsGroups gs, NsItems its, float mu, int nesterov, float eps) {
  __shared__ float tile[64][65];
  __shared__ double red[4];
  const int k = item_of(its, blockIdx.x);
  const NsItem& it = its.it[k];
  const NsGroup& g = gs.g[it.group];
  const int tj = g.np / 64, per = (g.mp / 64) * tj;
  const int local = static_cast<int>(blockIdx.x) - it.first, mat = local / per, t = local - mat * per;
  const int i0 = (t / tj) * 64, j0 = (t % tj) * 64;
  const long long row = g.target + it.index + mat;
  const double* sums = reinterpret_cast<const double*>(gs.ws + gs.sums) + row * kMaxChunks;
  double s = static_cast<int>(threadIdx.x) < g.chunks ? sums[threadIdx.x] : 0.0;
  const int rows = g.tall ? g.n : g.m, cols = g.tall ? g.m : g.n;
  const int r0 = g.tall ? j0 : i0, c0 = g.tall ? i0 : j0;
  const T* src = static_cast<const T*>(it.src) + mat * it.sb;
  const float* buf = STEP ? it.buf + mat * it.sb : nullptr;
  const int lc = threadIdx.x & 63, lr = threadIdx.x >> 6;
  float v[16], o[16];
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    const long long i = static_cast<long long>(min(r0 + lr + 4 * u, rows - 1)) * cols + min(c0 + lc, cols - 1);
    v[u] = src_at<T>(src, i);
    if constexpr (STEP) o[u] = buf[i];
  }
  pin_batch(v);
  if constexpr (STEP) pin_batch(o);
  for (int m = 1; m < 64; m <<= 1) s += __shfl_xor(s, m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  const double norm = sqrt(((red[0] + red[1]) + red[2]) + red[3]);
  const double part = norm / (norm + static_cast<double>(eps));
  const int small = part > 0.0 ? max(0, -ilogb(part) - 1) : 0;
  const double inv = scalbn(static_cast<double>(kScale) / (norm + static_cast<double>(eps)), small);
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    float w = v[u];
    if constexpr (STEP) w = nesterov ? fmaf(mu, o[u], v[u]) : o[u];
    const bool in = r0 + lr + 4 * u < rows && c0 + lc < cols;
    tile[lr + 4 * u][lc] = in ? static_cast<float>(static_cast<double>(w) * inv) : 0.f;
  }
  __syncthreads();
  _Float16* hi = plane_of(gs, g, kX0, it.index + mat);
  _Float16* lo = hi + static_cast<long long>(g.mp) * g.np;
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  const int pj = 2 * (threadIdx.x & 31), pi = threadIdx.x >> 5;
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int i = pi + 8 * u;
    const Pair a = split_pair(g.tall ? tile[pj][i] : tile[i][pj]), b = split_pair(g.tall ? tile[pj + 1][i] : tile[i][pj + 1]);
    const long long at = static_cast<long long>(i0 + i) * g.np + j0 + pj;
    *reinterpret_cast<f16x2*>(hi + at) = f16x2{a.hi, b.hi};
    *reinterpret_cast<f16x2*>(lo + at) = f16x2{a.lo, b.lo};
  }
  if (t == 0 && threadIdx.x == 0) {
    NsTarget* tg = reinterpret_cast<NsTarget*>(gs.ws + gs.targets) + row;
    *tg = NsTarget{STEP ? static_cast<void*>(it.p + mat * it.sb) : static_cast<void*>(reinterpret_cast<T*>(it.p) + mat * it.ob),
                   it.rate, it.keep, small};
  }
}

// ---- products ---------------------------------------------------------------------------------------

// One product L R^T of symmetric m x m matrices (or X X^T), and what becomes of it.
struct NsJob {
  int l, r, out;
  int poly;        // out = a I + b A + c (L R^T) instead of L R^T
  float inv, so;   // 1 / (the operands' scales), the result's scale
  int grown, grows;  // X of this phase (and the next) is at most 2^grown (2^grows) times X0: x_shift
};
// X is held times kScale 2^x_shift: where eps outweighs |G|, X0 is far below 1, and a value times kScale
// alone would end in f16's subnormals. The Gram matrix needs no such shift: it is added to a I.
__device__ __forceinline__ int x_shift(const NsTarget& t, int grown) { return max(0, t.small - grown); }
__device__ __forceinline__ const NsTarget& target_of(const NsGroups& gs, const NsGroup& g, int mat) {
  return reinterpret_cast<const NsTarget*>(gs.ws + gs.targets)[g.target + mat];
}
struct NsJobs {
  NsJob j[2];
  int n;
  float a, b, c;   // poly
  int partial;     // groups with split > 1 leave f32 partials (ns_join_kernel makes the result)
};

enum NsMode { kSym = 0, kApply = 1, kWide = 2, kTall = 3 };

// LDS image of a 32-k stage. Operands with k along their rows (NT): [row][32 k], 64-B rows, 16-B chunk c of
// row r at c ^ ((r >> 2) & 3). X as the right operand of Q X has k down its rows: [k][T columns], chunk c
// of row r XORed so that the four k rows of one transposed read start on different banks.
__device__ __forceinline__ constexpr int nt_swz(int r) { return (r >> 2) & 3; }
template <int T>
__device__ __forceinline__ constexpr int kx_swz(int r) {
  return T == 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : ((r >> 1) & 1) << 2;
}

constexpr int kStages = 3;
constexpr int stage_bytes(int T) { return 2 * 2 * T * 64; }  // two operands of two planes

// T x T output tile, 4 waves of (T / 2) x (T / 2). Three LDS stages filled by LDS-DMA two stages ahead of
// the products (one barrier a stage); 3 MFMAs per 32 x 32 x 16 block.
template <int T, int MODE, int OUT>
__global__ __launch_bounds__(256, 1) void ns_product_kernel(NsGroups gs, NsJobs js) {
  constexpr int MI = T / 64, kPieces = T / 32;  // 1-KiB DMA pieces per operand plane and wave
  constexpr int kPlane = T * 64;                // bytes of one operand plane of a stage
  constexpr bool KX = MODE != kSym;             // the right operand's k runs down its rows
  extern __shared__ __attribute__((aligned(16))) unsigned char sm[];
  const unsigned S0 = static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)sm));
  const int lane = threadIdx.x & 63, wave = bf16l::wave_id(), j = lane & 31, h = lane >> 5;
  const NsGroup& g = gs.g[group_of(gs, blockIdx.x)];
  int local = static_cast<int>(blockIdx.x) - g.first;
  const int nt = (g.mp + T - 1) / T, nc = KX ? (g.np + T - 1) / T : nt;
  const int tiles = KX ? nt * nc : nt * (nt + 1) / 2;
  const int splits = MODE == kSym && js.partial ? g.split : 1;
  const int per = tiles * splits * (MODE == kSym ? js.n : 1);
  const int mat = local / per;
  local -= mat * per;
  const int jb = MODE == kSym ? local / (tiles * splits) : 0;
  local -= jb * tiles * splits;
  const int z = local / tiles;
  int tile = local - z * tiles, ti = 0, tc;
  if constexpr (KX) {
    ti = tile % nt;  // row tiles fastest: neighbours share X's columns
    tc = tile / nt;
  } else {
    while (tile >= nt - ti) tile -= nt - ti, ++ti;
    tc = ti + tile;
  }
  NsJob job = js.j[jb];
  if (MODE == kSym && job.l <= kX1) job.inv = ldexpf(job.inv, -2 * x_shift(target_of(gs, g, mat), job.grown));
  const int K = MODE == kSym && job.l <= kX1 ? g.np : g.mp;
  const int i0 = ti * T, c0 = tc * T;
  const _Float16* L = plane_of(gs, g, job.l, mat);
  const _Float16* R = plane_of(gs, g, job.r, mat);
  const unsigned lbytes = static_cast<unsigned>(2LL * g.mp * K);  // one plane
  const unsigned rbytes = KX ? static_cast<unsigned>(2LL * g.mp * g.np) : lbytes;
  const int nst_all = K / 32;
  const int st0 = nst_all * z / splits, nst = nst_all * (z + 1) / splits - st0;

  const int pl = wave >> 1, half = wave & 1;
  const rsrc_t rl = make_rsrc(reinterpret_cast<const unsigned char*>(L) + static_cast<long long>(pl) * lbytes, lbytes);
  const rsrc_t rr = make_rsrc(reinterpret_cast<const unsigned char*>(R) + static_cast<long long>(pl) * rbytes, rbytes);
  unsigned vol[kPieces], vor[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int q = kPieces * half + i, r = 16 * q + (lane >> 2), lc = (lane & 3) ^ nt_swz(r);
    vol[i] = i0 + r < g.mp ? static_cast<unsigned>((static_cast<long long>(i0 + r) * K + 8 * lc) * 2) : kOOB;
    if constexpr (!KX) {
      vor[i] = c0 + r < g.mp ? static_cast<unsigned>((static_cast<long long>(c0 + r) * K + 8 * lc) * 2) : kOOB;
    } else {
      constexpr int kCh = T / 8, kRows = 64 / kCh;  // 16-B chunks a row, k rows a piece
      const int kr = kRows * q + lane / kCh, ch = (lane % kCh) ^ kx_swz<T>(kr);
      vor[i] = c0 + 8 * ch < g.np ? static_cast<unsigned>((static_cast<long long>(kr) * g.np + c0 + 8 * ch) * 2) : kOOB;
    }
  }
  auto issue = [&](int st) __attribute__((always_inline)) {
    const unsigned base = S0 + static_cast<unsigned>((st % kStages) * stage_bytes(T)) +
                          static_cast<unsigned>(pl * kPlane + kPieces * half * 1024);
    const unsigned sl = static_cast<unsigned>(st0 + st) * 64u;
    const unsigned sr = KX ? static_cast<unsigned>(st0 + st) * 64u * static_cast<unsigned>(g.np) : sl;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) dma16(rl, base + static_cast<unsigned>(i * 1024), vol[i], sl);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) dma16(rr, base + static_cast<unsigned>(2 * kPlane + i * 1024), vor[i], sr);
  };

  const int wi = (wave & 1) * (T / 2), wc = (wave >> 1) * (T / 2);
  const int gq = lane >> 4, q4 = (lane >> 2) & 3, p4 = lane & 3;
  // hi hi, and the cross terms apart: they are 2^-11 of it, and a sum of their own takes two of every three
  // roundings out of the large one
  f32x16 acc[MI][MI], cross[MI][MI];
#pragma unroll
  for (int a = 0; a < MI; ++a)
#pragma unroll
    for (int b = 0; b < MI; ++b) acc[a][b] = cross[a][b] = zero16();

  if (nst > 0) issue(0);
  if (nst > 1) issue(1);
  for (int st = 0; st < nst; ++st) {
    // this stage has landed (the next one's 2 kPieces loads of this wave may be in flight), and every
    // read of the stage before it has returned
    if (st + 1 < nst) {
      if constexpr (T == 128) asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
    if (st + 2 < nst) issue(st + 2);  // into the stage that every wave has read before this barrier
    const unsigned sb = S0 + static_cast<unsigned>((st % kStages) * stage_bytes(T));
    f16x8 lf[2][MI][2], rf[2][MI][2];
    auto read_step = [&](int ks) __attribute__((always_inline)) {
#pragma unroll
      for (int a = 0; a < MI; ++a) {
        const int r = wi + 32 * a + j, c = wc + 32 * a + j;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          lf[ks][a][t] = *reinterpret_cast<const __attribute__((address_space(3))) f16x8*>(static_cast<uintptr_t>(
              sb + static_cast<unsigned>(t * kPlane + r * 64 + 16 * ((2 * ks + h) ^ nt_swz(r)))));
          if constexpr (!KX) {
            rf[ks][a][t] = *reinterpret_cast<const __attribute__((address_space(3))) f16x8*>(static_cast<uintptr_t>(
                sb + static_cast<unsigned>((2 + t) * kPlane + c * 64 + 16 * ((2 * ks + h) ^ nt_swz(c)))));
          } else {
            s16x4 v[2];
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              const int kr = 16 * ks + 8 * h + 4 * hf + q4, ch = (wc + 32 * a) / 8 + 2 * (gq & 1) + (p4 >> 1);
              v[hf] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) s16x4*>(
                  static_cast<uintptr_t>(sb + static_cast<unsigned>((2 + t) * kPlane + kr * (2 * T) +
                                                                    16 * (ch ^ kx_swz<T>(kr)) + 8 * (p4 & 1)))));
            }
            rf[ks][a][t] = __builtin_bit_cast(f16x8, __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
          }
        }
      }
    };
    // kTall: the transposed block, so that lanes run along the result's rows
    auto mma = [&](f32x16 (&d)[MI][MI], int ks, int tl, int tr) __attribute__((always_inline)) {
#pragma unroll
      for (int a = 0; a < MI; ++a)
#pragma unroll
        for (int b = 0; b < MI; ++b) {
          if constexpr (MODE == kTall)
            d[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(rf[ks][b][tr], lf[ks][a][tl], d[a][b], 0, 0, 0);
          else
            d[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(lf[ks][a][tl], rf[ks][b][tr], d[a][b], 0, 0, 0);
        }
    };
    // the first 16 k's fragments, then one read of the second's behind each of the first's products
    read_step(0);
    __builtin_amdgcn_sched_barrier(0);
    read_step(1);
    mma(cross, 0, 1, 0);
    mma(cross, 0, 0, 1);
    mma(acc, 0, 0, 0);
#pragma unroll
    for (int k = 0; k < (KX ? 6 : 4) * MI; ++k) {
      if (k < 3 * MI * MI) __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // one MFMA
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);                       // one LDS read
    }
    __builtin_amdgcn_sched_barrier(0);
    mma(cross, 1, 1, 0);
    mma(cross, 1, 0, 1);
    mma(acc, 1, 0, 0);
  }
#pragma unroll
  for (int a = 0; a < MI; ++a)
#pragma unroll
    for (int b = 0; b < MI; ++b) acc[a][b] += cross[a][b];

#pragma unroll
  for (int a = 0; a < MI; ++a)
#pragma unroll
    for (int b = 0; b < MI; ++b) {
      const int ib = i0 + wi + 32 * a, cb = c0 + wc + 32 * b;  // the block's first row and column
      if (ib >= g.mp || cb >= (KX ? g.np : g.mp)) continue;
      if constexpr (MODE == kSym) {
        if (js.partial && g.split > 1) {
          float* dst = reinterpret_cast<float*>(gs.ws + g.part) +
                       (static_cast<long long>(mat) * g.split + z) * g.mp * g.mp + static_cast<long long>(ib) * g.mp + cb + j;
#pragma unroll
          for (int r = 0; r < 16; ++r) dst[static_cast<long long>(acc_row(r, h)) * g.mp] = acc[a][b][r];
          continue;
        }
        float v[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) v[r] = acc[a][b][r] * job.inv;
        const long long psz = static_cast<long long>(g.mp) * g.mp;
        const long long mir = static_cast<long long>(cb + j) * g.mp + ib + 4 * h;  // + 8 q: four rows of column cb + j
        if (job.poly) {
          const _Float16* A = plane_of(gs, g, kA, mat);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f16x4 ah = *reinterpret_cast<const f16x4*>(A + mir + 8 * q), al = *reinterpret_cast<const f16x4*>(A + psz + mir + 8 * q);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = (static_cast<float>(ah[e]) + static_cast<float>(al[e])) * (1.f / kScale);
              v[4 * q + e] = fmaf(js.c, v[4 * q + e], js.b * x);
              if (ib + 8 * q + 4 * h + e == cb + j) v[4 * q + e] += js.a;
            }
          }
        }
        _Float16* hi = plane_of(gs, g, job.out, mat);
        Pair p[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          p[r] = split_pair(v[r] * job.so);
          const long long at = static_cast<long long>(ib + acc_row(r, h)) * g.mp + cb + j;
          hi[at] = p[r].hi;
          hi[psz + at] = p[r].lo;
        }
        if (tc != ti) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            *reinterpret_cast<f16x4*>(hi + mir + 8 * q) = f16x4{p[4 * q].hi, p[4 * q + 1].hi, p[4 * q + 2].hi, p[4 * q + 3].hi};
            *reinterpret_cast<f16x4*>(hi + psz + mir + 8 * q) = f16x4{p[4 * q].lo, p[4 * q + 1].lo, p[4 * q + 2].lo, p[4 * q + 3].lo};
          }
        }
      } else if constexpr (MODE == kApply) {
        _Float16* hi = plane_of(gs, g, job.out, mat);
        const long long psz = static_cast<long long>(g.mp) * g.np;
        const NsTarget& tg = target_of(gs, g, mat);
        const float so = ldexpf(job.inv * job.so, x_shift(tg, job.grows) - x_shift(tg, job.grown));
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const Pair p = split_pair(acc[a][b][r] * so);
          const long long at = static_cast<long long>(ib + acc_row(r, h)) * g.np + cb + j;
          hi[at] = p.hi;
          hi[psz + at] = p.lo;
        }
      } else {
        const NsTarget tg = target_of(gs, g, mat);
        const int shift = x_shift(tg, job.grown);
        const int rb = MODE == kTall ? cb : ib, col = (MODE == kTall ? ib : cb) + j;
        const int rows = MODE == kTall ? g.n : g.m, cols = MODE == kTall ? g.m : g.n;
        if (col >= cols) continue;
        float old[16];
        if constexpr (OUT == kOutStep) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            old[r] = static_cast<const float*>(tg.out)[static_cast<long long>(min(rb + acc_row(r, h), rows - 1)) * cols + col];
          pin_batch(old);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int row = rb + acc_row(r, h);
          if (row >= rows) continue;
          const float v = ldexpf(acc[a][b][r] * job.inv, -shift);
          const long long at = static_cast<long long>(row) * cols + col;
          if constexpr (OUT == kOutF32) static_cast<float*>(tg.out)[at] = v;
          if constexpr (OUT == kOutBF16) static_cast<__bf16*>(tg.out)[at] = static_cast<__bf16>(v);
          if constexpr (OUT == kOutF16) static_cast<_Float16*>(tg.out)[at] = static_cast<_Float16>(v);
          if constexpr (OUT == kOutStep) static_cast<float*>(tg.out)[at] = fmaf(-tg.rate, v, tg.keep * old[r]);
        }
      }
    }
}

// The partials of a split Gram product joined in a fixed order: a workgroup takes one 32 x 32 block on or
// above the diagonal, each wave every fourth split, and stores it with its mirror image.
__global__ __launch_bounds__(256) void ns_join_kernel(NsGroups gs, float inv, int grown) {
  __shared__ float red[3][16][64];
  const NsGroup& g = gs.g[group_of(gs, blockIdx.x)];
  const int nb = g.mp / 32, per = nb * (nb + 1) / 2;
  const int local = static_cast<int>(blockIdx.x) - g.first, mat = local / per;
  int blk = local - mat * per, bi = 0;
  while (blk >= nb - bi) blk -= nb - bi, ++bi;
  const int bc = bi + blk, lane = threadIdx.x & 63, wave = bf16l::wave_id(), j = lane & 31, h = lane >> 5;
  const long long psz = static_cast<long long>(g.mp) * g.mp;
  const float* src = reinterpret_cast<const float*>(gs.ws + g.part) + static_cast<long long>(mat) * g.split * psz +
                     static_cast<long long>(32 * bi + 4 * h) * g.mp + 32 * bc + j;
  float v[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) v[r] = 0.f;
#pragma unroll 4
  for (int z = wave; z < g.split; z += 4) {
#pragma unroll
    for (int r = 0; r < 16; ++r) v[r] += src[z * psz + static_cast<long long>(row_of(r)) * g.mp];
  }
  if (wave) {
#pragma unroll
    for (int r = 0; r < 16; ++r) red[wave - 1][r][lane] = v[r];
  }
  __syncthreads();
  if (wave) return;
  inv = ldexpf(inv, -2 * x_shift(target_of(gs, g, mat), grown));
  _Float16* hi = plane_of(gs, g, kA, mat);
  Pair p[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    p[r] = split_pair((((v[r] + red[0][r][lane]) + red[1][r][lane]) + red[2][r][lane]) * inv);
    const long long at = static_cast<long long>(32 * bi + acc_row(r, h)) * g.mp + 32 * bc + j;
    hi[at] = p[r].hi;
    hi[psz + at] = p[r].lo;
  }
  if (bc != bi) {
    const long long mir = static_cast<long long>(32 * bc + j) * g.mp + 32 * bi + 4 * h;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      *reinterpret_cast<f16x4*>(hi + mir + 8 * q) = f16x4{p[4 * q].hi, p[4 * q + 1].hi, p[4 * q + 2].hi, p[4 * q + 3].hi};
      *reinterpret_cast<f16x4*>(hi + psz + mir + 8 * q) = f16x4{p[4 * q].lo, p[4 * q + 1].lo, p[4 * q + 2].lo, p[4 * q + 3].lo};
    }
  }
}

// ---- host -------------------------------------------------------------------------------------------

struct NsPlan {
  int phases[kMaxSteps], nphase;
  float a, b, c;
  float sp[kMaxSteps], sq[kMaxSteps];  // scales of P and of Q after each step
  int grown[kMaxSteps + 1];            // X before each phase is at most 2^grown times X0
};

float scale_for(double most) {  // the largest power of two up to kScale that keeps `most` below 2^15
  float s = kScale;
  while (s > 1e-3f && most * s > 32768.0) s *= 0.5f;
  return s;
}

// Phases, and scales that keep every f16 in range: the singular values of X0 are at most 1 (the Frobenius
// norm is), the scalar map carries that bound on, and P and Q are functions of the Gram matrix.
int ns_plan(NsPlan& pl, int steps, float a, float b, float c) {
  if (steps < 1 || steps > kMaxSteps) return fail(PROTOSEG_ERR_INVALID, "orthogonalize steps %d (1..%d)", steps, kMaxSteps);
  if (!(std::isfinite(a) && std::isfinite(b) && std::isfinite(c)))
    return fail(PROTOSEG_ERR_INVALID, "orthogonalize coefficients (%g, %g, %g)", a, b, c);
  pl.a = a, pl.b = b, pl.c = c;
  int longest = 1;  // 2^-22 a^(2 (L - 1)) <= 2^-13
  for (double f = 1.0; longest < 3 && f * a * a <= 512.0; ++longest) f *= static_cast<double>(a) * a;
  pl.nphase = (steps + longest - 1) / longest;
  for (int p = 0, left = steps; p < pl.nphase; ++p) {
    pl.phases[p] = (left + pl.nphase - p - 1) / (pl.nphase - p);
    left -= pl.phases[p];
  }
  constexpr int kGrid = 2048;
  double most = 1.001, factor = 1.0;
  for (int p = 0, st = 0; p < pl.nphase; ++p) {
    std::vector<double> s(kGrid + 1), q(kGrid + 1, 1.0);
    pl.grown[p] = static_cast<int>(ceil(log2(factor)));
    for (int i = 0; i <= kGrid; ++i) s[i] = most * i / kGrid;
    double next = 0.0, qm = 0.0;
    for (int k = 0; k < pl.phases[p]; ++k, ++st) {
      double pm = 0.0;
      qm = 0.0;
      next = 0.0;
      for (int i = 0; i <= kGrid; ++i) {
        const double l = s[i] * s[i], pv = a + b * l + c * l * l;
        s[i] *= pv;
        q[i] *= pv;
        pm = fmax(pm, fabs(pv));
        qm = fmax(qm, fabs(q[i]));
        next = fmax(next, fabs(s[i]));
      }
      if (!(next <= 3.9))
        return fail(PROTOSEG_ERR_UNSUPPORTED,
                    "orthogonalize coefficients (%g, %g, %g) let singular values grow to %g within %d steps (below 4 is served)",
                    a, b, c, next, st + 1);
      pl.sp[st] = scale_for(1.02 * pm);
      pl.sq[st] = scale_for(1.02 * qm);
    }
    most = 1.01 * next;
    factor = fmax(1.0, factor * 1.02 * qm);
    pl.grown[p + 1] = static_cast<int>(ceil(log2(factor)));
  }
  return PROTOSEG_OK;
}

struct NsMatrix {
  int rows, cols, count;
};

int pad_of(long long v) { return static_cast<int>((v + kPad - 1) / kPad * kPad); }

// Groups of `mats` (at most kMaxGroups shapes, equal ones joined) and their buffers; returns the bytes in
// all. which[i]: the group of mats[i]; index[i]: its first matrix there.
size_t ns_layout(NsGroups& gs, const std::vector<NsMatrix>& mats, std::vector<int>* which, std::vector<int>* index) {
  gs = NsGroups{};
  for (size_t i = 0; i < mats.size(); ++i) {
    int k = 0;
    while (k < gs.n && !((gs.g[k].tall ? gs.g[k].n : gs.g[k].m) == mats[i].rows && (gs.g[k].tall ? gs.g[k].m : gs.g[k].n) == mats[i].cols)) ++k;
    if (k == gs.n) {
      NsGroup& g = gs.g[gs.n++];
      g = NsGroup{};
      g.tall = mats[i].rows > mats[i].cols;
      g.m = g.tall ? mats[i].cols : mats[i].rows;
      g.n = g.tall ? mats[i].rows : mats[i].cols;
      g.mp = pad_of(g.m);
      g.np = pad_of(g.n);
    }
    if (which) {
      which->push_back(k);
      index->push_back(gs.g[k].count);
    }
    gs.g[k].count += mats[i].count;
  }
  // the matrices with the most work a tile first, so that a launch does not end on them
  std::vector<int> order(gs.n), place(gs.n);
  for (int k = 0; k < gs.n; ++k) order[k] = k;
  std::stable_sort(order.begin(), order.end(), [&](int p, int q) { return gs.g[p].mp > gs.g[q].mp; });
  const NsGroups was = gs;
  for (int k = 0; k < gs.n; ++k) gs.g[k] = was.g[order[k]], place[order[k]] = k;
  if (which)
    for (int& w : *which) w = place[w];
  long long tiles = 0;  // 64 x 64 Gram tiles in all
  for (int k = 0; k < gs.n; ++k) tiles += static_cast<long long>(gs.g[k].count) * (gs.g[k].mp / 64) * (gs.g[k].mp / 64 + 1) / 2;
  long long at = 0, total = 0;
  auto take = [&](long long bytes) {
    const long long o = at;
    at += (bytes + 255) & ~255LL;
    return o;
  };
  for (int k = 0; k < gs.n; ++k) {
    NsGroup& g = gs.g[k];
    // The Gram contraction is split where it is long (a split is at least 8 stages) and the launch has
    // fewer tiles than the chip has places for, or its chain of stages would outlast everything else's.
    const long long stages = g.np / 32;
    long long split = 384 / (tiles < 1 ? 1 : tiles);
    const long long chain = (stages + 63) / 64, most = stages / 8;
    if (split < chain) split = chain;
    if (split > most) split = most;
    if (split > 32) split = 32;
    g.split = static_cast<int>(split < 1 ? 1 : split);
    const long long e = static_cast<long long>(g.m) * g.n, ch = ceil_div(e, kNormLeast);
    g.chunks = static_cast<int>(ch < kMaxChunks ? ch : kMaxChunks);
    g.target = static_cast<int>(total);
    total += g.count;
    g.x = take(2LL * g.count * 4 * g.mp * g.np);
    g.sq = take(5LL * g.count * 4 * g.mp * g.mp);
    g.part = g.split > 1 ? take(4LL * g.count * g.split * g.mp * g.mp) : 0;
  }
  gs.targets = take(total * static_cast<long long>(sizeof(NsTarget)));
  gs.sums = take(total * kMaxChunks * 8LL);
  return static_cast<size_t>(at);
}

int ns_check(int rows, int cols) {
  if (rows < 0 || cols < 0) return fail(PROTOSEG_ERR_INVALID, "orthogonalize: %d x %d matrix", rows, cols);
  const long long m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
  if (static_cast<long long>(pad_of(m)) * pad_of(n) > (1LL << 29) || m > 16384)
    return fail(PROTOSEG_ERR_UNSUPPORTED, "orthogonalize: %d x %d matrix (at most 2^29 padded elements, 16384 in the smaller dimension)",
                rows, cols);
  return PROTOSEG_OK;
}

// first[] of every group for a launch that gives each of its matrices per(g) workgroups; the grid.
template <typename F>
long long ns_grid(NsGroups& gs, F per) {
  long long blocks = 0;
  for (int k = 0; k < gs.n; ++k) {
    gs.g[k].first = static_cast<int>(blocks < (1LL << 30) ? blocks : (1LL << 30));
    blocks += per(gs.g[k]) * gs.g[k].count;
  }
  return blocks;
}
int ns_blocks_ok(long long blocks) {
  return blocks < (1LL << 30) ? PROTOSEG_OK : fail(PROTOSEG_ERR_UNSUPPORTED, "orthogonalize: %lld workgroups", blocks);
}

template <int T, int MODE, int OUT>
int ns_launch(NsGroups gs, const NsJobs& js, hipStream_t st) {
  const long long blocks = ns_grid(gs, [&](const NsGroup& g) -> long long {
    const long long nt = ceil_div(g.mp, T);
    if (MODE == kSym) return nt * (nt + 1) / 2 * js.n * (js.partial ? g.split : 1);
    if ((MODE == kWide && g.tall) || (MODE == kTall && !g.tall)) return 0;
    return nt * ceil_div(g.np, T);
  });
  if (blocks == 0) return PROTOSEG_OK;
  if (int e = ns_blocks_ok(blocks)) return e;
  constexpr size_t lds = kStages * stage_bytes(T);
  if (int e = ensure_lds<ns_product_kernel<T, MODE, OUT>, lds>()) return e;
  KernelTimer t("ns_product_kernel", st);
  hipLaunchKernelGGL((ns_product_kernel<T, MODE, OUT>), dim3(static_cast<unsigned>(blocks)), dim3(256), lds, st, gs, js);
  return check_launch("ns_product_kernel");
}

// All products of a prepared X0, ending in the targets.
template <int T, int OUT>
int ns_products(NsGroups gs, const NsPlan& pl, hipStream_t st) {
  int x = kX0, step = 0;
  auto sym = [&](std::initializer_list<NsJob> jobs, int partial = 0) {
    NsJobs js{};
    for (const NsJob& j : jobs) js.j[js.n++] = j;
    js.a = pl.a, js.b = pl.b, js.c = pl.c, js.partial = partial;
    return ns_launch<T, kSym, kOutF32>(gs, js, st);
  };
  bool split = false;
  for (int k = 0; k < gs.n; ++k) split = split || gs.g[k].split > 1;
  for (int p = 0; p < pl.nphase; ++p) {
    if (int e = sym({NsJob{x, x, kA, 0, 1.f / (kScale * kScale), kScale, pl.grown[p]}}, split)) return e;
    if (split) {
      NsGroups js = gs;
      const long long blocks = ns_grid(js, [](const NsGroup& g) -> long long {
        const long long nb = g.mp / 32;
        return g.split > 1 ? nb * (nb + 1) / 2 : 0;
      });
      hipLaunchKernelGGL(ns_join_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, js, 1.f / kScale, pl.grown[p]);
      if (int e = check_launch("ns_join_kernel")) return e;
    }
    int q = kQ0;
    float sq = 0.f;
    for (int k = 0; k < pl.phases[p]; ++k, ++step) {
      const float sp = pl.sp[step];
      const int pb = k == 0 ? kQ0 : kP;  // the first P is Q
      if (int e = sym({NsJob{kA, kA, pb, 1, 1.f / (kScale * kScale), sp}})) return e;
      const bool more = k + 1 < pl.phases[p];
      const NsJob mul{pb, kA, kT, 0, 1.f / (sp * kScale), kScale};
      if (k == 0) {
        sq = sp;
        if (more)
          if (int e = sym({mul})) return e;
      } else {
        const int qn = q == kQ0 ? kQ1 : kQ0;
        const NsJob acc{pb, q, qn, 0, 1.f / (sp * sq), pl.sq[step]};
        if (int e = more ? sym({mul, acc}) : sym({acc})) return e;
        q = qn;
        sq = pl.sq[step];
      }
      if (more)
        if (int e = sym({NsJob{kT, pb, kA, 0, 1.f / (sp * kScale), kScale}})) return e;
    }
    NsJobs js{};
    js.n = 1;
    if (p + 1 < pl.nphase) {
      const int xn = x == kX0 ? kX1 : kX0;
      js.j[0] = NsJob{q, x, xn, 0, 1.f / (sq * kScale), kScale, pl.grown[p], pl.grown[p + 1]};
      if (int e = ns_launch<T, kApply, kOutF32>(gs, js, st)) return e;
      x = xn;
    } else {
      js.j[0] = NsJob{q, x, x, 0, 1.f / (sq * kScale), 1.f, pl.grown[p]};
      if (int e = ns_launch<T, kWide, OUT>(gs, js, st)) return e;
      if (int e = ns_launch<T, kTall, OUT>(gs, js, st)) return e;
    }
  }
  return PROTOSEG_OK;
}

template <int OUT>
int ns_products(const NsGroups& gs, const NsPlan& pl, hipStream_t st) {
  long long tiles = 0;
  for (int k = 0; k < gs.n; ++k) {
    const long long nt = ceil_div(gs.g[k].mp, 128);
    tiles += nt * (nt + 1) / 2 * gs.g[k].count;
  }
  return tiles >= kBigTiles ? ns_products<128, OUT>(gs, pl, st) : ns_products<64, OUT>(gs, pl, st);
}

// Sums of squares and X0 of all items, kMaxItems a launch.
template <typename T, bool STEP>
int ns_load(const NsGroups& gs, const std::vector<NsItem>& items, float mu, int nesterov, float eps, hipStream_t st) {
  for (int pass = 0; pass < 2; ++pass)
    for (size_t i0 = 0; i0 < items.size(); i0 += kMaxItems) {
      NsItems its{};
      long long blocks = 0;
      for (size_t i = i0; i < items.size() && i < i0 + kMaxItems; ++i) {
        NsItem it = items[i];
        const NsGroup& g = gs.g[it.group];
        it.first = static_cast<int>(blocks);
        blocks += static_cast<long long>(it.count) * (pass ? static_cast<long long>(g.mp / 64) * (g.np / 64) : g.chunks);
        if (int e = ns_blocks_ok(blocks)) return e;
        its.it[its.n++] = it;
      }
      if (pass == 0)
        hipLaunchKernelGGL((ns_norm_kernel<T, STEP>), dim3(static_cast<unsigned>(blocks)), dim3(kNormThreads), 0, st, gs, its, mu, nesterov);
      else
        hipLaunchKernelGGL((ns_load_kernel<T, STEP>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, gs, its, mu, nesterov, eps);
      if (int e = check_launch(pass ? "ns_load_kernel" : "ns_norm_kernel")) return e;
    }
  return PROTOSEG_OK;
}

}  // namespace

}  // namespace protoseg

using namespace protoseg;

extern "C" size_t protoseg_orthogonalize_workspace_size(int count, int rows, int cols) {
  if (count <= 0 || rows <= 0 || cols <= 0 || ns_check(rows, cols) != PROTOSEG_OK) return 0;
  NsGroups gs;
  return ns_layout(gs, {NsMatrix{rows, cols, count}}, nullptr, nullptr);
}

extern "C" int protoseg_orthogonalize(const void* g, int dtype, int count, int rows, int cols, int64_t stride, int steps, float a,
                                      float b, float c, float eps, void* out, void* workspace, size_t workspace_bytes,
                                      protoseg_stream_t stream) {
  if (dtype != PROTOSEG_F32 && dtype != PROTOSEG_BF16 && dtype != PROTOSEG_F16)
    return fail(PROTOSEG_ERR_UNSUPPORTED, "orthogonalize dtype %d (f32, bf16 or f16)", dtype);
  if (count < 0) return fail(PROTOSEG_ERR_INVALID, "orthogonalize: %d matrices", count);
  if (int e = ns_check(rows, cols)) return e;
  if (!(eps >= 0.f)) return fail(PROTOSEG_ERR_INVALID, "orthogonalize eps %g", eps);
  NsPlan pl;
  if (int e = ns_plan(pl, steps, a, b, c)) return e;
  if (count == 0 || rows == 0 || cols == 0) return PROTOSEG_OK;
  const long long size = static_cast<long long>(rows) * cols;
  if (!g || !out) return fail(PROTOSEG_ERR_INVALID, "orthogonalize: matrices and result must be non-null");
  if (count > 1 && stride < size) return fail(PROTOSEG_ERR_INVALID, "orthogonalize: matrices %lld elements apart overlap", static_cast<long long>(stride));
  NsGroups gs;
  const size_t need = ns_layout(gs, {NsMatrix{rows, cols, count}}, nullptr, nullptr);
  if (!workspace || workspace_bytes < need)
    return fail(PROTOSEG_ERR_INVALID, "orthogonalize workspace %zu bytes, needs %zu", workspace ? workspace_bytes : 0, need);
  gs.ws = static_cast<unsigned char*>(workspace);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const std::vector<NsItem> items{NsItem{g, static_cast<float*>(out), nullptr, stride, size, count, 0, 0, 0, 0.f, 0.f}};
  auto go = [&](auto tag, auto kind) -> int {
    if (int e = ns_load<decltype(tag), false>(gs, items, 0.f, 0, eps, st)) return e;
    return ns_products<decltype(kind)::value>(gs, pl, st);
  };
  if (dtype == PROTOSEG_F32) return go(float{}, std::integral_constant<int, kOutF32>());
  if (dtype == PROTOSEG_BF16) return go(__bf16{}, std::integral_constant<int, kOutBF16>());
  return go(_Float16{}, std::integral_constant<int, kOutF16>());
}

namespace {
// A call's matrices in runs of at most kMaxGroups shapes (one launch covers a run).
struct MuonRun {
  std::vector<NsMatrix> mats;
  std::vector<int> from;  // tensor of the call
};
int muon_runs(std::vector<MuonRun>& runs, int n, const int32_t* rows, const int32_t* cols) {
  std::vector<std::pair<int, int>> shapes;
  for (int i = 0; i < n; ++i) {
    if (int e = ns_check(rows[i], cols[i])) return e;
    if (rows[i] == 0 || cols[i] == 0) continue;
    size_t k = 0;
    while (k < shapes.size() && shapes[k] != std::make_pair(rows[i], cols[i])) ++k;
    if (k == shapes.size()) shapes.emplace_back(rows[i], cols[i]);
    if (k / kMaxGroups == runs.size()) runs.emplace_back();
    runs[k / kMaxGroups].mats.push_back(NsMatrix{rows[i], cols[i], 1});
    runs[k / kMaxGroups].from.push_back(i);
  }
  return PROTOSEG_OK;
}
}  // namespace

extern "C" size_t protoseg_muon_workspace_size(int n_tensors, const int32_t* rows, const int32_t* cols) {
  std::vector<MuonRun> runs;
  if (n_tensors <= 0 || !rows || !cols || muon_runs(runs, n_tensors, rows, cols) != PROTOSEG_OK) return 0;
  size_t most = 0;
  for (const MuonRun& r : runs) {
    NsGroups gs;
    const size_t n = ns_layout(gs, r.mats, nullptr, nullptr);
    most = n > most ? n : most;
  }
  return most;
}

extern "C" int protoseg_muon_step(int n_tensors, float* const* params, const float* const* grads, float* const* momentum_bufs,
                                  const int32_t* rows, const int32_t* cols, float momentum, int nesterov, float lr,
                                  float weight_decay, int scale_kind, int steps, float a, float b, float c, float eps,
                                  void* workspace, size_t workspace_bytes, protoseg_stream_t stream) {
  if (n_tensors < 0 || (n_tensors > 0 && (!params || !grads || !momentum_bufs || !rows || !cols)))
    return fail(PROTOSEG_ERR_INVALID, "muon: %d tensors, pointer and size arrays must be non-null", n_tensors);
  if (!(momentum >= 0.f && momentum < 1.f) || !(eps >= 0.f) || !std::isfinite(lr) || !std::isfinite(weight_decay))
    return fail(PROTOSEG_ERR_INVALID, "muon: momentum %g in [0, 1), eps %g >= 0, lr %g, weight decay %g", momentum, eps, lr, weight_decay);
  if (scale_kind != 0 && scale_kind != 1) return fail(PROTOSEG_ERR_INVALID, "muon scale kind %d (0 or 1)", scale_kind);
  NsPlan pl;
  if (int e = ns_plan(pl, steps, a, b, c)) return e;
  std::vector<MuonRun> runs;
  if (int e = muon_runs(runs, n_tensors, rows, cols)) return e;
  size_t need = 0;
  for (const MuonRun& r : runs) {
    for (int i : r.from)
      if (!params[i] || !grads[i] || !momentum_bufs[i]) return fail(PROTOSEG_ERR_INVALID, "muon tensor %d: null pointer", i);
    NsGroups gs;
    const size_t n = ns_layout(gs, r.mats, nullptr, nullptr);
    need = n > need ? n : need;
  }
  if (need && (!workspace || workspace_bytes < need))
    return fail(PROTOSEG_ERR_INVALID, "muon workspace %zu bytes, needs %zu", workspace ? workspace_bytes : 0, need);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  for (const MuonRun& run : runs) {
    NsGroups gs;
    std::vector<int> which, index;
    ns_layout(gs, run.mats, &which, &index);
    gs.ws = static_cast<unsigned char*>(workspace);
    std::vector<NsItem> items;
    for (size_t k = 0; k < run.mats.size(); ++k) {
      const int i = run.from[k];
      const double r = rows[i], q = cols[i];
      const double scale = scale_kind == 0 ? sqrt(r > q ? r / q : 1.0) : 0.2 * sqrt(r > q ? r : q);
      items.push_back(NsItem{grads[i], params[i], momentum_bufs[i], 0, 0, 1, which[k], index[k], 0, static_cast<float>(lr * scale),
                             static_cast<float>(1.0 - static_cast<double>(lr) * weight_decay)});
    }
    if (int e = ns_load<float, true>(gs, items, momentum, nesterov ? 1 : 0, eps, st)) return e;
    if (int e = ns_products<kOutStep>(gs, pl, st)) return e;
  }
  return PROTOSEG_OK;
}
