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
// a phase is cut after two steps at most (one where the result would lose by it, ns_longest), or where that
// could reach 2^-13, and the next one starts from a new X X^T, which has no negative eigenvalues. The default
// five steps run as 2 + 2 + 1 or one by one.
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
#include <exception>
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
typedef float f32x4 __attribute__((ext_vector_type(4)));

typedef __attribute__((address_space(3))) f16x8 lds_f16x8;
typedef __attribute__((address_space(3))) f16x4 lds_f16x4;
typedef __attribute__((address_space(3))) _Float16 lds_f16;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) float lds_f32;
template <typename P>
__device__ __forceinline__ P* lds_ptr(unsigned at) {
  return reinterpret_cast<P*>(static_cast<uintptr_t>(at));
}

constexpr int kPad = 64;
constexpr int kMaxGroups = 24, kMaxItems = 32, kMaxSteps = 32;
constexpr float kScale = 1024.f;  // of X, A and T: entries below 16 (checked) stay below 2^14
constexpr long long kThinTiles = 256;  // ns_thin_kernel's tiles at most: it has one workgroup a CU (22 matrices of 256, 792 tiles: 313 us for 204)
// Up to so many 64 x 64 tiles (one a CU), of contractions of 8 stages or more, the two halves of a contraction run
// beside each other (one matrix of 1024 x 1024: 236 us for 248; 60 of 128 x 500, 4 stages: 170 us for 164).
constexpr long long kHalvesTiles = 256, kHalvesStages = 8;
constexpr long long kApplyTiles = 384;  // from so many 128 x 128 tiles of Q X on, they beat 64 x 64 ones (backbone: 1406 us for 1468)
constexpr int kNormThreads = 256, kMaxChunks = 256;
constexpr long long kNormLeast = 16384;  // elements per workgroup of the sums of squares

enum NsOut { kOutF32 = 0, kOutBF16 = 1, kOutF16 = 2, kOutStep = 3 };

// Per matrix, written by ns_load_kernel for the last product: where the result goes.
struct NsTarget {
  void* out;
  float rate, keep;  // kOutStep: p <- keep p - rate O
  int small;         // X0's norm is at most 2^-small (above 0 where eps outweighs |G|)
};

// One shape. Buffers (byte offsets from the workspace): X0, X1 [count][mp][np] pairs at x; A, P, T, Q0, Q1
// [count][mp][mp] pairs at sq; Gram partials [count][split][mp][mp] f32 at part. Pairs are row-major, 32 hi
// values and their 32 lo values in turn: a 32-k stage of a row is one 128-B line. (With hi and lo in planes
// of their own it was two half lines and twice the requests to L2, at the same time.)
struct NsGroup {
  int m, n, mp, np, count, tall;
  int kind;          // which of a call's two plans its steps follow (ns_kind)
  int split;         // workgroups along the Gram contraction
  int chunks, target;  // chunks of the sums of squares; index of the first matrix's NsTarget and sums
  long long x, sq, part;
};
struct NsGroups {
  NsGroup g[kMaxGroups];
  int first[kMaxGroups];  // first workgroup of each group in this launch (no workgroup's from n on)
  int n;
  int thin;  // the symmetric products run on ns_thin_kernel
  unsigned char* ws;
  long long targets, sums;  // byte offsets: NsTarget[matrices], double[matrices][kMaxChunks]
};
enum NsBuf { kX0 = 0, kX1 = 1, kA = 2, kP = 3, kT = 4, kQ0 = 5, kQ1 = 6 };

// Equal-shaped matrices at a constant distance: the call's own arrays, or one parameter.
struct NsItem {
  const void* src;
  float *p, *buf;     // kOutStep: parameters and momentum; else p is the output
  long long sb, ob;   // elements from matrix to matrix
  int count, rows, cols;
  int group, index;  // the item's first matrix is the group's `index` (ns_small_kernel has no groups)
  float rate, keep;
};
struct NsItems {
  NsItem it[kMaxItems];
  int first[kMaxItems];
  int n;
};

__device__ __forceinline__ long long x_bytes(const NsGroup& g) { return 4LL * g.mp * g.np; }
__device__ __forceinline__ long long sq_bytes(const NsGroup& g) { return 4LL * g.mp * g.mp; }
__device__ __forceinline__ _Float16* pairs_of(const NsGroups& gs, const NsGroup& g, int buf, int mat) {
  const long long o = buf <= kX1 ? g.x + (static_cast<long long>(buf) * g.count + mat) * x_bytes(g)
                                 : g.sq + (static_cast<long long>(buf - kA) * g.count + mat) * sq_bytes(g);
  return reinterpret_cast<_Float16*>(gs.ws + o);
}

// hi of element (row, col) of a matrix of `ld` columns; lo is kLo further.
constexpr int kLo = 32;
__device__ __forceinline__ long long at_pair(int row, int col, int ld) {
  return static_cast<long long>(row) * (2 * ld) + (col >> 5) * 64 + (col & 31);
}

struct Pair {
  _Float16 hi, lo;
};
// The compiler may join a product in v with the conversion to f16 and round it once there, and twice where it forms
// hi again for lo: two different his. Products by powers of two are exact; others are pinned first.
__device__ __forceinline__ float pinned(float v) {
  asm volatile("" : "+v"(v));
  return v;
}
__device__ __forceinline__ Pair split_pair(float v) {
  Pair p;
  p.hi = static_cast<_Float16>(v);
  p.lo = static_cast<_Float16>(v - static_cast<float>(p.hi));
  return p;
}

// A 32 x 32 block of a product (lane: one column, acc_row's rows) as pairs at `dst`, the block's first hi.
// (8-B stores after a 4 x 4 exchange within quads measured 10 to 15 % slower over whole launches: the
// exchange is vector work of every wave.)
__device__ __forceinline__ void store_block(_Float16* dst, const Pair (&p)[16], int ld, int lane) {
  const int j = lane & 31, h = lane >> 5;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const long long at = static_cast<long long>(acc_row(r, h)) * (2 * ld) + j;
    dst[at] = p[r].hi;
    dst[at + kLo] = p[r].lo;
  }
}

// The block transposed in place, through 4 KiB of LDS of the wave's own (both sides on distinct banks).
// (Stored from the registers it came in, 8 B down each column, a block took 4 times the cache lines.)
__device__ __forceinline__ void mirror_block(Pair (&p)[16], unsigned lds, int lane) {
  const int j = lane & 31, h = lane >> 5;
  wave_lds_fence();  // the sums that a caller read from here, of a type that the stores below need not wait for
#pragma unroll
  for (int r = 0; r < 16; ++r)
    *reinterpret_cast<__attribute__((address_space(3))) unsigned*>(
        static_cast<uintptr_t>(lds + static_cast<unsigned>(4 * (32 * j + (acc_row(r, h) ^ j))))) =
        static_cast<unsigned>(__builtin_bit_cast(uint16_t, p[r].hi)) |
        (static_cast<unsigned>(__builtin_bit_cast(uint16_t, p[r].lo)) << 16);
  wave_lds_fence();
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int row = acc_row(r, h);
    const unsigned v = *reinterpret_cast<const __attribute__((address_space(3))) unsigned*>(
        static_cast<uintptr_t>(lds + static_cast<unsigned>(4 * (32 * row + (j ^ row)))));
    p[r].hi = __builtin_bit_cast(_Float16, static_cast<uint16_t>(v));
    p[r].lo = __builtin_bit_cast(_Float16, static_cast<uint16_t>(v >> 16));
  }
  wave_lds_fence();
}

template <typename T>
__device__ __forceinline__ float src_at(const void* p, long long i) {
  return static_cast<float>(static_cast<const T*>(p)[i]);
}

// The group (item) of a workgroup: a binary search, since each probe is a scalar load that the next one
// waits for (22 matrices of 256 x 1024: 204 us for 211 in order). first[] is an array of its own, two lines of
// the arguments and not one per group.
template <int N>
__device__ __forceinline__ int place_of(const int (&first)[N], int blk) {
  int k = 0;
#pragma unroll
  for (int step = 16; step; step >>= 1)
    if (k + step < N && blk >= first[k + step < N ? k + step : 0]) k += step;
  return k;
}

// A launch gives group g n = per matrix x count workgroups, rounded up to a multiple of 8, and XCD x (which runs
// the workgroups i % 8 == x) the x-th eighth of them in order: neighbouring tiles of a matrix share operands,
// and an XCD finds them in its own 4 MiB L2 (22 matrices of 256 x 1024: 204 us for 236). -1: past the end.
__device__ __forceinline__ int xcd_local(int b, int n) {
  const int chunk = (n + 7) >> 3, i = (b & 7) * chunk + (b >> 3);
  return i < n && (b >> 3) < chunk ? i : -1;
}

// Sum of squares of one chunk of a matrix, in f64 (squares of every f32 stay in range). Bound by memory: 122 us for
// 47e6 elements' gradients and momentum, 4.6 TB/s. STEP: the momentum
// B <- mu B + g is written here, and the squares are those of the update U = g + mu B (nesterov) or B.
template <typename T, bool STEP>
__global__ __launch_bounds__(kNormThreads) void ns_norm_kernel(NsGroups gs, NsItems its, float mu, int nesterov) {
  __shared__ double red[kNormThreads / 64];
  const int k = place_of(its.first, blockIdx.x);
  const NsItem& it = its.it[k];
  const NsGroup& g = gs.g[it.group];
  const int local = static_cast<int>(blockIdx.x) - its.first[k], mat = local / g.chunks, chunk = local - mat * g.chunks;
  const long long total = static_cast<long long>(g.m) * g.n;
  const long long per = ((total + g.chunks - 1) / g.chunks + 3) & ~3LL;
  const long long e1 = min(total, per * (chunk + 1));
  const T* src = static_cast<const T*>(it.src) + mat * it.sb;
  float* buf = STEP ? it.buf + mat * it.sb : nullptr;
  double s = 0.0;
  constexpr int kU = 4;
  typedef T vec4 __attribute__((ext_vector_type(4)));
  long long e = per * chunk;
  if (((reinterpret_cast<uintptr_t>(src) & (sizeof(vec4) - 1)) | (reinterpret_cast<uintptr_t>(buf) & 15)) == 0) {
    for (; e + kU * 4 * kNormThreads <= e1; e += kU * 4 * kNormThreads) {  // 4 elements a load
      vec4 v[kU];
      f32x4 o[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const long long i = e + 4 * (u * kNormThreads + static_cast<int>(threadIdx.x));
        v[u] = *reinterpret_cast<const vec4*>(src + i);
        if constexpr (STEP) o[u] = *reinterpret_cast<const f32x4*>(buf + i);
      }
#pragma unroll
      for (int u = 0; u < kU; ++u) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float x = static_cast<float>(v[u][c]);
          float w = x;
          if constexpr (STEP) {
            o[u][c] = fmaf(mu, o[u][c], x);
            w = nesterov ? fmaf(mu, o[u][c], x) : o[u][c];
          }
          s = fma(static_cast<double>(w), static_cast<double>(w), s);
        }
        if constexpr (STEP)
          *reinterpret_cast<f32x4*>(buf + e + 4 * (u * kNormThreads + static_cast<int>(threadIdx.x))) = o[u];
      }
    }
  }
  for (e += threadIdx.x; e < e1; e += kU * kNormThreads) {
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

// What takes an update's value to X0's: ldexpf(w, e) f, kScale 2^small / (norm + eps) as a factor in [0.5, 1)
// and a power of two. The power comes first: it takes the largest values to some 2^11 for any norm, also from
// f32's subnormals, where a product would round to few bits.
struct NsScale {
  float f;
  int e, small;
};
__device__ __forceinline__ NsScale scale_of(double squares, float eps) {
  const double norm = sqrt(squares), all = norm + static_cast<double>(eps), part = norm / all;
  NsScale s;
  if (all == 0.0) return NsScale{0.f, 0, 0};  // a zero matrix without eps: zeros
  s.small = part > 0.0 ? max(0, -ilogb(part) - 1) : 0;
  s.f = static_cast<float>(frexp(static_cast<double>(kScale) / all, &s.e));
  s.e += s.small;
  return s;
}

// X0 of one 64 x 64 tile: the (update's) values over their norm, transposed where the matrix is tall, as
// f16 pairs, zeros in the padding. 102 us for 47e6 elements: 5.5 TB/s, the reads from the last-level cache.
template <typename T, bool STEP>
__global__ __launch_bounds__(256) void ns_load_kernel(NsGroups gs, NsItems its, float mu, int nesterov, float eps) {
  __shared__ float tile[64][65];
  __shared__ double red[4];
  const int k = place_of(its.first, blockIdx.x);
  const NsItem& it = its.it[k];
  const NsGroup& g = gs.g[it.group];
  const int tj = g.np / 64, per = (g.mp / 64) * tj;
  const int local = static_cast<int>(blockIdx.x) - its.first[k], mat = local / per, t = local - mat * per;
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
  const NsScale sc = scale_of(((red[0] + red[1]) + red[2]) + red[3], eps);
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    float w = v[u];
    if constexpr (STEP) w = nesterov ? fmaf(mu, o[u], v[u]) : o[u];
    const bool in = r0 + lr + 4 * u < rows && c0 + lc < cols;
    tile[lr + 4 * u][lc] = in ? ldexpf(w, sc.e) * sc.f : 0.f;
  }
  __syncthreads();
  _Float16* dst = pairs_of(gs, g, kX0, it.index + mat);
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  const int pj = 2 * (threadIdx.x & 31), pi = threadIdx.x >> 5;
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int i = pi + 8 * u;
    const Pair a = split_pair(g.tall ? tile[pj][i] : tile[i][pj]), b = split_pair(g.tall ? tile[pj + 1][i] : tile[i][pj + 1]);
    const long long at = at_pair(i0 + i, j0 + pj, g.np);
    *reinterpret_cast<f16x2*>(dst + at) = f16x2{a.hi, b.hi};
    *reinterpret_cast<f16x2*>(dst + at + kLo) = f16x2{a.lo, b.lo};
  }
  if (t == 0 && threadIdx.x == 0) {
    NsTarget* tg = reinterpret_cast<NsTarget*>(gs.ws + gs.targets) + row;
    *tg = NsTarget{STEP ? static_cast<void*>(it.p + mat * it.sb) : static_cast<void*>(reinterpret_cast<T*>(it.p) + mat * it.ob),
                   it.rate, it.keep, sc.small};
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
struct NsPart {    // what a group does in a launch (n = 0: nothing)
  NsJob j[2];
  int n;
  int partial;     // groups with split > 1 leave f32 partials (ns_join_kernel makes the result)
};
// Per group, not per kind: read with the group itself, where a second level of loads from the arguments costs every
// launch 1.3 us (22 matrices of 256 x 1024: 210 us for 187).
struct NsJobs {
  NsPart of[kMaxGroups];
  float a, b, c;   // poly
};

enum NsMode { kSym = 0, kApply = 1, kWide = 2, kTall = 3 };

// LDS image of a 32-k stage, rows of hi and lo as in memory, 16-B chunk c of row r at c ^ swizzle(r).
// Operands with k along their rows (NT): 128-B rows, and 16 lanes read one chunk of 16 consecutive rows. X as
// the right operand of Q X has k down its rows (4 T bytes each), and a transposed read takes 64 B of 4
// consecutive rows.
__device__ __forceinline__ constexpr int nt_swz(int r) { return (r >> 1) & 7; }
__device__ __forceinline__ constexpr int kx_swz(int r) { return (r & 3) << 2; }

// Stages of the ring: three workgroups a CU at 64, two at 128. Deeper rings measured slower (5 at 64: +3 %, 4 at
// 128: +5 %): a workgroup beside another hides more than a stage further ahead.
constexpr int ring_of(int T) { return T == 128 ? 2 : 3; }
constexpr int stage_bytes(int T) { return 2 * T * 128; }

// Waits until at most min(later, MOST) stages of PER loads each are in flight, then for the other waves.
template <int PER, int MOST>
__device__ __forceinline__ void stage_wait(int later) {
  if constexpr (MOST > 0) {
    if (later < MOST) {
      stage_wait<PER, MOST - 1>(later);
      return;
    }
  }
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(PER * MOST) : "memory");
}

// T x T output tile, 4 waves of (T / 2) x (T / 2), 3 MFMAs per 32 x 32 x 16 block. LDS-DMA fills a ring of
// stages of 32 k, ring_of - 1 ahead of the products, with one barrier a stage. In the step over a ResNet-101's
// convolutions (109 matrices, 47e6 elements) the Gram product takes 109 us, Q X 142 us, Q X with the parameters'
// update 177 us, a product of squares 30 us: 524, 677, 545 and 410 TFLOP/s of f16, where a large library product
// reaches 1100. No single unit is full in the Gram product: a stage of a 64 x 64 tile is 192 cycles of MFMA on each
// SIMD (23 us in all) and 384 of LDS (32 KiB read and 16 KiB written at 128 B a cycle: 45 us), and L2 serves 10 TB/s;
// without MFMAs 84 % of its time stayed, without the loads 67 %: it waits for loads, with three workgroups a CU. At
// 128 x 128 LDS is read half as often, but the symmetric products would compute a fifth more and leave half the
// chip's places empty at the end (measured slower).
// G = 2: a second set of 4 waves takes the second half of the stages and hands its sums over at the end.
template <int T, int MODE, int OUT, int G = 1>
__global__ __launch_bounds__(256 * G, 160 * 1024 / (G * ring_of(T) * stage_bytes(T))) void ns_product_kernel(NsGroups gs, NsJobs js) {
  static_assert(G == 1 || (G == 2 && T == 64 && MODE == kSym), "sums are handed over as one block a wave");
  constexpr int MI = T / 64, kPieces = T / 32;  // 1-KiB DMA pieces per operand and wave
  constexpr int kOperand = T * 128;             // bytes of one operand of a stage
  constexpr int kStages = ring_of(T);
  constexpr bool KX = MODE != kSym;             // the right operand's k runs down its rows
  extern __shared__ __attribute__((aligned(16))) unsigned char sm[];
  const int lane = threadIdx.x & 63, wave = bf16l::wave_id() & 3, half = G == 2 ? bf16l::wave_id() >> 2 : 0, j = lane & 31, h = lane >> 5;
  const unsigned S0 = static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)sm)) +
                      static_cast<unsigned>(half * kStages * stage_bytes(T));
  const int gi = place_of(gs.first, blockIdx.x);
  const NsGroup& g = gs.g[gi];
  const int nt = (g.mp + T - 1) / T, nc = KX ? (g.np + T - 1) / T : nt;
  const int tiles = KX ? nt * nc : nt * (nt + 1) / 2;
  const NsPart& jp = js.of[gi];
  const int splits = MODE == kSym && jp.partial ? g.split : 1;
  const int per = tiles * splits * (MODE == kSym ? jp.n : 1);
  int local = xcd_local(static_cast<int>(blockIdx.x) - gs.first[gi], per * g.count);
  if (local < 0) return;
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
  NsJob job = jp.j[jb];
  if (MODE == kSym && job.l <= kX1) job.inv = ldexpf(job.inv, -2 * x_shift(target_of(gs, g, mat), job.grown));
  const int K = MODE == kSym && job.l <= kX1 ? g.np : g.mp;
  const int i0 = ti * T, c0 = tc * T;
  const _Float16* L = pairs_of(gs, g, job.l, mat);
  const _Float16* R = pairs_of(gs, g, job.r, mat);
  const unsigned lbytes = static_cast<unsigned>(4LL * g.mp * K), rbytes = KX ? static_cast<unsigned>(x_bytes(g)) : lbytes;
  const int nst_all = K / 32;
  const int z0 = nst_all * z / splits, z1 = nst_all * (z + 1) / splits;
  const int turns = (z1 - z0 + G - 1) / G, st0 = z0 + half * turns, nst = G == 2 && half ? z1 - st0 : turns;  // turns or one less

  const rsrc_t rl = make_rsrc(L, lbytes), rr = make_rsrc(R, rbytes);
  unsigned vol[kPieces], vor[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int q = kPieces * wave + i, r = 8 * q + (lane >> 3), ch = (lane & 7) ^ nt_swz(r);
    vol[i] = i0 + r < g.mp ? static_cast<unsigned>(static_cast<long long>(i0 + r) * K * 4 + 16 * ch) : kOOB;
    if constexpr (!KX) {
      vor[i] = c0 + r < g.mp ? static_cast<unsigned>(static_cast<long long>(c0 + r) * K * 4 + 16 * ch) : kOOB;
    } else {
      constexpr int kCh = T / 4, kRows = 64 / kCh;  // 16-B chunks a row, k rows a piece
      const int kr = kRows * q + lane / kCh, cx = (lane % kCh) ^ kx_swz(kr);
      vor[i] = c0 + 4 * cx < g.np ? static_cast<unsigned>((static_cast<long long>(kr) * g.np + c0) * 4 + 16 * cx) : kOOB;
    }
  }
  auto issue = [&](int st) __attribute__((always_inline)) {
    const unsigned base = S0 + static_cast<unsigned>((st % kStages) * stage_bytes(T) + kPieces * wave * 1024);
    const unsigned sl = static_cast<unsigned>(st0 + st) * 128u;
    const unsigned sr = KX ? static_cast<unsigned>(st0 + st) * 128u * static_cast<unsigned>(g.np) : sl;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) dma16(rl, base + static_cast<unsigned>(i * 1024), vol[i], sl);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) dma16(rr, base + static_cast<unsigned>(kOperand + i * 1024), vor[i], sr);
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

  for (int st = 0; st < kStages - 1 && st < nst; ++st) issue(st);
  for (int st = 0; st < turns; ++st) {
    // this stage has landed (what was issued after it may be in flight), and every read of the stage before
    // it has returned
    stage_wait<2 * kPieces, kStages - 2>(nst - 1 - st);
    if (st + kStages - 1 < nst) issue(st + kStages - 1);  // into the stage that every wave has read before this barrier
    if (G == 2 && st >= nst) break;  // the barrier above was the last
    const unsigned sb = S0 + static_cast<unsigned>((st % kStages) * stage_bytes(T));
    f16x8 lf[2][MI][2], rf[2][MI][2];
    auto read_step = [&](int ks) __attribute__((always_inline)) {
#pragma unroll
      for (int a = 0; a < MI; ++a) {
        const int r = wi + 32 * a + j, c = wc + 32 * a + j;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          lf[ks][a][t] = *reinterpret_cast<const __attribute__((address_space(3))) f16x8*>(static_cast<uintptr_t>(
              sb + static_cast<unsigned>(r * 128 + 16 * ((4 * t + 2 * ks + h) ^ nt_swz(r)))));
          if constexpr (!KX) {
            rf[ks][a][t] = *reinterpret_cast<const __attribute__((address_space(3))) f16x8*>(static_cast<uintptr_t>(
                sb + static_cast<unsigned>(kOperand + c * 128 + 16 * ((4 * t + 2 * ks + h) ^ nt_swz(c)))));
          } else {
            s16x4 v[2];
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              const int kr = 16 * ks + 8 * h + 4 * hf + q4, ch = (wc + 32 * a) / 4 + 4 * t + 2 * (gq & 1) + (p4 >> 1);
              v[hf] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) s16x4*>(
                  static_cast<uintptr_t>(sb + static_cast<unsigned>(kOperand + kr * (4 * T) + 16 * (ch ^ kx_swz(kr)) + 8 * (p4 & 1)))));
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
  if constexpr (G == 2) {
    lds_f32* sums = lds_ptr<lds_f32>(S0 - static_cast<unsigned>(half * kStages * stage_bytes(T))) + wave * 1024 + lane;
    __syncthreads();  // no stage is read any more
    if (half) {
#pragma unroll
      for (int r = 0; r < 16; ++r) sums[64 * r] = acc[0][0][r];
    }
    __syncthreads();
    if (half) return;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[0][0][r] += sums[64 * r];
  }

#pragma unroll
  for (int a = 0; a < MI; ++a)
#pragma unroll
    for (int b = 0; b < MI; ++b) {
      const int ib = i0 + wi + 32 * a, cb = c0 + wc + 32 * b;  // the block's first row and column
      if (ib >= g.mp || cb >= (KX ? g.np : g.mp)) continue;
      if constexpr (MODE == kSym) {
        if (jp.partial && g.split > 1) {
          float* dst = reinterpret_cast<float*>(gs.ws + g.part) +
                       (static_cast<long long>(mat) * g.split + z) * g.mp * g.mp + static_cast<long long>(ib) * g.mp + cb + j;
#pragma unroll
          for (int r = 0; r < 16; ++r) dst[static_cast<long long>(acc_row(r, h)) * g.mp] = acc[a][b][r];
          continue;
        }
        float v[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) v[r] = acc[a][b][r] * job.inv;
        if (job.poly) {
          const _Float16* A = pairs_of(gs, g, kA, mat) + at_pair(ib, cb, g.mp) + j;
          _Float16 ah[16], al[16];
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            ah[r] = A[static_cast<long long>(acc_row(r, h)) * (2 * g.mp)];
            al[r] = A[static_cast<long long>(acc_row(r, h)) * (2 * g.mp) + kLo];
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float x = (static_cast<float>(ah[r]) + static_cast<float>(al[r])) * (1.f / kScale);
            v[r] = fmaf(js.c, v[r], js.b * x);
            if (ib + acc_row(r, h) == cb + j) v[r] += js.a;
          }
        }
        _Float16* hi = pairs_of(gs, g, job.out, mat);
        Pair p[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] = split_pair(v[r] * job.so);
        store_block(hi + at_pair(ib, cb, g.mp), p, g.mp, lane);
        if (tc != ti) {
          mirror_block(p, S0 + static_cast<unsigned>((nst % kStages) * stage_bytes(T) + wave * 4096), lane);
          store_block(hi + at_pair(cb, ib, g.mp), p, g.mp, lane);
        }
      } else if constexpr (MODE == kApply) {
        _Float16* hi = pairs_of(gs, g, job.out, mat);
        const NsTarget& tg = target_of(gs, g, mat);
        const float so = ldexpf(job.inv * job.so, x_shift(tg, job.grows) - x_shift(tg, job.grown));
        Pair p[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] = split_pair(acc[a][b][r] * so);
        store_block(hi + at_pair(ib, cb, g.np), p, g.np, lane);
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

// The symmetric products of few matrices: a 32 x 32 tile a workgroup, whose 4 waves take every fourth 32-k stage
// (a ring of 4 stages of its own each, no barrier in the loop) and then a quarter of the tile's rows each. A
// launch of few tiles is a chain of load latencies along k: a quarter of it, and four times the workgroups. A
// launch takes 6.8 us at m = 512 (64 x 64 tiles: 10) and 5.0 at m = 128, of which 2.4 are the launch alone.
constexpr int kThinRing = 4, kThinStage = 2 * 32 * 128;
template <int MOST>
__device__ __forceinline__ void thin_wait(int later) {  // at most min(later, MOST) stages of 8 loads in flight
  if constexpr (MOST > 0) {
    if (later < MOST) {
      thin_wait<MOST - 1>(later);
      return;
    }
  }
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(8 * MOST) : "memory");
}
__global__ __launch_bounds__(256, 1) void ns_thin_kernel(NsGroups gs, NsJobs js) {
  extern __shared__ __attribute__((aligned(16))) unsigned char sm[];
  const unsigned S0 = static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)sm));
  const int lane = threadIdx.x & 63, wave = bf16l::wave_id(), j = lane & 31, h = lane >> 5;
  const int gi = place_of(gs.first, blockIdx.x);
  const NsGroup& g = gs.g[gi];
  const NsPart& jp = js.of[gi];
  const int nt = g.mp / 32, tiles = nt * (nt + 1) / 2, splits = jp.partial ? g.split : 1, per = tiles * splits * jp.n;
  int local = xcd_local(static_cast<int>(blockIdx.x) - gs.first[gi], per * g.count);
  if (local < 0) return;
  const int mat = local / per;
  local -= mat * per;
  const int jb = local / (tiles * splits);
  local -= jb * tiles * splits;
  const int z = local / tiles;
  int tile = local - z * tiles, ti = 0;
  while (tile >= nt - ti) tile -= nt - ti, ++ti;
  const int i0 = 32 * ti, c0 = 32 * (ti + tile);
  NsJob job = jp.j[jb];
  if (job.l <= kX1) job.inv = ldexpf(job.inv, -2 * x_shift(target_of(gs, g, mat), job.grown));
  const int K = job.l <= kX1 ? g.np : g.mp, nst_all = K / 32;
  const int st0 = nst_all * z / splits, nst = nst_all * (z + 1) / splits - st0;
  const int mine = (nst - wave + 3) / 4;  // stages st0 + wave + 4 t
  const unsigned bytes = static_cast<unsigned>(4LL * g.mp * K);
  const rsrc_t rl = make_rsrc(pairs_of(gs, g, job.l, mat), bytes), rr = make_rsrc(pairs_of(gs, g, job.r, mat), bytes);
  unsigned vol[4], vor[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 8 * i + (lane >> 3), ch = (lane & 7) ^ nt_swz(r);
    vol[i] = static_cast<unsigned>(static_cast<long long>(i0 + r) * K * 4 + 16 * ch);
    vor[i] = static_cast<unsigned>(static_cast<long long>(c0 + r) * K * 4 + 16 * ch);
  }
  const unsigned W0 = S0 + static_cast<unsigned>(wave * kThinRing * kThinStage);
  auto issue = [&](int t) __attribute__((always_inline)) {
    const unsigned base = W0 + static_cast<unsigned>((t % kThinRing) * kThinStage);
    const unsigned so = static_cast<unsigned>(st0 + wave + 4 * t) * 128u;
#pragma unroll
    for (int i = 0; i < 4; ++i) dma16(rl, base + static_cast<unsigned>(i * 1024), vol[i], so);
#pragma unroll
    for (int i = 0; i < 4; ++i) dma16(rr, base + static_cast<unsigned>(4096 + i * 1024), vor[i], so);
  };
  for (int t = 0; t < kThinRing && t < mine; ++t) issue(t);
  f32x16 acc = zero16(), cross = zero16();
  for (int t = 0; t < mine; ++t) {
    thin_wait<kThinRing - 1>(mine - 1 - t);
    const unsigned sb = W0 + static_cast<unsigned>((t % kThinRing) * kThinStage);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      f16x8 lf[2], rf[2];
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2) {
        const unsigned at = sb + static_cast<unsigned>(j * 128 + 16 * ((4 * t2 + 2 * ks + h) ^ nt_swz(j)));
        lf[t2] = *reinterpret_cast<const __attribute__((address_space(3))) f16x8*>(static_cast<uintptr_t>(at));
        rf[t2] = *reinterpret_cast<const __attribute__((address_space(3))) f16x8*>(static_cast<uintptr_t>(at + 4096));
      }
      cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(lf[1], rf[0], cross, 0, 0, 0);
      cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(lf[0], rf[1], cross, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(lf[0], rf[0], acc, 0, 0, 0);
    }
    if (t + kThinRing < mine) {
      wave_lds_fence();  // the reads of this place have returned
      issue(t + kThinRing);
    }
  }
  // this wave's place holds nothing any more: its sums, then everyone's rows 8 wave + 4 h .. + 3 of column j
  float* mysum = reinterpret_cast<float*>(sm + wave * kThinRing * kThinStage);
#pragma unroll
  for (int r = 0; r < 16; ++r) mysum[64 * r + lane] = acc[r] + cross[r];
  __syncthreads();
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) v[e] += reinterpret_cast<const float*>(sm + w * kThinRing * kThinStage)[64 * (4 * wave + e) + lane];
  }
  const int row = i0 + 8 * wave + 4 * h, col = c0 + j;
  if (jp.partial && g.split > 1) {
    float* dst = reinterpret_cast<float*>(gs.ws + g.part) +
                 (static_cast<long long>(mat) * g.split + z) * g.mp * g.mp + static_cast<long long>(row) * g.mp + col;
#pragma unroll
    for (int e = 0; e < 4; ++e) dst[static_cast<long long>(e) * g.mp] = v[e];
    return;
  }
  const long long at = at_pair(row, col, g.mp), mir = at_pair(col, row, g.mp);
  const _Float16* A = pairs_of(gs, g, kA, mat);
  _Float16* out = pairs_of(gs, g, job.out, mat);
  f16x4 hi, lo;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] *= job.inv;
    if (job.poly) {
      const long long a = at + static_cast<long long>(e) * (2 * g.mp);
      const float x = (static_cast<float>(A[a]) + static_cast<float>(A[a + kLo])) * (1.f / kScale);
      v[e] = fmaf(js.c, v[e], js.b * x);
      if (row + e == col) v[e] += js.a;
    }
    const Pair p = split_pair(v[e] * job.so);
    hi[e] = p.hi;
    lo[e] = p.lo;
    out[at + static_cast<long long>(e) * (2 * g.mp)] = p.hi;
    out[at + static_cast<long long>(e) * (2 * g.mp) + kLo] = p.lo;
  }
  if (tile) {
    *reinterpret_cast<f16x4*>(out + mir) = hi;
    *reinterpret_cast<f16x4*>(out + mir + kLo) = lo;
  }
}

// The partials of a split Gram product joined in a fixed order (8.0 us in the 109 matrices' step, bound by reading
// them): a workgroup takes one 32 x 32 block on or
// above the diagonal, each wave every fourth split, and stores it with its mirror image.
__global__ __launch_bounds__(256) void ns_join_kernel(NsGroups gs, NsJobs js) {
  __shared__ float red[3][16][64];
  const int gi = place_of(gs.first, blockIdx.x);
  const NsGroup& g = gs.g[gi];
  const int nb = g.mp / 32, per = nb * (nb + 1) / 2;
  const int local = xcd_local(static_cast<int>(blockIdx.x) - gs.first[gi], per * g.count);
  if (local < 0) return;
  const int mat = local / per;
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
  const NsJob& job = js.of[gi].j[0];
  const float inv = ldexpf(job.inv * job.so, -2 * x_shift(target_of(gs, g, mat), job.grown));
  _Float16* hi = pairs_of(gs, g, kA, mat);
  Pair p[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) p[r] = split_pair((((v[r] + red[0][r][lane]) + red[1][r][lane]) + red[2][r][lane]) * inv);
  store_block(hi + at_pair(32 * bi, 32 * bc, g.mp), p, g.mp, lane);
  if (bc != bi) {
    mirror_block(p, static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)&red[0][0][0])), lane);
    store_block(hi + at_pair(32 * bc, 32 * bi, g.mp), p, g.mp, lane);
  }
}

// ---- one workgroup per matrix ---------------------------------------------------------------------------

// Matrices of up to 64 rows and 384 columns (padded), whose phases are single steps: norm, X and all products of one
// matrix in one workgroup, X and four 64 x 64 matrices in LDS (64 * 384 * 4 + 4 * 16 KiB = 160 KiB). Such a matrix is
// a chain of 15 products of about 2 us each, and a launch each costs 4 to 5 us: 361 x 64 f32 takes 41 us. What
// bounds it is the chain of LDS reads, MFMAs, LDS writes and barriers (a step 6.7 us, load and store 7.5), so the
// blocks of a square lie on as many waves: 12 for 10 blocks.
constexpr int kSmallM = 64, kSmallN = 384, kSmallThreads = 768;
constexpr int kSmallSquare = 64 * 256;  // bytes of a 64 x 64 matrix of pairs

struct NsPlan {
  int phases[kMaxSteps], nphase;
  float a, b, c;
  float sp[kMaxSteps], sq[kMaxSteps];  // scales of P and of Q after each step
  int grown[kMaxSteps + 1];            // X before each phase is at most 2^grown times X0
};

// LDS rows of pairs (32 hi, 32 lo, ...), pitch a multiple of 256 B; 16-B chunk c of row r at c ^ sm_swz(r):
// 16 rows of one chunk lie on distinct banks, and so do 64 B of 4 consecutive rows (a transposed read).
// The lo chunk of hi chunk c is c + 4, at the hi chunk's address ^ 64.
__device__ __forceinline__ constexpr int sm_swz(int r) { return ((r & 3) << 2) | ((r >> 2) & 3); }
__device__ __forceinline__ unsigned sm_at(unsigned base, int pitch, int r, int chunk) {
  return base + static_cast<unsigned>(r * pitch + 16 * (chunk ^ sm_swz(r)));
}
__device__ __forceinline__ int chunk_of(int c) { return (c >> 5) * 8 + ((c & 31) >> 3); }  // of column c's hi
// The 32x32x16 fragment of rows r0 + (lane & 31), k = 16 step + 8 (lane >> 5) .. + 7.
__device__ __forceinline__ void sm_rows(f16x8 (&f)[2], unsigned base, int pitch, int r0, int step, int lane) {
  const unsigned at = sm_at(base, pitch, r0 + (lane & 31), (step >> 1) * 8 + 2 * (step & 1) + (lane >> 5));
  f[0] = *lds_ptr<lds_f16x8>(at);
  f[1] = *lds_ptr<lds_f16x8>(at ^ 64);
}
// The 16x16x32 fragment of rows r0 + (lane & 15), k = 32 step + 8 (lane >> 4) .. + 7.
__device__ __forceinline__ void sm_rows16(f16x8 (&f)[2], unsigned base, int r0, int step, int lane) {
  const unsigned at = sm_at(base, 256, r0 + (lane & 15), step * 8 + (lane >> 4));
  f[0] = *lds_ptr<lds_f16x8>(at);
  f[1] = *lds_ptr<lds_f16x8>(at ^ 64);
}
// sm_rows of columns c0 + (lane & 31), with k down the rows.
__device__ __forceinline__ void sm_cols(f16x8 (&f)[2], unsigned base, int pitch, int c0, int step, int lane) {
  const int g = lane >> 4, q = (lane >> 2) & 3, p = lane & 3;
  s16x4 v[2][2];
#pragma unroll
  for (int hf = 0; hf < 2; ++hf) {
    const int r = 16 * step + 8 * (lane >> 5) + 4 * hf + q;
    const unsigned at = sm_at(base, pitch, r, (c0 >> 5) * 8 + 2 * (g & 1) + (p >> 1)) + 8 * (p & 1);
    v[0][hf] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_ptr<lds_s16x4>(at));
    v[1][hf] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_ptr<lds_s16x4>(at ^ 64));
  }
#pragma unroll
  for (int t = 0; t < 2; ++t) f[t] = __builtin_bit_cast(f16x8, __builtin_shufflevector(v[t][0], v[t][1], 0, 1, 2, 3, 4, 5, 6, 7));
}
// full: with lo lo, 2^-22 of the product, which the rounding of a long sum hides and that of a short one does not. Error
// over that of f32 products without it and with it: 1.3 and 0.97 (8 x 16 to 8 x 128), 1.20 and 0.92 (32 x 64);
// 19 x 361 takes 2.4 us more. Matrices of 64 rows have 0.96 of that error without it.
__device__ __forceinline__ void mma_pairs(f32x16& acc, f32x16& cross, const f16x8 (&l)[2], const f16x8 (&r)[2], bool full) {
  if (full) cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(l[1], r[1], cross, 0, 0, 0);
  cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(l[1], r[0], cross, 0, 0, 0);
  cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(l[0], r[1], cross, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(l[0], r[0], acc, 0, 0, 0);
}
// Lane-dependent addresses of one product are formed where they are used: kept for the next one, they spill.
__device__ __forceinline__ int anew(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// The square of a symmetric 64 x 64 matrix: the 10 blocks of
// 16 x 16 on and above the diagonal, block w to wave w. A lane has column lane & 15 and rows 4 (lane >> 4) .. + 3
// of its block. Blocks above the diagonal are stored with their mirror images.
struct SmBlock {
  int r0, c0;
  bool on;
};
__device__ __forceinline__ SmBlock sm_block(int t) {
  const int bi = t < 4 ? 0 : t < 7 ? 1 : t < 9 ? 2 : 3, bc = t < 4 ? t : t < 7 ? t - 3 : t < 9 ? t - 5 : 3;
  return SmBlock{16 * bi, 16 * bc, t < 10};
}
__device__ __forceinline__ f32x4 sm_gram_square(unsigned a, float mul, const SmBlock& bl, int lane, bool full) {
  const int ln = anew(lane);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f}, cross = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int st = 0; st < 2; ++st) {
    f16x8 lf[2], rf[2];
    sm_rows16(lf, a, bl.r0, st, ln);
    sm_rows16(rf, a, bl.c0, st, ln);
    if (full) cross = __builtin_amdgcn_mfma_f32_16x16x32_f16(lf[1], rf[1], cross, 0, 0, 0);
    cross = __builtin_amdgcn_mfma_f32_16x16x32_f16(lf[1], rf[0], cross, 0, 0, 0);
    cross = __builtin_amdgcn_mfma_f32_16x16x32_f16(lf[0], rf[1], cross, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(lf[0], rf[0], acc, 0, 0, 0);
  }
  return (acc + cross) * mul;
}
// Of the mirror image, a lane has four columns of one row: 8 B.
__device__ __forceinline__ unsigned sm_mirror(unsigned base, const SmBlock& bl, int lane) {
  const int col = bl.r0 + 4 * (lane >> 4);
  return sm_at(base, 256, bl.c0 + (lane & 15), chunk_of(col)) + static_cast<unsigned>(2 * (col & 7));
}
__device__ __forceinline__ void sm_put(unsigned base, const f32x4& v, const SmBlock& bl, int lane) {
  const int ln = anew(lane);
  f16x4 hi, lo;
  const int col = bl.c0 + (ln & 15), row = bl.r0 + 4 * (ln >> 4);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const Pair p = split_pair(v[e]);
    hi[e] = p.hi;
    lo[e] = p.lo;
    const unsigned at = sm_at(base, 256, row + e, chunk_of(col)) + static_cast<unsigned>(2 * (col & 7));
    *lds_ptr<lds_f16>(at) = p.hi;
    *lds_ptr<lds_f16>(at ^ 64) = p.lo;
  }
  if (bl.r0 != bl.c0) {
    const unsigned at = sm_mirror(base, bl, ln);
    *lds_ptr<lds_f16x4>(at) = hi;
    *lds_ptr<lds_f16x4>(at ^ 64) = lo;
  }
}

template <typename T, bool STEP>
__global__ __launch_bounds__(kSmallThreads, 1) void ns_small_kernel(NsItems its, NsPlan pl, float mu, int nesterov, float eps) {
  extern __shared__ __attribute__((aligned(256))) unsigned char sm[];
  const unsigned S0 = static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)sm));
  const int k = place_of(its.first, blockIdx.x);
  const NsItem& it = its.it[k];
  const int mat = static_cast<int>(blockIdx.x) - its.first[k];
  const int rows = it.rows, cols = it.cols, tall = rows > cols;
  const int m = tall ? cols : rows, n = tall ? rows : cols, np = (n + 63) & ~63;
  const int lane = threadIdx.x & 63, wave = bf16l::wave_id();
  const unsigned MA = S0, MP = S0 + kSmallSquare, MQ = S0 + 2 * kSmallSquare, MT = S0 + 3 * kSmallSquare, X = S0 + 4 * kSmallSquare;
  const int xp = np * 4;  // pitch of X
  const T* src = static_cast<const T*>(it.src) + mat * it.sb;
  float* buf = STEP ? it.buf + mat * it.sb : nullptr;

  // The update (and the momentum) in registers, and its squares in f64. A thread takes runs of 8 values along
  // X's rows, which are one 16-B chunk of hi and one of lo: row i, columns 8 kc .. + 7.
  constexpr int kRuns = kSmallM * kSmallN / 8 / kSmallThreads;
  const int nc = (n + 7) >> 3, runs = m * nc;
  struct SmRun {
    int i, kc, at, step, left;  // row, chunk; its first value's place, the next one's distance, values there are
    bool on;
  };
  int place[kRuns];  // i + 64 kc
#pragma unroll
  for (int q = 0; q < kRuns; ++q) {
    const int id = min(static_cast<int>(threadIdx.x) + q * kSmallThreads, runs - 1);
    place[q] = tall ? id % m + 64 * (id / m) : id / nc + 64 * (id % nc);
  }
  auto run_of = [&](int q) __attribute__((always_inline)) {
    const int i = place[q] & 63, kc = place[q] >> 6;
    return SmRun{i, kc, tall ? 8 * kc * cols + i : i * cols + 8 * kc, tall ? cols : 1, n - 8 * kc,
                 static_cast<int>(threadIdx.x) + q * kSmallThreads < runs};
  };
  // Whole runs of a wide matrix's aligned rows in 16-B loads (64 x 384 f32: 41 us
  // for 51 one by one).
  typedef T vec8 __attribute__((ext_vector_type(8)));
  typedef float f32x8 __attribute__((ext_vector_type(8)));
  const bool vec = !tall && cols % 8 == 0 && ((reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(buf)) & 31) == 0;
  float v0[kRuns][8], o[kRuns][8];
#pragma unroll
  for (int q = 0; q < kRuns; ++q) {  // all loads in flight at once
    if (q * kSmallThreads < runs) {
      const SmRun r = run_of(q);
      if (vec) {
        const vec8 x = *reinterpret_cast<const vec8*>(src + r.at);
        f32x8 y;
        if constexpr (STEP) y = *reinterpret_cast<const f32x8*>(buf + r.at);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v0[q][e] = static_cast<float>(x[e]);
          if constexpr (STEP) o[q][e] = y[e];
        }
        continue;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int a = r.at + min(e, r.left - 1) * r.step;
        v0[q][e] = src_at<T>(src, a);
        if constexpr (STEP) o[q][e] = buf[a];
      }
    }
  }
  double s = 0.0;
#pragma unroll
  for (int q = 0; q < kRuns; ++q) {
    if (q * kSmallThreads < runs) {
      pin_batch(v0[q]);
      if constexpr (STEP) pin_batch(o[q]);
      const SmRun r = run_of(q);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool in = r.on && e < r.left;
        float w = v0[q][e];
        if constexpr (STEP) {
          const float nb = fmaf(mu, o[q][e], w);
          if (in) buf[r.at + e * r.step] = nb;
          w = nesterov ? fmaf(mu, nb, w) : nb;
        }
        w = in ? w : 0.f;
        s = fma(static_cast<double>(w), static_cast<double>(w), s);
        v0[q][e] = w;
      }
    }
  }
  // X is zero where no run lies: rows m .. 63, columns 8 nc .. np - 1
  for (int e = threadIdx.x; e < 64 * np / 4; e += kSmallThreads) *lds_ptr<lds_f16x8>(X + 16 * e) = f16x8{};
  for (int b = 1; b < 64; b <<= 1) s += __shfl_xor(s, b);
  double* red = reinterpret_cast<double*>(sm);
  if (lane == 0) red[wave] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int w = 0; w < kSmallThreads / 64; ++w) s += red[w];
  const NsScale sc = scale_of(s, eps);
  const NsTarget tg{nullptr, 0.f, 0.f, sc.small};
#pragma unroll
  for (int q = 0; q < kRuns; ++q) {
    const SmRun r = run_of(q);
    if (r.on) {
      f16x8 hi, lo;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const Pair p = split_pair(pinned(ldexpf(v0[q][e], sc.e) * sc.f));
        hi[e] = p.hi;
        lo[e] = p.lo;
      }
      const unsigned at = sm_at(X, xp, r.i, chunk_of(8 * r.kc));
      *lds_ptr<lds_f16x8>(at) = hi;
      *lds_ptr<lds_f16x8>(at ^ 64) = lo;
    }
  }
  __syncthreads();

  const int bi = 32 * (wave & 1), bc = 32 * ((wave >> 1) & 1), part = wave >> 2;
  const SmBlock bl = sm_block(wave);
  const bool full = m < kSmallM;
  for (int p = 0; p < pl.nphase; ++p) {  // phases of one step (kind 0)
    {  // A = X X^T, a 32 x 32 block and every third 16 k a wave; the thirds meet in MT and MP
      f32x16 acc = zero16(), cross = zero16();
      const int ln = anew(lane);
      for (int st = part; st < np / 16; st += 3) {
        f16x8 lf[2], rf[2];
        sm_rows(lf, X, xp, bi, st, ln);
        sm_rows(rf, X, xp, bc, st, ln);
        mma_pairs(acc, cross, lf, rf, full);
      }
      const int mine = (wave & 3) * 1024 + lane;
      const lds_f32 *sum1 = lds_ptr<lds_f32>(MT) + mine, *sum2 = lds_ptr<lds_f32>(MP) + mine;
      if (part) {
        lds_f32* sum = lds_ptr<lds_f32>(part == 1 ? MT : MP) + mine;
#pragma unroll
        for (int r = 0; r < 16; ++r) sum[64 * r] = acc[r] + cross[r];
      }
      __syncthreads();
      if (!part) {
        const float mul = ldexpf(1.f / kScale, -2 * x_shift(tg, pl.grown[p]));
        if (bi <= bc) {  // the block below the diagonal is the one above it, mirrored
#pragma unroll
          for (int q = 0; q < 4; ++q) {  // four rows of a column: the mirror image's four columns of a row
            f16x4 hi, lo;
            const int row = bi + 8 * q + 4 * (ln >> 5), col = bc + (ln & 31);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const Pair pr = split_pair((((acc[4 * q + e] + cross[4 * q + e]) + sum1[64 * (4 * q + e)]) + sum2[64 * (4 * q + e)]) * mul);
              hi[e] = pr.hi;
              lo[e] = pr.lo;
              const unsigned at = sm_at(MA, 256, row + e, chunk_of(col)) + static_cast<unsigned>(2 * (col & 7));
              *lds_ptr<lds_f16>(at) = pr.hi;
              *lds_ptr<lds_f16>(at ^ 64) = pr.lo;
            }
            if (bi < bc) {
              const unsigned at = sm_at(MA, 256, col, chunk_of(row)) + static_cast<unsigned>(2 * (row & 7));
              *lds_ptr<lds_f16x4>(at) = hi;
              *lds_ptr<lds_f16x4>(at ^ 64) = lo;
            }
          }
        }
      }
      __syncthreads();
    }
    const float sp = pl.sp[p];
    if (bl.on) {  // Q = a I + b A + c A A
      f32x4 v = sm_gram_square(MA, 1.f / (kScale * kScale), bl, lane, full);
      const int ln = anew(lane);
      const unsigned at = sm_mirror(MA, bl, ln);
      const f16x4 ah = *lds_ptr<lds_f16x4>(at), al = *lds_ptr<lds_f16x4>(at ^ 64);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = (static_cast<float>(ah[e]) + static_cast<float>(al[e])) * (1.f / kScale);
        v[e] = fmaf(pl.c, v[e], pl.b * x);
        if (bl.r0 + 4 * (ln >> 4) + e == bl.c0 + (ln & 15)) v[e] += pl.a;
        v[e] *= sp;
      }
      sm_put(MQ, v, bl, lane);
    }
    __syncthreads();
    // X <- Q X, 32 columns a wave; a wave reads its columns whole before it writes them
    const bool last = p + 1 == pl.nphase;
    const float mul = 1.f / (sp * kScale);
    for (int c0 = 32 * wave; c0 < np; c0 += 32 * (kSmallThreads / 64)) {
      f32x16 acc[2], cross[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) acc[b] = cross[b] = zero16();
      const int ln = anew(lane), j = ln & 31, h = ln >> 5;
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        f16x8 xf[2], qf[2];
        sm_cols(xf, X, xp, c0, st, ln);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          sm_rows(qf, MQ, 256, 32 * b, st, ln);
          if (last && tall) mma_pairs(acc[b], cross[b], xf, qf, full);  // transposed: lanes along the result's rows
          else mma_pairs(acc[b], cross[b], qf, xf, full);
        }
      }
      if (!last) {
        const float so = ldexpf(mul * kScale, x_shift(tg, pl.grown[p + 1]) - x_shift(tg, pl.grown[p]));
        // lane: column c0 + j; row 32 b + 4 h + row_of(r), whose swizzle is a constant of r ^ h
        const int chunk = chunk_of(c0) + (j >> 3);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const unsigned at = X + static_cast<unsigned>((32 * b + 4 * h) * xp + 2 * (j & 7));
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const Pair pr = split_pair((acc[b][r] + cross[b][r]) * so);
            const unsigned o = at + static_cast<unsigned>(row_of(r) * xp + 16 * (chunk ^ h ^ sm_swz(row_of(r))));
            *lds_ptr<lds_f16>(o) = pr.hi;
            *lds_ptr<lds_f16>(o ^ 64) = pr.lo;
          }
        }
        continue;
      }
      T* out = STEP ? nullptr : reinterpret_cast<T*>(it.p) + mat * it.ob;
      const int shift = x_shift(tg, pl.grown[p]);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int r0 = tall ? c0 : 32 * b, col = (tall ? 32 * b : c0) + j;
        if (col >= cols) continue;
        float old[16];
        if constexpr (STEP) {
#pragma unroll
          for (int r = 0; r < 16; ++r) old[r] = it.p[min(r0 + acc_row(r, h), rows - 1) * cols + col];
          pin_batch(old);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int row = r0 + acc_row(r, h);
          if (row >= rows) continue;
          const float v = ldexpf((acc[b][r] + cross[b][r]) * mul, -shift);
          if constexpr (STEP) it.p[row * cols + col] = fmaf(-it.rate, v, it.keep * old[r]);
          else out[row * cols + col] = static_cast<T>(v);
        }
      }
    }
    __syncthreads();
  }
}

// ---- host -------------------------------------------------------------------------------------------

float scale_for(double most) {  // the largest power of two up to kScale that keeps `most` below 2^15
  float s = kScale;
  while (s > 1e-3f && most * s > 32768.0) s *= 0.5f;
  return s;
}

// The longest phase. A's rounding, amplified along a phase, falls on the small singular directions, and narrow or
// near-square matrices have them, while the sums of a wide product hide it. Error of five steps over that of
// the formula in f32 products, noise matrices in f32, by phases:
//             16x64  32x128  64x64  64x256  96x96  96x192  256x1024
//   3 + 2      1.31    1.19   2.01    1.18   1.68    1.74      1.19
//   2 + 2 + 1  2.05    2.25   1.52    1.50   1.35    0.77      0.54
//   single     1.08    1.19   0.64    0.92   0.53    0.46      0.53
// A 16-bit result shows it in its last bits (64 x 128 bf16: with 3 + 2 2.8e-3 of the elements rounded to the other
// side, 1.0e-3 by the formula), an update in its parameters (the step over a ResNet-101's convolutions: 7.1e-8 of
// them with 3 + 2, 6.4e-8 by the formula). So every type takes single steps below kNarrow rows and where n < 1.5 m,
// and 2 + 2 + 1 elsewhere. Longer phases save products of m^2 n only: 22 x 256 x 1024 bf16 takes 172 us with 3 + 2,
// 187 with 2 + 2 + 1, 201 with single steps.
constexpr int kNarrow = 96;
constexpr int kLongest[2] = {1, 2};  // of each kind
// A call that has both kinds takes single steps for all, unless m^2 n of the wider ones (kind 1) is beyond this: the
// kinds' launches go together only in part. 2 of 64 x 576 and 12, 24, 48 of 256 x 1024 (8e8, 1.6e9, 3.2e9):
// 182, 225, 374 us with single steps for 202, 229, 369; 109 convolutions (1.6e10): 1544 for 1357.
constexpr double kMixedLeast = 1.5e9;
int ns_kind(int rows, int cols) {
  const long long m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
  return m < kNarrow || 2 * n < 3 * m ? 0 : 1;
}

// Phases, and scales that keep every f16 in range: the singular values of X0 are at most 1 (the Frobenius
// norm is), the scalar map carries that bound on, and P and Q are functions of the Gram matrix.
int ns_plan(NsPlan& pl, int steps, float a, float b, float c, int limit) {
  if (steps < 1 || steps > kMaxSteps) return fail(PROTOSEG_ERR_INVALID, "orthogonalize steps %d (1..%d)", steps, kMaxSteps);
  if (!(std::isfinite(a) && std::isfinite(b) && std::isfinite(c)))
    return fail(PROTOSEG_ERR_INVALID, "orthogonalize coefficients (%g, %g, %g)", a, b, c);
  pl.a = a, pl.b = b, pl.c = c;
  int longest = 1;  // 2^-22 a^(2 (L - 1)) <= 2^-13
  for (double f = 1.0; longest < limit && f * a * a <= 512.0; ++longest) f *= static_cast<double>(a) * a;
  pl.nphase = (steps + longest - 1) / longest;
  for (int p = 0, left = steps; p < pl.nphase; ++p) {
    pl.phases[p] = (left + pl.nphase - p - 1) / (pl.nphase - p);
    left -= pl.phases[p];
  }
  constexpr int kGrid = 256;  // between two points a map of slope 4 and curvature 50 rises by 1e-4
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

long long pad64_of(long long v) { return (v + kPad - 1) / kPad * kPad; }
int pad_of(long long v) { return static_cast<int>(pad64_of(v)); }  // of sizes that ns_check let pass

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
      g.kind = ns_kind(g.m, g.n);
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
  long long tiles = 0, thin = 0;  // 64 x 64 and 32 x 32 tiles of a symmetric product in all
  for (int k = 0; k < gs.n; ++k) {
    const long long nt = gs.g[k].mp / 64;
    tiles += gs.g[k].count * (nt * (nt + 1) / 2);
    thin += gs.g[k].count * (nt * (2 * nt + 1));
  }
  gs.thin = thin <= kThinTiles;
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
    long long split = gs.thin ? 1 : 384 / tiles;
    const long long chain = gs.thin ? (stages + 255) / 256 : (stages + 63) / 64, most = stages / 8;
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
  if (pad64_of(m) * pad64_of(n) > (1LL << 29) || m > 16384)
    return fail(PROTOSEG_ERR_UNSUPPORTED, "orthogonalize: %d x %d matrix (at most 2^29 padded elements, 16384 in the smaller dimension)",
                rows, cols);
  return PROTOSEG_OK;
}

// first[] of every group for a launch that gives each matrix of group k per(k) workgroups; the grid.
template <typename F>
long long ns_grid(NsGroups& gs, F per) {
  long long blocks = 0;
  for (int k = gs.n; k < kMaxGroups; ++k) gs.first[k] = 0x7fffffff;
  for (int k = 0; k < gs.n; ++k) {
    gs.first[k] = static_cast<int>(blocks < (1LL << 30) ? blocks : (1LL << 30));
    blocks += (per(k) * gs.g[k].count + 7) / 8 * 8;
  }
  return blocks;
}
int ns_blocks_ok(long long blocks) {
  return blocks < (1LL << 30) ? PROTOSEG_OK : fail(PROTOSEG_ERR_UNSUPPORTED, "orthogonalize: %lld workgroups", blocks);
}

template <int MODE>
long long ns_tiles(const NsGroup& g, const NsPart& jp, int T) {
  const long long nt = ceil_div(g.mp, T);
  if (MODE == kSym) return nt * (nt + 1) / 2 * jp.n * (jp.partial ? g.split : 1);
  if (!jp.n || (MODE == kWide && g.tall) || (MODE == kTall && !g.tall)) return 0;
  return nt * ceil_div(g.np, T);
}

template <int T, int MODE, int OUT, int G = 1>
int ns_launch_tile(NsGroups& gs, const NsJobs& js, hipStream_t st) {
  const long long blocks = ns_grid(gs, [&](int k) { return ns_tiles<MODE>(gs.g[k], js.of[k], T); });
  if (blocks == 0) return PROTOSEG_OK;
  if (int e = ns_blocks_ok(blocks)) return e;
  if constexpr (MODE == kSym && G == 1) {
    long long stages = 0;
    for (int k = 0; k < gs.n; ++k) {
      const NsGroup& g = gs.g[k];
      const NsPart& jp = js.of[k];
      if (jp.n) stages = std::max<long long>(stages, jp.j[0].l <= kX1 ? g.np / 32 / (jp.partial ? g.split : 1) : g.mp / 32);
    }
    if (blocks <= kHalvesTiles && stages >= kHalvesStages) return ns_launch_tile<T, MODE, OUT, 2>(gs, js, st);
  }
  constexpr size_t lds = static_cast<size_t>(G) * ring_of(T) * stage_bytes(T);
  if (int e = ensure_lds<ns_product_kernel<T, MODE, OUT, G>, lds>()) return e;
  KernelTimer t("ns_product_kernel", st);
  hipLaunchKernelGGL((ns_product_kernel<T, MODE, OUT, G>), dim3(static_cast<unsigned>(blocks)), dim3(256 * G), lds, st, gs, js);
  return check_launch("ns_product_kernel");
}
int ns_launch_thin(NsGroups& gs, const NsJobs& js, hipStream_t st) {
  const long long blocks = ns_grid(gs, [&](int k) { return ns_tiles<kSym>(gs.g[k], js.of[k], 32); });
  constexpr size_t lds = 4 * kThinRing * kThinStage;
  if (int e = ensure_lds<ns_thin_kernel, lds>()) return e;
  KernelTimer t("ns_thin_kernel", st);
  hipLaunchKernelGGL(ns_thin_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), lds, st, gs, js);
  return check_launch("ns_thin_kernel");
}
template <int MODE, int OUT>
int ns_launch(NsGroups gs, const NsJobs& js, hipStream_t st) {
  if constexpr (MODE == kSym) {
    return gs.thin ? ns_launch_thin(gs, js, st) : ns_launch_tile<64, MODE, OUT>(gs, js, st);
  } else {
    long long big = 0;
    for (int k = 0; k < gs.n; ++k) big += ns_tiles<MODE>(gs.g[k], js.of[k], 128) * gs.g[k].count;
    return big >= kApplyTiles ? ns_launch_tile<128, MODE, OUT>(gs, js, st) : ns_launch_tile<64, MODE, OUT>(gs, js, st);
  }
}

// The launches of a plan, in order.
enum NsLaunch { kSymmetric = 0, kNextX = 1, kResult = 2 };
struct NsOp {
  NsLaunch launch;
  NsPart part;
};
std::vector<NsOp> ns_program(const NsPlan& pl, bool split) {
  std::vector<NsOp> ops;
  int x = kX0, step = 0;
  auto add = [&](NsLaunch launch, std::initializer_list<NsJob> jobs, int partial = 0) {
    NsOp op{launch, NsPart{}};
    for (const NsJob& j : jobs) op.part.j[op.part.n++] = j;
    op.part.partial = partial;
    ops.push_back(op);
  };
  for (int p = 0; p < pl.nphase; ++p) {
    add(kSymmetric, {NsJob{x, x, kA, 0, 1.f / (kScale * kScale), kScale, pl.grown[p]}}, split);
    int q = kQ0;
    float sq = 0.f;
    for (int k = 0; k < pl.phases[p]; ++k, ++step) {
      const float sp = pl.sp[step];
      const int pb = k == 0 ? kQ0 : kP;  // the first P is Q
      add(kSymmetric, {NsJob{kA, kA, pb, 1, 1.f / (kScale * kScale), sp}});
      const bool more = k + 1 < pl.phases[p];
      const NsJob mul{pb, kA, kT, 0, 1.f / (sp * kScale), kScale};
      if (k == 0) {
        sq = sp;
        if (more) add(kSymmetric, {mul});
      } else {
        const int qn = q == kQ0 ? kQ1 : kQ0;
        const NsJob acc{pb, q, qn, 0, 1.f / (sp * sq), pl.sq[step]};
        if (more) add(kSymmetric, {mul, acc});
        else add(kSymmetric, {acc});
        q = qn;
        sq = pl.sq[step];
      }
      if (more) add(kSymmetric, {NsJob{kT, pb, kA, 0, 1.f / (sp * kScale), kScale}});
    }
    if (p + 1 < pl.nphase) {
      const int xn = x == kX0 ? kX1 : kX0;
      add(kNextX, {NsJob{q, x, xn, 0, 1.f / (sq * kScale), kScale, pl.grown[p], pl.grown[p + 1]}});
      x = xn;
    } else {
      add(kResult, {NsJob{q, x, x, 0, 1.f / (sq * kScale), 1.f, pl.grown[p]}});
    }
  }
  return ops;
}

// All products of a prepared X0, ending in the targets. pl[kind]: the plan of each kind that is there. Two kinds share
// launches: a kind whose X is due waits for no other, and symmetric products of both go together (five steps of
// 1 + 1 + 1 + 1 + 1 beside 2 + 2 + 1: 21 launches, 17 and 15 alone).
template <int OUT>
int ns_products(const NsGroups& gs, const NsPlan (&pl)[2], hipStream_t st) {
  bool split = false, there[2] = {false, false};
  for (int k = 0; k < gs.n; ++k) split = split || gs.g[k].split > 1, there[gs.g[k].kind] = true;
  std::vector<NsOp> ops[2];
  for (int c = 0; c < 2; ++c)
    if (there[c]) ops[c] = ns_program(pl[c], split);
  size_t at[2] = {0, 0};
  while (at[0] < ops[0].size() || at[1] < ops[1].size()) {
    NsLaunch launch = kSymmetric;
    for (int c = 0; c < 2; ++c)
      if (at[c] < ops[c].size()) launch = std::max(launch, ops[c][at[c]].launch);
    NsJobs js{};
    for (int c = 0; c < 2; ++c) {
      if (!there[c]) continue;
      js.a = pl[c].a, js.b = pl[c].b, js.c = pl[c].c;
      if (at[c] == ops[c].size() || ops[c][at[c]].launch != launch) continue;
      for (int k = 0; k < gs.n; ++k)
        if (gs.g[k].kind == c) js.of[k] = ops[c][at[c]].part;
      ++at[c];
    }
    if (launch == kNextX) {
      if (int e = ns_launch<kApply, kOutF32>(gs, js, st)) return e;
    } else if (launch == kResult) {
      if (int e = ns_launch<kWide, OUT>(gs, js, st)) return e;
      if (int e = ns_launch<kTall, OUT>(gs, js, st)) return e;
    } else {
      if (int e = ns_launch<kSym, kOutF32>(gs, js, st)) return e;
      NsGroups parts = gs;
      const long long blocks = ns_grid(parts, [&](int k) -> long long {
        const long long nb = gs.g[k].mp / 32;
        return js.of[k].partial && gs.g[k].split > 1 ? nb * (nb + 1) / 2 : 0;
      });
      if (blocks) {
        hipLaunchKernelGGL(ns_join_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, parts, js);
        if (int e = check_launch("ns_join_kernel")) return e;
      }
    }
  }
  return PROTOSEG_OK;
}

// Beside larger matrices a small one is nearly free in their launches; the kernel of its own is for calls
// that have no others. All of these are of kind 0.
bool ns_is_small(int rows, int cols) {
  const int m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
  return m <= kSmallM && pad_of(n) <= kSmallN;
}

template <typename T, bool STEP>
int ns_small(const std::vector<NsItem>& items, const NsPlan& pl, float mu, int nesterov, float eps, hipStream_t st) {
  for (size_t i0 = 0; i0 < items.size(); i0 += kMaxItems) {
    NsItems its{};
    long long blocks = 0;
    int n = 0;
    for (int k = 0; k < kMaxItems; ++k) its.first[k] = 0x7fffffff;
    for (size_t i = i0; i < items.size() && i < i0 + kMaxItems; ++i) {
      its.first[its.n] = static_cast<int>(blocks);
      its.it[its.n++] = items[i];
      blocks += items[i].count;
      if (int e = ns_blocks_ok(blocks)) return e;
      const int l = items[i].rows > items[i].cols ? items[i].rows : items[i].cols;
      n = pad_of(l) > n ? pad_of(l) : n;
    }
    if (int e = ensure_lds<ns_small_kernel<T, STEP>>()) return e;
    KernelTimer t("ns_small_kernel", st);
    hipLaunchKernelGGL((ns_small_kernel<T, STEP>), dim3(static_cast<unsigned>(blocks)), dim3(kSmallThreads),
                       4 * kSmallSquare + static_cast<size_t>(n) * 4 * kSmallM, st, its, pl, mu, nesterov, eps);
    if (int e = check_launch("ns_small_kernel")) return e;
  }
  return PROTOSEG_OK;
}

// Sums of squares and X0 of all items, kMaxItems a launch.
template <typename T, bool STEP>
int ns_load(const NsGroups& gs, const std::vector<NsItem>& items, float mu, int nesterov, float eps, hipStream_t st) {
  for (size_t i0 = 0; i0 < items.size(); i0 += kMaxItems)
    for (int pass = 0; pass < 2; ++pass) {  // the second pass finds what the first one read in the last-level cache
      NsItems its{};
      long long blocks = 0;
      for (int k = 0; k < kMaxItems; ++k) its.first[k] = 0x7fffffff;
      for (size_t i = i0; i < items.size() && i < i0 + kMaxItems; ++i) {
        const NsItem& it = items[i];
        const NsGroup& g = gs.g[it.group];
        its.first[its.n] = static_cast<int>(blocks);
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

// No C++ exception leaves a C entry: the only ones here are allocation failures of the host lists.
extern "C" size_t protoseg_orthogonalize_workspace_size(int count, int rows, int cols) try {
  if (count <= 0 || rows <= 0 || cols <= 0 || ns_check(rows, cols) != PROTOSEG_OK) return 0;
  NsGroups gs;
  return ns_is_small(rows, cols) ? 0 : ns_layout(gs, {NsMatrix{rows, cols, count}}, nullptr, nullptr);
} catch (const std::exception&) {
  return 0;
}

extern "C" int protoseg_orthogonalize(const void* g, int dtype, int count, int rows, int cols, int64_t stride, int steps, float a,
                                      float b, float c, float eps, void* out, void* workspace, size_t workspace_bytes,
                                      protoseg_stream_t stream) try {
  if (dtype != PROTOSEG_F32 && dtype != PROTOSEG_BF16 && dtype != PROTOSEG_F16)
    return fail(PROTOSEG_ERR_UNSUPPORTED, "orthogonalize dtype %d (f32, bf16 or f16)", dtype);
  if (count < 0) return fail(PROTOSEG_ERR_INVALID, "orthogonalize: %d matrices", count);
  if (int e = ns_check(rows, cols)) return e;
  if (!(eps >= 0.f)) return fail(PROTOSEG_ERR_INVALID, "orthogonalize eps %g", eps);
  NsPlan pl[2];
  const int kind = ns_kind(rows, cols);
  if (int e = ns_plan(pl[kind], steps, a, b, c, kLongest[kind])) return e;
  if (count == 0 || rows == 0 || cols == 0) return PROTOSEG_OK;
  const long long size = static_cast<long long>(rows) * cols;
  if (!g || !out) return fail(PROTOSEG_ERR_INVALID, "orthogonalize: matrices and result must be non-null");
  if (count > 1 && stride < size) return fail(PROTOSEG_ERR_INVALID, "orthogonalize: matrices %lld elements apart overlap", static_cast<long long>(stride));
  NsGroups gs;
  const bool is_small = ns_is_small(rows, cols);
  const size_t need = is_small ? 0 : ns_layout(gs, {NsMatrix{rows, cols, count}}, nullptr, nullptr);
  if (need && (!workspace || workspace_bytes < need))
    return fail(PROTOSEG_ERR_INVALID, "orthogonalize workspace %zu bytes, needs %zu", workspace ? workspace_bytes : 0, need);
  gs.ws = static_cast<unsigned char*>(workspace);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const std::vector<NsItem> items{NsItem{g, static_cast<float*>(out), nullptr, stride, size, count, rows, cols, 0, 0, 0.f, 0.f}};
  auto go = [&](auto tag, auto kind) -> int {
    if (is_small) return ns_small<decltype(tag), false>(items, pl[0], 0.f, 0, eps, st);
    if (int e = ns_load<decltype(tag), false>(gs, items, 0.f, 0, eps, st)) return e;
    return ns_products<decltype(kind)::value>(gs, pl, st);
  };
  if (dtype == PROTOSEG_F32) return go(float{}, std::integral_constant<int, kOutF32>());
  if (dtype == PROTOSEG_BF16) return go(__bf16{}, std::integral_constant<int, kOutBF16>());
  return go(_Float16{}, std::integral_constant<int, kOutF16>());
} catch (const std::exception& e) {
  return fail(PROTOSEG_ERR_INVALID, "orthogonalize: %s", e.what());
}

namespace {
// A call's matrices in runs of at most kMaxGroups shapes (one launch covers a run).
struct MuonRun {  // none where all matrices are small (ns_small_kernel)
  std::vector<NsMatrix> mats;
  std::vector<int> from;  // tensor of the call
};
int muon_runs(std::vector<MuonRun>& runs, int n, const int32_t* rows, const int32_t* cols) {
  std::vector<std::pair<int, int>> shapes;
  bool all_small = true;
  for (int i = 0; i < n; ++i) {
    if (int e = ns_check(rows[i], cols[i])) return e;
    all_small = all_small && ns_is_small(rows[i], cols[i]);
  }
  for (int i = 0; i < n; ++i) {
    if (rows[i] == 0 || cols[i] == 0 || all_small) continue;
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

extern "C" size_t protoseg_muon_workspace_size(int n_tensors, const int32_t* rows, const int32_t* cols) try {
  std::vector<MuonRun> runs;
  if (n_tensors <= 0 || !rows || !cols || muon_runs(runs, n_tensors, rows, cols) != PROTOSEG_OK) return 0;
  size_t most = 0;
  for (const MuonRun& r : runs) {
    NsGroups gs;
    const size_t n = ns_layout(gs, r.mats, nullptr, nullptr);
    most = n > most ? n : most;
  }
  return most;
} catch (const std::exception&) {
  return 0;
}

extern "C" int protoseg_muon_step(int n_tensors, float* const* params, const float* const* grads, float* const* momentum_bufs,
                                  const int32_t* rows, const int32_t* cols, float momentum, int nesterov, float lr,
                                  float weight_decay, int scale_kind, int steps, float a, float b, float c, float eps,
                                  void* workspace, size_t workspace_bytes, protoseg_stream_t stream) try {
  if (n_tensors < 0 || (n_tensors > 0 && (!params || !grads || !momentum_bufs || !rows || !cols)))
    return fail(PROTOSEG_ERR_INVALID, "muon: %d tensors, pointer and size arrays must be non-null", n_tensors);
  if (!(momentum >= 0.f && momentum < 1.f) || !(eps >= 0.f) || !std::isfinite(lr) || !std::isfinite(weight_decay))
    return fail(PROTOSEG_ERR_INVALID, "muon: momentum %g in [0, 1), eps %g >= 0, lr %g, weight decay %g", momentum, eps, lr, weight_decay);
  if (scale_kind != 0 && scale_kind != 1) return fail(PROTOSEG_ERR_INVALID, "muon scale kind %d (0 or 1)", scale_kind);
  NsPlan pl[2];
  bool there[2] = {n_tensors == 0, false};
  double wide = 0.0;  // m^2 n of the matrices of kind 1
  for (int i = 0; i < n_tensors; ++i) {
    const int k = ns_kind(rows[i], cols[i]);
    there[k] = true;
    if (k) wide += static_cast<double>(std::min(rows[i], cols[i])) * rows[i] * cols[i];
  }
  const bool single = there[0] && wide < kMixedLeast;
  if (single) there[1] = false;
  for (int k = 0; k < 2; ++k)
    if (there[k])
      if (int e = ns_plan(pl[k], steps, a, b, c, kLongest[k])) return e;
  std::vector<MuonRun> runs;
  if (int e = muon_runs(runs, n_tensors, rows, cols)) return e;
  size_t need = 0;
  for (int i = 0; i < n_tensors; ++i)
    if (rows[i] && cols[i] && (!params[i] || !grads[i] || !momentum_bufs[i]))
      return fail(PROTOSEG_ERR_INVALID, "muon tensor %d: null pointer", i);
  for (float* const* list : {params, momentum_bufs}) {  // twice in the call, two workgroups would write it at once
    std::vector<const float*> seen;
    for (int i = 0; i < n_tensors; ++i)
      if (rows[i] && cols[i]) seen.push_back(list[i]);
    std::sort(seen.begin(), seen.end());
    if (std::adjacent_find(seen.begin(), seen.end()) != seen.end())
      return fail(PROTOSEG_ERR_INVALID, "muon: a parameter or momentum buffer is in the call twice");
  }
  for (const MuonRun& r : runs) {
    NsGroups gs;
    const size_t n = ns_layout(gs, r.mats, nullptr, nullptr);
    need = n > need ? n : need;
  }
  if (need && (!workspace || workspace_bytes < need))
    return fail(PROTOSEG_ERR_INVALID, "muon workspace %zu bytes, needs %zu", workspace ? workspace_bytes : 0, need);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  auto item = [&](int i, int group, int index) {
    const double r = rows[i], q = cols[i];
    const double scale = scale_kind == 0 ? sqrt(r > q ? r / q : 1.0) : 0.2 * sqrt(r > q ? r : q);
    return NsItem{grads[i], params[i], momentum_bufs[i], 0, 0, 1, rows[i], cols[i], group, index, static_cast<float>(lr * scale),
                  static_cast<float>(1.0 - static_cast<double>(lr) * weight_decay)};
  };
  std::vector<NsItem> items;
  for (const MuonRun& run : runs) {
    NsGroups gs;
    std::vector<int> which, index;
    ns_layout(gs, run.mats, &which, &index);
    for (int k = 0; single && k < gs.n; ++k) gs.g[k].kind = 0;
    gs.ws = static_cast<unsigned char*>(workspace);
    items.clear();
    for (size_t k = 0; k < run.mats.size(); ++k) items.push_back(item(run.from[k], which[k], index[k]));
    if (int e = ns_load<float, true>(gs, items, momentum, nesterov ? 1 : 0, eps, st)) return e;
    if (int e = ns_products<kOutStep>(gs, pl, st)) return e;
  }
  if (!runs.empty()) return PROTOSEG_OK;
  for (int i = 0; i < n_tensors; ++i)
    if (rows[i] && cols[i]) items.push_back(item(i, 0, 0));
  return ns_small<float, true>(items, pl[0], momentum, nesterov ? 1 : 0, eps, st);
} catch (const std::exception& e) {
  return fail(PROTOSEG_ERR_INVALID, "muon: %s", e.what());
}
