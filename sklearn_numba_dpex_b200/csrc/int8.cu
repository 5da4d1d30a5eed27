// Products in 8-bit integers with a scale for each row of both operands, and the quantisation of
// rows that feeds them.
//
//   q[i, f] = round_half_even(127 x[i, f] / max_f |x[i, f]|),   scale[i] = max_f |x[i, f]| / 127
//   out[i, j] = sa[i] * sb[j] * sum_f qa[i, f] qb[j, f]  (+ bias[j])
//
// dense, or by group: rows [offsets[g], offsets[g + 1]) of the left operand meet the g-th matrix of
// the right one (the experts' products of a mixture of experts).  The sum is an int32 and exact for
// d <= 131 071 (127 and 128 in magnitude: 131 072 products of 2^14 reach 2^31).
//
// No counterpart in the reference; they stand beside the products of matmul_hook.cu.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdlib.h>

#include "early_launch.cuh"
#include "kmb_common.cuh"
#include "row_types.cuh"
#include "tc_ptx.cuh"

namespace kmb {

// =============================================================================== quantisation
// A row per block, or per warp (WARP) where a warp holds one.  A thread holds up to VECS pieces of eight
// elements, and the launch takes as many threads as a row needs: four pieces where there are rows enough to
// fill the GPU, so that enough bytes are on their way while other blocks wait at their barrier or round; one or
// two with few rows, for the latency of a row.  The pieces stay in registers, as they lie in memory, between
// the maximum and the rounding; rows longer than 8192 (VECS = 0) are read a second time, from L1 and L2.
// 8192 rows of 4096 bf16 take 28 us (100 MB, 3.6 TB/s), bound by instruction issue (0.75 a scheduler and cycle,
// 16 instructions an element and lane); with two pieces a thread they took 32 us, with a warp per row and 16
// pieces a lane, which left 12 warps on an SM, 80.
constexpr int QR_THREADS = 256, QR_WARP_ROWS = 4;

// How near to the middle between two whole numbers a product is in doubt (see QrPiece::round).
constexpr float QR_SURE = 0.49999f;

// The numbers in doubt of a piece in 64 bits, one at a time from memory: one piece in 6000 comes here, and
// the registers of the others are not indexed for its sake.
template <typename T>
__device__ __noinline__ void quantize_exactly(const T* row, int f, int d, float top, float inv, int8_t* q) {
  for (int j = 0; j < 8 && f + j < d; ++j) {
    const float x = to_float(row[f + j]), r = x * inv;
    if (!(fabsf(r - rintf(r)) < 0.4999f)) q[f + j] = (int8_t)(int)rint((double)x * 127.0 / (double)top);
  }
}

template <typename T>
struct Pair;
template <>
struct Pair<__half> { typedef __half2 type; };
template <>
struct Pair<__nv_bfloat16> { typedef __nv_bfloat162 type; };

template <typename T>
struct QrPiece {
  alignas(16) T t[8];
  __device__ __forceinline__ void load(const T* row, int f, int d, bool vec) {
    if (vec) {       // rows of whole 16-byte pieces; a piece of eight floats may end behind the row
      uint4* dst = reinterpret_cast<uint4*>(t);
#pragma unroll
      for (int q = 0; q < (int)sizeof(T) / 2; ++q)
        dst[q] = f + q * (16 / (int)sizeof(T)) < d ? *reinterpret_cast<const uint4*>(row + f + q * (16 / (int)sizeof(T)))
                                                   : make_uint4(0u, 0u, 0u, 0u);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = f + j < d ? row[f + j] : from_float<T>(0.f);
    }
  }
  // bits of the greatest |x|: whole numbers in the order of the values, NaN above infinity
  __device__ __forceinline__ uint32_t top() const {
    if constexpr (sizeof(T) == 2) {
      typedef typename Pair<T>::type P;
      const P* pairs = reinterpret_cast<const P*>(t);
      const P m = __hmax2_nan(__hmax2_nan(__habs2(pairs[0]), __habs2(pairs[1])),
                              __hmax2_nan(__habs2(pairs[2]), __habs2(pairs[3])));
      return max(__float_as_uint(to_float(m.x)), __float_as_uint(to_float(m.y)));
    } else {
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(to_float(t[j])) & 0x7fffffffu);
      return m;
    }
  }
  // The eight 8-bit numbers, and whether one of them is in doubt.  With f = 127 / top in 32 bits, x f is off
  // 127 x / top by at most 127 * 2^-24 = 7.6e-6, so round_half_even(127 x / top) as exact arithmetic has it is
  // the rounding of x f unless that lies closer than 1e-5 to the middle between two whole numbers; then the
  // quotient in 64 bits decides (127 x is exact there, and a quotient of such short numbers is never rounded
  // onto a middle that it does not hit).  x f + 1.5 * 2^23 in one operation is rounded to a whole number, whose
  // low byte is the result; a second one gives what the rounding took away.
  __device__ __forceinline__ uint2 round(float inv, bool& doubt) const {
    const float magic = 12582912.f;
    uint32_t n[8];
    float off = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = to_float(t[j]);
      const float s = fmaf(x, inv, magic);
      n[j] = __float_as_uint(s);
      off = fmaxf(off, fabsf(fmaf(x, inv, magic - s)));
    }
    doubt = !(off < QR_SURE);
    uint2 p;
    p.x = __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410);
    p.y = __byte_perm(__byte_perm(n[4], n[5], 0x0040), __byte_perm(n[6], n[7], 0x0040), 0x5410);
    return p;
  }
};

template <typename T, bool WARP, int VECS>
__global__ void __launch_bounds__(QR_THREADS, sizeof(T) == 2 ? 5 : 4)
quantize_rows_kernel(const T* x, int64_t n, int d, const int32_t* rows, int64_t m,
                     int8_t* __restrict__ q, int64_t q_pitch, float* __restrict__ scales, int vec) {
  next_grid_may_start();
  grid_dependency_wait();
  __shared__ uint32_t red[QR_THREADS / 32];
  const int threads = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int64_t i = WARP ? (int64_t)blockIdx.x * QR_WARP_ROWS + (threadIdx.x >> 5) : blockIdx.x;
  if (WARP && i >= m) return;
  int64_t src = i;
  if (rows) {
    src = rows[i];
    if (src >= n) src = -1;
  }
  int8_t* qi = q + i * q_pitch;
  const T* xi = x + (src < 0 ? 0 : src) * d;
  const int end = src < 0 ? 0 : d;       // a row that is not there is a row of zeros
  constexpr int HELD = VECS > 0 ? VECS : 1;
  QrPiece<T> v[HELD];
  uint32_t top = 0;
  if (VECS > 0) {
#pragma unroll
    for (int r = 0; r < HELD; ++r) v[r].load(xi, (r * threads + tid) * 8, end, vec != 0);
#pragma unroll
    for (int r = 0; r < HELD; ++r) top = max(top, v[r].top());
  } else {
    for (int f = tid * 8; f < end; f += threads * 8) {
      v[0].load(xi, f, end, vec != 0);
      top = max(top, v[0].top());
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (!WARP) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();
    top = red[0];
    for (int w = 1; w < threads / 32; ++w) top = max(top, red[w]);
  }
  const float topf = __uint_as_float(top);
  // a row that holds an infinity or NaN has no 8-bit image: NaN as its scale makes its products NaN
  const bool bad = top >= 0x7f800000u;
  if (tid == 0) scales[i] = bad ? __uint_as_float(0x7fffffffu) : topf / 127.f;
  const bool zero = bad || top == 0u;
  const float inv = 127.f / topf;
  const bool tiny = topf < 1e-30f;       // the factor runs out of range
  // the pitch is a multiple of 16, so the eight bytes of a piece lie inside the row's own storage
  auto put = [&](const QrPiece<T>& piece, int f) {
    bool doubt;
    const uint2 p = piece.round(inv, doubt);
    *reinterpret_cast<uint2*>(qi + f) = zero ? make_uint2(0u, 0u) : p;
    if ((doubt || tiny) && !zero) quantize_exactly(xi, f, end, topf, inv, qi);
  };
  if (VECS > 0) {
#pragma unroll
    for (int r = 0; r < HELD; ++r)
      if ((r * threads + tid) * 8 < d) put(v[r], (r * threads + tid) * 8);
  } else {
    for (int f = tid * 8; f < d; f += threads * 8) {
      v[0].load(xi, f, end, vec != 0);
      put(v[0], f);
    }
  }
}

template <typename T>
int quantize_run(const T* x, int64_t n, int d, const int32_t* rows, int64_t m, int8_t* q,
                 int64_t q_pitch, float* scales, cudaStream_t s) {
  const int vec = rows_are_vec(x, d) ? 1 : 0;
  const bool many = m >= (int64_t)sm_count() * 8;
  const int pieces = (int)ceil_div(d, 8);
#define KMB_RUN(WARP, VECS, THREADS)                                                            \
  return launch_early(quantize_rows_kernel<T, WARP, VECS>, (unsigned)(WARP ? ceil_div(m, QR_WARP_ROWS) : m), THREADS, \
                      0, 1, s, x, n, d, rows, m, q, q_pitch, scales, vec)
  if (pieces <= 32) KMB_RUN(true, 1, 32 * QR_WARP_ROWS);
  if (pieces <= 64) KMB_RUN(true, 2, 32 * QR_WARP_ROWS);
  if (many && pieces <= 128) KMB_RUN(true, 4, 32 * QR_WARP_ROWS);
  if (pieces > QR_THREADS * 4) KMB_RUN(false, 0, QR_THREADS);
  // as many pieces a thread as leave the fewest threads without one
  const auto width = [pieces](int v) { return (int)ceil_div(pieces, v * 32) * 32; };
  if (!many && pieces <= QR_THREADS) KMB_RUN(false, 1, width(1));
  if (!many && pieces <= QR_THREADS * 2) KMB_RUN(false, 2, width(2));
  if (pieces <= QR_THREADS * 3 && width(3) * 3 < width(4) * 4) KMB_RUN(false, 3, width(3));
  KMB_RUN(false, 4, width(4));
#undef KMB_RUN
}

// ==================================================================================== product
// tcgen05 kind::i8, int32 accumulators in tensor memory.  The matrix instruction's M side (128 lanes)
// takes 128 rows of the RIGHT operand (output features), its N side BN rows of the left one (tokens):
// a few tokens then cost a narrow instruction, and the weights, which bound small batches, stream
// through at full width.
//
// One persistent CTA per SM, twelve warps: 0 loads (TMA, 128-byte swizzle, a ring of stages of 128
// bytes of the contraction), 1 issues the MMAs, 2 owns tensor memory, 4..11 scale and store (one
// feature per lane, half of the tokens each).  Two accumulators, so that the stores of a tile overlap the
// MMAs of the next.  (With four storing warps a tile of 256 tokens and 2056 features took longer to store
// than to multiply: 88 us for 16 396 rows of 32 groups and 1408 outputs.)
//
// PAIR: many wide tiles.  Two CTAs multiply 256 features by BN tokens with one instruction
// (cta_group::2); each loads its own 128 features and HALF of the tokens, 32 KB a stage instead of 48.  One
// CTA alone asks for 94 bytes a cycle to keep its tensor core busy and an SM receives 64 from L2: 8192 x 8192 x
// 4096 took 192 us that way, at 16.7 TB/s from L2 and 61 bytes a cycle and SM.
//
// Measured: 8192 x 8192 x 4096 in 166 us = 3.3e15 operations a second, the tensor pipe active 92 % of the time;
// 16 396 rows of 32 groups, 1408 x 2056, 61 us (weights at a pitch of 2064 bytes; 56 us at whole lines), bound by
// what an SM receives from L2; 384 rows of 64 groups, 2048 x 1024, 26 us for 134 MB of weights (5.2 TB/s).
//
// SPLIT: few tiles (one row against 4096 x 4096 weights: 7.5 us, 12.1 with a CTA per tile).  A cluster of CTAs
// shares a tile, each summing a run of the contraction, so that more
// SMs stream weights; the int32 partial sums meet through distributed shared memory, exactly, and each
// CTA stores a share of the tokens.  A cluster has one tile at most.
constexpr int I8_BM = 128;
constexpr int I8_KB = 128;            // bytes (= 8-bit features) per stage
constexpr int I8_EPI_WARPS = 8;
constexpr int I8_THREADS = 128 + I8_EPI_WARPS * 32;
constexpr int I8_SCAN_THREADS = 256;
constexpr int I8_PAIR_BOX = 64;       // token rows that one load brings for a pair's narrow tile (boxes of 32
                                      // for whole tiles too took 207 us where one load a stage takes 166)
constexpr int I8_MAX_GROUPS = 1024;
constexpr long long I8_TIMEOUT_CYCLES = 4000000000LL;   // ~2 s at 2 GHz

enum I8Mode { I8_SINGLE, I8_SPLIT, I8_PAIR };

template <int BN, I8Mode MODE>
struct I8Cfg {
  static constexpr int CTAS = MODE == I8_PAIR ? 2 : 1;          // that one instruction spans
  static constexpr int A_BYTES = I8_BM * I8_KB, B_BYTES = BN / CTAS * I8_KB;
  static constexpr int FIT = (212 * 1024) / (A_BYTES + B_BYTES);
  static constexpr int STAGES = FIT > 12 ? 12 : FIT;
  static constexpr int TMEM_COLS = 2 * BN < 32 ? 32 : 2 * BN;
  // int32 += s8 * s8, both K-major, `cols` tokens wide
  __host__ __device__ static constexpr uint32_t idesc(int cols) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(cols >> 3) << 17) | ((uint32_t)(CTAS * I8_BM >> 4) << 24);
  }
  // tokens that a tile of `rows` is multiplied as: a group's last tile in a pair is as narrow as its rows
  // allow, in steps of two boxes (one in each CTA)
  __device__ static __forceinline__ int cols(int rows) {
    return MODE == I8_PAIR ? (rows + 2 * I8_PAIR_BOX - 1) / (2 * I8_PAIR_BOX) * (2 * I8_PAIR_BOX) : BN;
  }
};

template <int BN, I8Mode MODE>
struct I8Smem {
  typedef I8Cfg<BN, MODE> Cfg;
  unsigned char a[Cfg::STAGES][Cfg::A_BYTES];
  unsigned char b[Cfg::STAGES][Cfg::B_BYTES];
  int first_tile[I8_MAX_GROUPS + 1];   // tiles before each group
  int scan[I8_SCAN_THREADS / 32];
  float sa[BN];
  int bad;                             // SPLIT: this CTA's partial sums are not to be used
  int far;                             // SPLIT: a scale of the tile's tokens lies far from 1
  unsigned long long full[Cfg::STAGES], empty[Cfg::STAGES];
  unsigned long long acc_full[2], acc_empty[2], drain;
  long long timeout_cycles;
  unsigned int tmem_base;
  volatile int abort_flag;
};
constexpr size_t I8_SMEM_LIMIT = 232448 - 1024;      // 227 KB, less the alignment of the stages
static_assert(sizeof(I8Smem<256, I8_PAIR>) <= I8_SMEM_LIMIT && sizeof(I8Smem<256, I8_SINGLE>) <= I8_SMEM_LIMIT && sizeof(I8Smem<128, I8_SINGLE>) <= I8_SMEM_LIMIT &&
                  sizeof(I8Smem<64, I8_SINGLE>) <= I8_SMEM_LIMIT && sizeof(I8Smem<32, I8_SINGLE>) <= I8_SMEM_LIMIT &&
                  sizeof(I8Smem<16, I8_SINGLE>) <= I8_SMEM_LIMIT,
              "the stages exceed the 227 KB a CTA may use");

struct I8Params {
  const float* sa;
  const float* sb;
  const float* bias;          // or NULL
  const int32_t* offsets;     // or NULL: one group of all m rows
  void* out;
  int64_t m;
  int groups, n, d;
  int feature_tiles;
  long long timeout_cycles;
  int test_stall;             // test hook: the loading warp stops after its first tile
};

__device__ __forceinline__ bool mbar_try_wait_cluster(void* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Address that `p` has in the shared memory of CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t address_in(const void* p, uint32_t rank) {
  uint32_t addr;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(p)), "r"(rank));
  return addr;
}

// Raised by a wait that ran out, on the GPU that ran it; read and cleared by kmb_int8_wait_error.
static __device__ int g_i8_wait_error;

// REMOTE: the other CTA of a pair arrives there too.
template <bool REMOTE = false, typename Smem>
__device__ __forceinline__ bool i8_wait(void* bar, uint32_t parity, Smem* sm) {
  const auto done = [&] { return REMOTE ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity); };
  if (done()) return true;
  const long long t0 = clock64();
  while (true) {
    for (int i = 0; i < 64; ++i)
      if (done()) return true;
    if (sm->abort_flag) return false;
    if (clock64() - t0 > sm->timeout_cycles) {
      sm->abort_flag = 1;
      atomicExch(&g_i8_wait_error, 1);
      return false;
    }
  }
}

// The forms that span the two CTAs of a pair: tensor memory in both, loads that report to CTA 0's barrier, the
// product, and completion that arrives at the same place in both.
__device__ __forceinline__ void pair_tmem_alloc(void* smem_dst, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem_dst)), "r"(ncols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void pair_tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void pair_tma_load(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar0) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
      "%4}], [%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(bar0), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void pair_umma_i8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void pair_commit(void* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t remote_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote_bar) : "memory");
}

__device__ __forceinline__ void umma_i8_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                           uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}

// First row of group g, clamped so that no offset, however wrong, leads outside the m rows.
__device__ __forceinline__ int64_t i8_row_of(const I8Params& p, int g) {
  if (p.offsets == nullptr) return g == 0 ? 0 : p.m;
  const int64_t o = p.offsets[g];
  return o < 0 ? 0 : (o > p.m ? p.m : o);
}

// Sum of two numbers of tiles.  Offsets that go up and down may name every row once for each group, more tiles than
// 32 bits hold; the sum then stays at the greatest number there is, so that every tile lies in its group all the same.
constexpr int I8_MAX_TILES = 1 << 30;
__device__ __forceinline__ int i8_add_tiles(int a, int b) {
  const unsigned sum = (unsigned)a + (unsigned)b;          // both are at most 2^30
  return sum < (unsigned)I8_MAX_TILES ? (int)sum : I8_MAX_TILES;
}

struct I8Tile {
  int g;
  int64_t row0;     // first token row
  int rows;         // token rows of the tile that belong to the group
  int feature0;
};

// `wide`: features of a tile; `skip`: where this CTA's 128 of them begin.
template <int BN>
__device__ __forceinline__ I8Tile i8_tile(const I8Params& p, const int* first_tile, int t, int wide = I8_BM,
                                          int skip = 0) {
  int lo = 0, hi = p.groups;                 // last group with first_tile[g] <= t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first_tile[mid] <= t) lo = mid; else hi = mid;
  }
  const int local = t - first_tile[lo];
  I8Tile r;
  r.g = lo;
  const int mt = local / p.feature_tiles;
  r.feature0 = (local - mt * p.feature_tiles) * wide + skip;
  const int64_t start = i8_row_of(p, lo);
  r.row0 = start + (int64_t)mt * BN;
  const int64_t left = i8_row_of(p, lo + 1) - r.row0;
  r.rows = left < BN ? (int)left : BN;
  return r;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
// A word of the shared memory of CTA `rank` of the cluster, at the place `p` has in this one's.
__device__ __forceinline__ int load_from(const void* p, uint32_t rank) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(address_in(p, rank)) : "memory");
  return v;
}

// Barrier of the storing warps; whether any of their threads says so.
__device__ __forceinline__ bool i8_any_of_storing_warps(bool mine) {
  static_assert(I8_EPI_WARPS * 32 == 256, "the barrier's count");
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, 1, 256, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"((uint32_t)mine)
      : "memory");
  return any != 0;
}
// Whether a product with this scale may leave the range of 32 bits although the result does not: the other scale
// lies within 2^60 of 1 then, or is such a one itself.  (Infinities and NaN come out the same either way.)
__device__ __forceinline__ bool i8_far(float scale) {
  const float a = fabsf(scale);
  return (a > 0x1p60f && a < INFINITY) || (a < 0x1p-60f && a != 0.f);
}
// One result.  FAR: in 64 bits, rounded once to 32.
template <bool FAR, typename T>
__device__ __forceinline__ T i8_scaled(int sum, float sa, float sb, float bias) {
  if (FAR) return from_float<T>((float)((double)sum * (double)sa * (double)sb + (double)bias));
  return from_float<T>((float)sum * (sa * sb) + bias);
}

// Scales COLS accumulator columns (tokens) of one feature and stores them; FULL: all of them are rows.
template <int COLS, bool FULL, typename T>
__device__ __forceinline__ void i8_store(const uint32_t (&v)[COLS], const float* sa, float sb, float bias, T* o,
                                         int64_t stride, int rows) {
#pragma unroll
  for (int j = 0; j < COLS; ++j) {
    if (FULL || j < rows) *o = i8_scaled<false, T>((int)v[j], sa[j], sb, bias);
    o += stride;
  }
}
// All of a warp's columns with scales far from 1, by its 32 lanes together; out of line, since inlined it made the
// stores of every tile slower (32 groups of 512 rows, 1408 x 2048: 52.8 -> 53.9 us).
template <typename T>
__device__ __noinline__ void i8_store_far(uint32_t acc, int cols, const float* sa, float sb, float bias, T* o,
                                          int64_t stride, int rows) {
#pragma unroll 1
  for (int c = 0; c < cols; c += 16) {
    uint32_t v[16];
    tmem_ld16(acc + c, v);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (c + j < rows) o[(c + j) * stride] = i8_scaled<true, T>((int)v[j], sa[c + j], sb, bias);
  }
}

template <int BN, typename T, I8Mode MODE>
__global__ void __launch_bounds__(I8_THREADS, 1)
int8_matmul_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                   const __grid_constant__ CUtensorMap map_tail, const __grid_constant__ I8Params p) {
  using Cfg = I8Cfg<BN, MODE>;
  constexpr bool SPLIT = MODE == I8_SPLIT, PAIR = MODE == I8_PAIR;
  extern __shared__ __align__(16) unsigned char i8_dyn[];
  I8Smem<BN, MODE>* sm = reinterpret_cast<I8Smem<BN, MODE>*>(((uintptr_t)i8_dyn + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int splits = SPLIT ? (int)cluster_size() : 1, split = SPLIT ? (int)cluster_rank() : 0;
  const int in_pair = PAIR ? (int)cluster_rank() : 0;            // CTA 0 of a pair issues its products
  const int per_tile = PAIR ? 2 : splits;                        // CTAs that work on a tile
  const int first = blockIdx.x / per_tile;                       // this CTA's (or cluster's) first tile
  const int step = gridDim.x / per_tile;
  const int wide = PAIR ? 2 * I8_BM : I8_BM, skip = in_pair * I8_BM;

  if (threadIdx.x == 32) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::STAGES; ++s) {
      mbar_init(&sm->full[s], 1);
      mbar_init(&sm->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sm->acc_full[b], 1);
      mbar_init(&sm->acc_empty[b], Cfg::CTAS * I8_EPI_WARPS);
    }
    mbar_init(&sm->drain, 1);
    sm->timeout_cycles = p.timeout_cycles;
    sm->abort_flag = 0;
    sm->bad = 0;
    sm->far = 0;
    fence_barrier_init();
  }
  if (warp == 2) {
    if (PAIR) {
      pair_tmem_alloc(&sm->tmem_base, Cfg::TMEM_COLS);
    } else {
      tmem_alloc(&sm->tmem_base, Cfg::TMEM_COLS);
      tmem_relinquish();
    }
  }
  // what came before on the stream is not waited for until here: the set-up above overlaps it
  grid_dependency_wait();
  // tiles before each group: a block-wide exclusive sum, four consecutive groups per thread
  if (p.groups == 1) {
    if (threadIdx.x == 0) {
      const int64_t rows = i8_row_of(p, 1) - i8_row_of(p, 0);
      sm->first_tile[0] = 0;
      sm->first_tile[1] = rows > 0 ? (int)((rows + BN - 1) / BN) * p.feature_tiles : 0;
    }
  } else {
    constexpr int PER = I8_MAX_GROUPS / I8_SCAN_THREADS;
    const bool scans = threadIdx.x < I8_SCAN_THREADS;
    int cnt[PER], sum = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int g = threadIdx.x * PER + j;
      cnt[j] = 0;
      if (scans && g < p.groups) {
        const int64_t rows = i8_row_of(p, g + 1) - i8_row_of(p, g);
        cnt[j] = rows > 0 ? (int)((rows + BN - 1) / BN) * p.feature_tiles : 0;
      }
      sum = i8_add_tiles(sum, cnt[j]);
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc = i8_add_tiles(inc, v);
    }
    if (scans && lane == 31) sm->scan[warp] = inc;
    const int ahead = __shfl_up_sync(0xffffffffu, inc, 1);
    __syncthreads();
    if (scans) {
      int base = lane > 0 ? ahead : 0;
      for (int w = 0; w < warp; ++w) base = i8_add_tiles(base, sm->scan[w]);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int g = threadIdx.x * PER + j;
        if (g <= p.groups) sm->first_tile[g] = base;
        base = i8_add_tiles(base, cnt[j]);
      }
      if (threadIdx.x == I8_SCAN_THREADS - 1 && p.groups == I8_MAX_GROUPS) sm->first_tile[I8_MAX_GROUPS] = base;
    }
  }
  tc_fence_before();
  if (PAIR) {
    __syncwarp();
    cluster_sync();        // the barriers of both CTAs are set up
  } else {
    __syncthreads();
  }
  tc_fence_after();
  const uint32_t tmem_base = sm->tmem_base;
  const int tiles = sm->first_tile[p.groups];
  const int all_chunks = (p.d + I8_KB - 1) / I8_KB;
  // this CTA's run of the contraction (each has one chunk at least: the host sees to it)
  const int c_begin = SPLIT ? (int)((int64_t)all_chunks * split / splits) : 0;
  const int c_end = SPLIT ? (int)((int64_t)all_chunks * (split + 1) / splits) : all_chunks;

  if (warp == 0) {
    // ------------------------------------------------------------------------ loads
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += step) {
        const I8Tile tile = i8_tile<BN>(p, sm->first_tile, t, wide, skip);
        const int w_row = tile.g * p.n + tile.feature0;
        const int my_rows = Cfg::cols(tile.rows) / 2;        // PAIR: the half of the tokens in this CTA
        for (int c = c_begin; c < c_end; ++c, ++it) {
          const uint32_t s = it % Cfg::STAGES, lap = it / Cfg::STAGES;
          if (!i8_wait(&sm->empty[s], (lap & 1u) ^ 1u, sm)) {
            ok = false;
            break;
          }
          if (PAIR) {
            // both CTAs' bytes count at CTA 0's barrier; its phase needs CTA 0's own arrival as well
            if (in_pair == 0) mbar_expect_tx(&sm->full[s], 2 * (Cfg::A_BYTES + my_rows * I8_KB));
            const uint32_t full0 = address_in(&sm->full[s], 0);
            pair_tma_load(sm->a[s], &map_w, c * I8_KB, w_row, full0);
            if (my_rows == BN / 2)
              pair_tma_load(sm->b[s], &map_x, c * I8_KB, (int)tile.row0 + in_pair * my_rows, full0);
            else
              for (int r = 0; r < my_rows; r += I8_PAIR_BOX)
                pair_tma_load(sm->b[s] + r * I8_KB, &map_tail, c * I8_KB, (int)tile.row0 + in_pair * my_rows + r, full0);
          } else {
            mbar_expect_tx(&sm->full[s], Cfg::A_BYTES + Cfg::B_BYTES);
            tma_load_2d(sm->a[s], &map_w, c * I8_KB, w_row, &sm->full[s]);
            tma_load_2d(sm->b[s], &map_x, c * I8_KB, (int)tile.row0, &sm->full[s]);
          }
          if (p.test_stall && c == c_end - 1 - SPLIT) ok = false;
          if (!ok) {
            ++it;
            break;
          }
        }
      }
      // (CTA 0 of a pair waits for both CTAs' copies, as far as it issued its own; the other one does not
      // leave before it)
      if (sm->abort_flag && in_pair == 0) drain_ring(sm->full, Cfg::STAGES, it);
    }
  } else if (warp == 1 && in_pair == 0) {
    // ------------------------------------------------------------------------- MMAs
    const uint64_t a0 = make_sdesc(smem_u32(sm->a[0])), b0 = make_sdesc(smem_u32(sm->b[0]));
    const int last_steps = ((p.d - (all_chunks - 1) * I8_KB) + 31) / 32;   // 32 features per instruction
    uint32_t it = 0, nt = 0;
    bool ok = true;
    for (int t = first; t < tiles && ok; t += step, ++nt) {
      const uint32_t ab = nt & 1u;
      if (!__all_sync(0xffffffffu, i8_wait<PAIR>(&sm->acc_empty[ab], ((nt >> 1) & 1u) ^ 1u, sm))) break;
      tc_fence_after();
      const uint32_t d_tmem = tmem_base + ab * BN;
      const uint32_t idesc = PAIR ? Cfg::idesc(Cfg::cols(i8_tile<BN>(p, sm->first_tile, t, wide, skip).rows)) : Cfg::idesc(BN);
      for (int c = c_begin; c < c_end; ++c, ++it) {
        const uint32_t s = it % Cfg::STAGES, lap = it / Cfg::STAGES;
        if (!__all_sync(0xffffffffu, i8_wait(&sm->full[s], lap & 1u, sm))) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (elect_one()) {
          const uint64_t ad = a0 + (uint64_t)(s * (Cfg::A_BYTES >> 4));
          const uint64_t bd = b0 + (uint64_t)(s * (Cfg::B_BYTES >> 4));
          const int steps = c == all_chunks - 1 ? last_steps : 4;
          for (int ks = 0; ks < steps; ++ks)
            if (PAIR) pair_umma_i8(d_tmem, ad + 2 * ks, bd + 2 * ks, idesc, (c > c_begin || ks > 0) ? 1u : 0u);
            else umma_i8_ss(d_tmem, ad + 2 * ks, bd + 2 * ks, idesc, (c > c_begin || ks > 0) ? 1u : 0u);
          if (PAIR) {
            pair_commit(&sm->empty[s]);
            if (c == c_end - 1) pair_commit(&sm->acc_full[ab]);
          } else {
            umma_commit(&sm->empty[s]);
            if (c == c_end - 1) umma_commit(&sm->acc_full[ab]);
          }
        }
        __syncwarp();
      }
    }
    if (sm->abort_flag) {
      if (PAIR) {
        if (elect_one()) {
          pair_commit(&sm->drain);
          drain_wait(&sm->drain, 0u);
        }
        __syncwarp();
      } else {
        mma_drain(&sm->drain);
      }
    }
  } else if (warp >= 4) {
    // --------------------------------------------------------------- scales and stores
    const int q = warp & 3, half = (warp - 4) >> 2;
    const int etid = threadIdx.x - 128;
    constexpr int EPI = I8_EPI_WARPS * 32;
    T* out = reinterpret_cast<T*>(p.out);
    if (p.offsets) {
      // rows ahead of the first group and behind the last belong to nobody: zeros
      const int64_t head = i8_row_of(p, 0) * p.n, tail = i8_row_of(p, p.groups) * p.n, all = p.m * p.n;
      for (int64_t e = (int64_t)blockIdx.x * EPI + etid; e < head + (all - tail); e += (int64_t)gridDim.x * EPI)
        out[e < head ? e : tail + (e - head)] = from_float<T>(0.f);
    }
    // columns of this warp: half of the tile's tokens (all, where that would be less than 16)
    constexpr int COLS = BN >= 64 ? 32 : 16;
    constexpr int MINE = BN >= 32 ? BN / 2 : BN;
    const int col0 = BN >= 32 ? half * MINE : 0;
    const bool works = BN >= 32 || half == 0;
    uint32_t nt = 0;
    bool ok = true;        // no wait has run out; one that did says nothing about the phases after it
    for (int t = first; t < tiles; t += step, ++nt) {
      const I8Tile tile = i8_tile<BN>(p, sm->first_tile, t, wide, skip);
      const uint32_t ab = nt & 1u;
      asm volatile("bar.sync 1, 256;" ::: "memory");   // everybody is done with the last tile's scales
      bool far = false;
      for (int r = etid; r < BN; r += EPI) {
        const float sa = r < tile.rows ? p.sa[tile.row0 + r] : 0.f;
        sm->sa[r] = sa;
        far = far || i8_far(sa);
      }
      const int feature = tile.feature0 + q * 32 + lane;
      const bool mine = feature < p.n;
      const int64_t wrow = (int64_t)tile.g * p.n + feature;
      float sb = mine ? p.sb[wrow] : 0.f;
      const float bias = (mine && p.bias) ? p.bias[wrow] : 0.f;
      far = i8_any_of_storing_warps(far);      // and the scales of the tile's tokens are there
      ok = ok && __all_sync(0xffffffffu, i8_wait(&sm->acc_full[ab], (nt >> 1) & 1u, sm));
      tc_fence_after();
      const uint32_t acc = tmem_base + ab * BN + ((uint32_t)(q * 32) << 16);
      if (SPLIT) {
        // partial sums [token][feature] into the stages, which nobody needs any more
        int* part = reinterpret_cast<int*>(sm->a[0]);
        if (!ok && lane == 0) sm->bad = 1;
        if (far && etid == 0) sm->far = 1;
        if (works) {
#pragma unroll 1
          for (int c = 0; c < MINE && col0 + c < tile.rows; c += 16) {
            uint32_t v[16];
            tmem_ld16(acc + col0 + c, v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) part[(col0 + c + j) * I8_BM + q * 32 + lane] = (int)v[j];
          }
        }
      } else {
        if (!ok) sb = __uint_as_float(0x7fffffffu);      // a wait ran out: the tile becomes NaN
        if (works) {
          T* o = out + (tile.row0 + col0) * p.n + feature;
          const int rows = mine ? tile.rows - col0 : 0;
          if (__any_sync(0xffffffffu, far || i8_far(sb))) {
            i8_store_far<T>(acc + col0, MINE < tile.rows - col0 ? MINE : tile.rows - col0, sm->sa + col0, sb, bias, o, p.n, rows);
          } else {
#pragma unroll 1
            for (int c = 0; c < MINE && col0 + c < tile.rows; c += COLS, o += (int64_t)COLS * p.n) {
              uint32_t v[COLS];
              if constexpr (COLS == 32) tmem_ld32(acc + col0 + c, v);
              else tmem_ld16(acc + col0 + c, v);
              tmem_ld_wait();
              if (rows - c >= COLS) i8_store<COLS, true>(v, sm->sa + col0 + c, sb, bias, o, p.n, 0);
              else i8_store<COLS, false>(v, sm->sa + col0 + c, sb, bias, o, p.n, rows - c);
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR) arrive_at(address_in(&sm->acc_empty[ab], 0));
        else mbar_arrive(&sm->acc_empty[ab]);
      }
    }
  }
  tc_fence_before();
  if (PAIR) {
    __syncwarp();
    cluster_sync();        // nothing of either CTA is in the other's hands any more
  } else if (SPLIT) {
    __syncwarp();
    cluster_sync();        // every partial sum of the cluster lies in shared memory
    if (warp >= 4 && first < tiles) {
      const I8Tile tile = i8_tile<BN>(p, sm->first_tile, first);
      const int q = warp & 3, half = (warp - 4) >> 2;
      const int feature = tile.feature0 + q * 32 + lane;
      bool bad = false;
      for (int r = 0; r < splits; ++r) bad = bad || load_from(&sm->bad, r) != 0;
      if (feature < p.n) {
        const int64_t wrow = (int64_t)tile.g * p.n + feature;
        const float sb = bad ? __uint_as_float(0x7fffffffu) : p.sb[wrow];
        const float bias = p.bias ? p.bias[wrow] : 0.f;
        const bool far = sm->far != 0 || i8_far(sb);
        // this warp's tokens: every 2 * splits-th of the tile, AT_ONCE of them in flight from each CTA
        constexpr int AT_ONCE = BN >= 64 ? 8 : 4;
        const int hop = splits * 2;
        const int* part = reinterpret_cast<const int*>(sm->a[0]) + q * 32 + lane;
        for (int c0 = split * 2 + half; c0 < tile.rows; c0 += hop * AT_ONCE) {
          int sum[AT_ONCE];
#pragma unroll
          for (int u = 0; u < AT_ONCE; ++u) sum[u] = 0;
          for (int r = 0; r < splits; ++r) {
            int v[AT_ONCE];
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u)
              v[u] = c0 + u * hop < tile.rows ? load_from(part + (c0 + u * hop) * I8_BM, r) : 0;
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) sum[u] += v[u];
          }
#pragma unroll
          for (int u = 0; u < AT_ONCE; ++u) {
            const int c = c0 + u * hop;
            if (c < tile.rows)
              reinterpret_cast<T*>(p.out)[(tile.row0 + c) * p.n + feature] =
                  far ? i8_scaled<true, T>(sum[u], sm->sa[c], sb, bias) : i8_scaled<false, T>(sum[u], sm->sa[c], sb, bias);
          }
        }
      }
    }
    __syncwarp();
    cluster_sync();        // and nobody reads this CTA's any more
  } else {
    __syncthreads();
  }
  if (warp == 2) {
    tc_fence_after();
    if (PAIR) pair_tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
    else tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
  }
}

// (rows, d) 8-bit row-major matrix at a pitch of ld bytes; box = 128 bytes x box_rows rows.
static int i8_make_map(CUtensorMap* map, const int8_t* base, int64_t rows, int d, int64_t ld, int box_rows) {
  EncodeTiledFn fn = get_encode_fn();
  if (fn == nullptr) {
    set_error("cuTensorMapEncodeTiled is not available from this driver");
    return KMB_ERR_CUDA;
  }
  cuuint64_t dims[2] = {(cuuint64_t)d, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {(cuuint32_t)I8_KB, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void*)base, dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed with CUresult %d (rows=%lld d=%d ld=%lld)", (int)r,
              (long long)rows, d, (long long)ld);
    return KMB_ERR_CUDA;
  }
  return KMB_OK;
}

template <int BN, typename T, I8Mode MODE>
int i8_launch(const CUtensorMap& map_w, const CUtensorMap& map_x, const CUtensorMap& map_tail, const I8Params& p,
              int64_t grid, int cluster, cudaStream_t s) {
  const int smem = (int)sizeof(I8Smem<BN, MODE>) + 1024;
  const auto kernel = int8_matmul_kernel<BN, T, MODE>;
  KMB_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  return launch_early(kernel, (unsigned)grid, I8_THREADS, smem, cluster, s, map_w, map_x, map_tail, p);
}

// How a product is cut: tokens per tile, CTAs per tile, and whether pairs of CTAs work on tiles twice as wide.
struct I8Plan {
  int bn, splits;
  bool pairs;
  int64_t tiles;      // an upper bound: every group may end inside a tile
};

// The cycles of a plan, near enough to choose by.  A CTA goes through `rounds` tiles.  A chunk of the
// contraction takes as long as its bytes take to arrive (60 a cycle and SM) or its products (2 cycles a token);
// a tile's stores overlap the next tile, but not the last one; partial sums in a cluster are stored, fetched and
// added behind the last chunk.  Measured, and by this estimate at 1.85 GHz with 2.7 us for the start (us):
// 500 x 4096 x 4096 with 64, 128, 256 tokens a tile 22.3, 14.8, 17.2 and 18.8, 14.6, 17.8; 128 x 8192 x 2048 with
// 32, 64, 128 12.0, 8.0, 10.6 and 10.2, 8.1, 10.3; 1000 x 1000 x 1000 with 32, 64, 128 7.9, 6.4, 9.4 and 7.4, 6.4,
// 9.1.
static int64_t i8_cycles(const I8Plan& plan, int64_t m, int groups, int feature_tiles, int chunks, int sms) {
  // tiles to expect: half a tile is lost at the end of each group
  int64_t token_tiles = groups == 1 ? ceil_div(m, plan.bn) : m / plan.bn + groups / 2;
  const int64_t busy = m < groups ? m : groups;
  if (token_tiles < busy) token_tiles = busy;
  const int64_t tiles = token_tiles * feature_tiles;
  const int64_t workers = plan.pairs ? sms / 2 : sms;
  const int64_t rounds = plan.splits > 1 ? 1 : ceil_div(tiles, workers);
  const int64_t bytes = I8_BM * I8_KB + (int64_t)plan.bn * I8_KB / (plan.pairs ? 2 : 1);
  const int64_t chunk = bytes / 60 > 2 * plan.bn ? bytes / 60 : 2 * plan.bn;
  const int64_t work = ceil_div(chunks, plan.splits) * chunk;
  const int64_t store = plan.splits > 1 ? 4500 + 40 * plan.bn : 2500 + 16 * plan.bn;
  return rounds * work + store + (rounds - 1) * (store > work ? store - work : 0);
}

static I8Plan i8_plan(int64_t m, int groups, int n, int d) {
  const int sms = sm_count(), chunks = (d + I8_KB - 1) / I8_KB;
  I8Plan best = {};
  int64_t least = 0;
  for (int bn = 16; bn <= 256; bn *= 2) {
    const int64_t token_tiles = ceil_div(m, bn) + groups - 1;
    I8Plan plan;
    plan.bn = bn;
    plan.splits = 1;
    // pairs where there is a wide tile for each of them
    plan.pairs = bn == 256 && n > I8_BM && token_tiles * ceil_div(n, 2 * I8_BM) >= sms / 2;
    const int64_t feature_tiles = ceil_div(n, plan.pairs ? 2 * I8_BM : I8_BM);
    plan.tiles = token_tiles * feature_tiles;
    // CTAs that share a tile: as many as there are SMs for, while each has two chunks at least.  SMs come in
    // groups of uneven size: of 148, 15 clusters of eight and 33 of four find room at once.
    if (!plan.pairs)
      for (int s = 8; s > 1 && plan.splits == 1; s >>= 1) {
        const int64_t room = s == 8 ? sms / 8 * 5 / 6 : s == 4 ? sms / 4 * 9 / 10 : sms / 2;
        if (plan.tiles <= room && chunks >= 2 * s) plan.splits = s;
      }
    const int64_t c = i8_cycles(plan, m, groups, (int)feature_tiles, chunks, sms);
    if (bn == 16 || c < least) {
      least = c;
      best = plan;
    }
    if (bn >= m) break;       // wider tiles would be no fuller
  }
  return best;
}

template <int BN, typename T>
int i8_run_as(const I8Plan& plan, const int8_t* a, int64_t lda, const int8_t* b, int64_t ldb, I8Params p,
              cudaStream_t s) {
  KMB_REQUIRE(plan.tiles < I8_MAX_TILES, "kmb_int8_matmul: too many output tiles");
  const int sms = sm_count();
  CUtensorMap map_w, map_x;
  int rc = i8_make_map(&map_w, b, (int64_t)p.groups * p.n, p.d, ldb, I8_BM);
  if (rc != KMB_OK) return rc;
  rc = i8_make_map(&map_x, a, p.m, p.d, lda, plan.pairs ? BN / 2 : BN);
  if (rc != KMB_OK) return rc;
  CUtensorMap map_tail = map_x;
  if (plan.pairs) rc = i8_make_map(&map_tail, a, p.m, p.d, lda, I8_PAIR_BOX);
  if (rc != KMB_OK) return rc;
  p.feature_tiles = (int)ceil_div(p.n, plan.pairs ? 2 * I8_BM : I8_BM);
  if constexpr (BN == 256)
    if (plan.pairs) return i8_launch<BN, T, I8_PAIR>(map_w, map_x, map_tail, p, sms / 2 * 2, 2, s);
  if (plan.splits > 1)
    return i8_launch<BN, T, I8_SPLIT>(map_w, map_x, map_tail, p, plan.tiles * plan.splits, plan.splits, s);
  return i8_launch<BN, T, I8_SINGLE>(map_w, map_x, map_tail, p, plan.tiles < sms ? plan.tiles : sms, 1, s);
}

template <int BN>
int i8_run(const I8Plan& plan, int out_dtype, const int8_t* a, int64_t lda, const int8_t* b, int64_t ldb,
           const I8Params& p, cudaStream_t s) {
  if (out_dtype == KMB_F32) return i8_run_as<BN, float>(plan, a, lda, b, ldb, p, s);
  if (out_dtype == KMB_F16) return i8_run_as<BN, __half>(plan, a, lda, b, ldb, p, s);
  return i8_run_as<BN, __nv_bfloat16>(plan, a, lda, b, ldb, p, s);
}

}  // namespace kmb

using namespace kmb;

extern "C" {

int kmb_quantize_rows(int dtype, const void* x, int64_t n, int d, const int32_t* rows, int64_t m,
                      int8_t* q, int64_t q_pitch, float* scales, void* stream) {
  KMB_REQUIRE(n >= 0 && d > 0 && m >= 0 && m < (1ll << 31), "kmb_quantize_rows: bad sizes");
  KMB_REQUIRE(d < (1 << 30), "kmb_quantize_rows: d must be below 2^30");
  KMB_REQUIRE(rows != nullptr || m == n, "kmb_quantize_rows: m must be n when no rows are named");
  if (m == 0) return KMB_OK;
  KMB_REQUIRE((x || n == 0) && q && scales, "kmb_quantize_rows: NULL argument");
  KMB_REQUIRE(q_pitch >= d && q_pitch % 16 == 0 && ((uintptr_t)q & 15) == 0,
              "kmb_quantize_rows: q must be 16-byte aligned with a pitch of a multiple of 16, at least d");
  KMB_DISPATCH_ROWS(dtype, {
    return quantize_run<T>((const T*)x, n, d, rows, m, q, q_pitch, scales, (cudaStream_t)stream);
  });
}

int kmb_int8_matmul(int out_dtype, const int8_t* a, int64_t lda, const float* a_scales, const int8_t* b,
                    int64_t ldb, const float* b_scales, const float* bias, const int32_t* offsets,
                    int groups, void* out, int64_t m, int n, int d, void* stream) {
  KMB_REQUIRE(out_dtype == KMB_F32 || out_dtype == KMB_F16 || out_dtype == KMB_BF16,
              "kmb_int8_matmul: out_dtype must be KMB_F32, KMB_F16 or KMB_BF16, got %d", out_dtype);
  KMB_REQUIRE(m >= 0 && m < (1ll << 31) - 256 && n > 0 && d > 0, "kmb_int8_matmul: bad sizes");
  KMB_REQUIRE(d <= 131071, "kmb_int8_matmul: d must be at most 131071 (int32 sums), got %d", d);
  KMB_REQUIRE(groups >= 1 && groups <= I8_MAX_GROUPS && (offsets || groups == 1),
              "kmb_int8_matmul: groups must be in [1, %d], and 1 without offsets", I8_MAX_GROUPS);
  KMB_REQUIRE((int64_t)groups * n < (1ll << 31) - 256, "kmb_int8_matmul: groups * n must be below 2^31");
  if (m == 0) return KMB_OK;
  KMB_REQUIRE(a && a_scales && b && b_scales && out, "kmb_int8_matmul: NULL argument");
  KMB_REQUIRE(lda >= d && lda % 16 == 0 && ldb >= d && ldb % 16 == 0 && ((uintptr_t)a & 15) == 0 &&
                  ((uintptr_t)b & 15) == 0,
              "kmb_int8_matmul: a and b must be 16-byte aligned with row pitches of a multiple of 16");
  I8Params p;
  p.sa = a_scales;
  p.sb = b_scales;
  p.bias = bias;
  p.offsets = offsets;
  p.out = out;
  p.m = m;
  p.groups = groups;
  p.n = n;
  p.d = d;
  const char* e = getenv("KMB_TC_TIMEOUT_MS");
  const long ms = e ? atol(e) : 0;
  p.timeout_cycles = ms > 0 ? ms * 2000000LL : I8_TIMEOUT_CYCLES;
  e = getenv("KMB_TC_TEST_STALL");
  p.test_stall = e && atoi(e) != 0;
  cudaStream_t s = (cudaStream_t)stream;
  const I8Plan plan = i8_plan(m, groups, n, d);
  switch (plan.bn) {
    case 16: return i8_run<16>(plan, out_dtype, a, lda, b, ldb, p, s);
    case 32: return i8_run<32>(plan, out_dtype, a, lda, b, ldb, p, s);
    case 64: return i8_run<64>(plan, out_dtype, a, lda, b, ldb, p, s);
    case 128: return i8_run<128>(plan, out_dtype, a, lda, b, ldb, p, s);
    default: return i8_run<256>(plan, out_dtype, a, lda, b, ldb, p, s);
  }
}

int kmb_int8_wait_error(int* flag, void* stream) {
  KMB_REQUIRE(flag, "kmb_int8_wait_error: NULL argument");
  cudaStream_t s = (cudaStream_t)stream;
  const int zero = 0;
  *flag = 0;
  KMB_CHECK_CUDA(cudaMemcpyFromSymbolAsync(flag, g_i8_wait_error, sizeof(int), 0, cudaMemcpyDeviceToHost, s));
  KMB_CHECK_CUDA(cudaStreamSynchronize(s));
  if (*flag) {
    KMB_CHECK_CUDA(cudaMemcpyToSymbolAsync(g_i8_wait_error, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, s));
    KMB_CHECK_CUDA(cudaStreamSynchronize(s));
    set_error("a bounded wait of the 8-bit product ran out: its tiles were filled with NaN");
    return KMB_ERR_CUDA;
  }
  return KMB_OK;
}

}  // extern "C"
