// Matrix product in 8-bit integers with one scale a token and one a channel:
//   y[m, n] = (sum_k a[m, k] b[n, k]) * (sa[m] * sb[n]) + bias[n]
// and the quantisation that feeds it, row by row:
//   s = max_k |x_k| / 127,  code_k = rint(x_k * (127 / max))
// (all in fp32; the product of x and the reciprocal is rounded once, then to the
// nearest integer, ties to even). The integer sum is exact (K <= 131071 keeps it
// inside 32 bits), so neither the order of the sum nor a split of K can change a
// bit of y; what rounds is the conversion of the sum, the two products and the
// bias, each once.
//
// Both products run on the 8-bit tensor cores (tcgen05 kind::i8, 32-bit integer
// accumulators in TMEM, operands by TMA in 128-byte swizzled rows, K-major on
// both sides, as activations and nn.Linear weights lie). Two kernels:
//   narrow: few tokens. The weights stream once, so the kernel is bound by
//     memory; weight rows take the 128 accumulator lanes (they are the long
//     side) and 16 .. 128 tokens the columns. Two persistent CTAs an SM walk the
//     tiles, the next one's operands loading under this one's epilogue. Where the
//     tiles do not fill the machine, a cluster of 2 .. 8 CTAs splits K and adds its
//     integer partials through distributed shared memory. Measured, 32 tokens, K =
//     2048, N = 128256 with the quantisation: 48 us, 5.7 TB/s.
//   wide: many tokens. Bound by the tensor cores. A pair of CTAs (cta_group::2)
//     shares a 256 x 256 tile: each loads half of either operand, so a byte in
//     shared memory feeds twice the math; two accumulators of 256 TMEM columns
//     let the epilogue of a tile run under the next one's products. Measured, M =
//     32768, K = 8192, N = 2048: 321 us, 3.43 POP/s, the tensor pipe active 86 % of the
//     time, and 115 us for the quantisation before it. A form that quantised
//     in four more warps of this kernel, rows dealt over all CTAs in the order of the
//     tiles, took 484 us against 442 for the two launches: the rows are long waits for
//     few warps, and their traffic slows the operands'.
#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "tc.cuh"

namespace lz {
namespace {

constexpr int kMaxK = 131071;  // 128 * 128 * K < 2^31

__device__ __forceinline__ void launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
}

// ------------------------------------------------------------------ quantise
constexpr int kQT = 256;   // threads a CTA

template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ uint32_t top(const uint4& w) {  // largest |bits|
    return max(max(w.x & 0x7fffffffu, w.y & 0x7fffffffu), max(w.z & 0x7fffffffu, w.w & 0x7fffffffu));
  }
  static __device__ __forceinline__ float value(const float* p) { return *p; }
};
template <>
struct Vec<bf16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ uint32_t top(const uint4& w) {
    constexpr uint32_t m = 0x7fff7fffu;
    const uint32_t x = __vmaxu2(__vmaxu2(w.x & m, w.y & m), __vmaxu2(w.z & m, w.w & m));
    return max(x & 0xffff0000u, x << 16);  // as fp32 bits
  }
  static __device__ __forceinline__ float value(const bf16* p) { return __bfloat162float(*p); }
};

// One code: the product rounded to fp32, then to an integer by adding 1.5 * 2^23.
__device__ __forceinline__ uint32_t code_of(float x, float inv) {
  return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.f));
}
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// The codes of 16 bytes of x, the first in the lowest byte.
__device__ __forceinline__ uint32_t codes_of(const uint4& w, float inv, float) {
  return pack4(code_of(__uint_as_float(w.x), inv), code_of(__uint_as_float(w.y), inv),
               code_of(__uint_as_float(w.z), inv), code_of(__uint_as_float(w.w), inv));
}
__device__ __forceinline__ unsigned long long codes_of(const uint4& w, float inv, bf16) {
  return pack4(code_of(bf16_lo(w.x), inv), code_of(bf16_hi(w.x), inv),
               code_of(bf16_lo(w.y), inv), code_of(bf16_hi(w.y), inv)) |
         (unsigned long long)pack4(code_of(bf16_lo(w.z), inv), code_of(bf16_hi(w.z), inv),
                                   code_of(bf16_lo(w.w), inv), code_of(bf16_hi(w.w), inv)) << 32;
}
// Word `at` of the codes of a row that does not start on 16 bytes (`head` values, then the
// nv vectors rv): the last `head` codes of the vector before and the first ones of w,
// vector `at`. By a whole warp with consecutive `at`.
template <typename T>
__device__ __forceinline__ auto code_word(const T* row, const uint4* rv, int head, int nv, int at,
                                          const uint4& w, float inv) {
  constexpr int N = Vec<T>::N;
  auto cur = codes_of(w, inv, T()), before = __shfl_up_sync(0xffffffffu, cur, 1);
  if ((threadIdx.x & 31) == 0 && at < nv) {
    before = 0;
    if (at)
      before = codes_of(__ldg(rv + at - 1), inv, T());
    else
      for (int k = 0; k < head; ++k)
        before |= (decltype(cur))(code_of(Vec<T>::value(row + k), inv) & 0xffu)
                  << 8 * (N - head + k);
  }
  return cur << 8 * head | before >> 8 * (N - head);
}
template <typename T>
__device__ __forceinline__ int head_of(const T* row, int K) {
  return min(K, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15) & 15) / sizeof(T)));
}

// ROW threads a row (a warp for short rows, the CTA for long ones): the row is read
// once into registers, KEEP 16-byte vectors a thread (the part beyond twice). A row
// that does not start on 16 bytes has a head of a few values before its vectors; codes
// still leave in whole words, put together from two neighbours' vectors. The largest |x| is taken on the bits, where
// infinities and NaN are larger than every number: such a row gets the scale NaN, and
// so NaN outputs. Bound by memory: 32768 rows of 8192 bf16 in 117 us, 6.9 TB/s.
template <typename T, int ROW, int KEEP>
__global__ void __launch_bounds__(kQT)
i8_quantize_kernel(const T* __restrict__ x, long long ldx, int8_t* __restrict__ codes,
                   long long ldc, float* __restrict__ scale, int M, int K) {
  using V = Vec<T>;
  __shared__ uint32_t sTop[kQT / 32];
  launch_dependents();  // the product's CTAs may start on the weights
  const int tid = threadIdx.x % ROW;
  const long long m = (long long)blockIdx.x * (kQT / ROW) + threadIdx.x / ROW;
  if (m >= M) return;  // whole warps
  const T* row = x + m * ldx;
  int8_t* out = codes + m * ldc;
  const int head = head_of(row, K), nv = (K - head) / V::N;
  const uint4* rv = reinterpret_cast<const uint4*>(row + head);
  uint4 keep[KEEP];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < KEEP; ++i) {
    const int at = tid + i * ROW;
    keep[i] = at < nv ? __ldg(rv + at) : make_uint4(0, 0, 0, 0);
  }
  if (tid < head) top = __float_as_uint(V::value(row + tid)) & 0x7fffffffu;
#pragma unroll
  for (int i = 0; i < KEEP; ++i) top = max(top, V::top(keep[i]));
  for (int at = tid + KEEP * ROW; at < nv; at += ROW) top = max(top, V::top(rv[at]));
  for (int k = head + nv * V::N + tid; k < K; k += ROW)
    top = max(top, __float_as_uint(V::value(row + k)) & 0x7fffffffu);
  top = __reduce_max_sync(0xffffffffu, top);
  if constexpr (ROW == kQT) {
    if ((tid & 31) == 0) sTop[tid >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kQT / 32; ++w) top = max(top, sTop[w]);
  }
  const float t = __uint_as_float(top);
  // below 4e-37 the reciprocal leaves the fp32 range: the row counts as zero
  const bool live = t >= 4e-37f && t < INFINITY;
  const float inv = live ? 127.f / t : 0.f;
  if (tid == 0) scale[m] = live ? t / 127.f : (t < 1.f ? 0.f : __uint_as_float(0x7fc00000u));
  if (!live) {
    for (int k = tid; k < ldc; k += ROW) out[k] = 0;
    return;
  }
  const auto put = [&](int at, decltype(codes_of(keep[0], inv, T())) c) {
    if (at < nv) *reinterpret_cast<decltype(c)*>(out + at * V::N) = c;
  };
  if (head == 0) {
#pragma unroll
    for (int i = 0; i < KEEP; ++i) put(tid + i * ROW, codes_of(keep[i], inv, T()));
    for (int at = tid + KEEP * ROW; at < nv; at += ROW) put(at, codes_of(rv[at], inv, T()));
  } else {
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      put(tid + i * ROW, code_word(row, rv, head, nv, tid + i * ROW, keep[i], inv));
    for (int at0 = (tid & ~31) + KEEP * ROW; at0 < nv; at0 += ROW) {
      const int at = at0 + (tid & 31);
      put(at, code_word(row, rv, head, nv, at, at < nv ? rv[at] : make_uint4(0, 0, 0, 0), inv));
    }
  }
  for (int k = nv * V::N + tid; k < K; k += ROW)
    out[k] = (int8_t)(code_of(V::value(row + k), inv) & 0xffu);
  for (int k = K + tid; k < ldc; k += ROW) out[k] = 0;
}

// Rows of codes that do not start on 16 bytes, copied to ones that do.
__global__ void __launch_bounds__(kQT)
i8_repack_kernel(const int8_t* __restrict__ x, long long ldx, int8_t* __restrict__ out,
                 long long ldo, int K) {
  const int8_t* row = x + (size_t)blockIdx.x * ldx;
  int8_t* o = out + (size_t)blockIdx.x * ldo;
  for (int k = threadIdx.x; k < ldo; k += kQT) o[k] = k < K ? row[k] : 0;
}

// ---------------------------------------------------------------------- PTX
__device__ __forceinline__ void grid_dependency_wait() {
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
}
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void mma_i8_pair(uint32_t d, uint64_t adesc, uint64_t bdesc,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
// Signed 8-bit x signed 8-bit -> 32-bit integer, both operands K-major.
__host__ __device__ constexpr uint32_t idesc_i8(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int c0, int c1,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];\n" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(smem_u32(bar))
      : "memory");
}
// The same into this CTA's shared memory, completing on a barrier of the pair
// (a shared::cluster address).
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, int c0, int c1,
                                                 uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::"
      "bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int c0,
                                             int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];\n" ::"l"(
          reinterpret_cast<uint64_t>(map)),
      "r"(smem_u32(src)), "r"(c0), "r"(c1)
      : "memory");
}
// Arrive on the barrier at the same offset in both CTAs of the pair once every
// MMA issued so far has completed.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
      "[%0], %1;\n" ::"r"(smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void arrive_remote(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(bar)
               : "memory");
}
__device__ __forceinline__ int4 ld_cluster_int4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::
                   : "memory");
}

struct Out {  // y and what scales it
  const float *sa, *sb;
  const void* bias;  // [N] fp32 or bf16, or null
  void* y;           // [M, N] contiguous, fp32 or bf16
  int bias_bf16, y_bf16, M, N, K;
  const void* x;  // x itself, rows ldx elements apart, where the product quantises it
  long long ldx;
  int x_bf16;
  int withhold;  // a test: one load of the first stage is not issued
};
__device__ __forceinline__ float bias_at(const Out& o, int n) {
  if (!o.bias) return 0.f;
  return o.bias_bf16 ? __bfloat162float(static_cast<const bf16*>(o.bias)[n])
                     : static_cast<const float*>(o.bias)[n];
}
__device__ __forceinline__ float scaled(int acc, float sa, float sb, float bias) {
  return __fadd_rn(__fmul_rn(__int2float_rn(acc), __fmul_rn(sa, sb)), bias);
}

// -------------------------------------------------------------------- narrow
constexpr int kNStaging = 8192;  // bytes of y on their way out: 32 tokens x 128 channels (bf16)
constexpr int kNoSum = -2147483647 - 1;  // no sum of K <= kMaxK products: a CTA of a split gave up
constexpr int kFuseK = 4096;  // the largest K whose tokens a CTA quantises by itself
template <int BN, bool FUSE>
struct Narrow {
  static constexpr int kStages = BN <= 32 ? 5 : BN == 64 ? 4 : 3;
  static constexpr int kA = 128 * 128, kB = BN * 128;
  static constexpr int kStage = kA + (FUSE ? 0 : kB);
  static constexpr int kCols = BN < 32 ? 32 : BN;  // TMEM columns of an accumulator
  // operand stages (the partials of a split reuse them), staging, token scales,
  // barriers, TMEM address; with FUSE the codes of `steps` steps of K besides
  static constexpr size_t smem(int steps) {
    return 1024 + (size_t)kStages * kStage + kNStaging + (FUSE ? (size_t)steps * kB : 0) +
           2 * BN * 4 + 256;
  }
  static_assert((size_t)kStages * kStage >= (size_t)BN * 128 * 4, "partials fit");
  static_assert(FUSE || smem(0) <= 115712, "two CTAs an SM");
};

// The tokens of a small call, quantised by the CTA that multiplies them: rows M of x,
// codes of columns k0 .. k1 to the swizzled K-major tiles at `codes` ([step][BN]
// rows of 128 bytes), scales to sa. By 128 threads, a warp a row, 8 vectors of 16
// bytes a lane kept (the rest is read twice: registers for all of it would leave one
// CTA an SM, and clusters of eight then no longer all fit at once). The same
// arithmetic as i8_quantize_kernel.
template <typename T, int BN>
__device__ __forceinline__ void quantize_here(const T* x, long long ldx, int M, int K, int k0,
                                              int k1, unsigned char* codes, float* sa) {
  using V = Vec<T>;
  constexpr int KEEP = 8;
  const int lane = threadIdx.x & 31, w = (threadIdx.x >> 5) & 3;
  const auto at = [&](int m, int k) {
    const int c = k - k0;
    return codes + (c >> 7) * (BN * 128) + m * 128 + ((((c >> 4) & 7) ^ (m & 7)) << 4) + (c & 15);
  };
  for (int m = w; m < M; m += 4) {
    const T* row = x + m * ldx;
    const int head = head_of(row, K), nv = (K - head) / V::N;
    const uint4* rv = reinterpret_cast<const uint4*>(row + head);
    uint4 keep[KEEP];
    uint32_t top = lane < head ? __float_as_uint(V::value(row + lane)) & 0x7fffffffu : 0;
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      keep[i] = lane + 32 * i < nv ? __ldg(rv + lane + 32 * i) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < KEEP; ++i) top = max(top, V::top(keep[i]));
    for (int i = lane + 32 * KEEP; i < nv; i += 32) top = max(top, V::top(__ldg(rv + i)));
    for (int k = head + nv * V::N + lane; k < K; k += 32)
      top = max(top, __float_as_uint(V::value(row + k)) & 0x7fffffffu);
    top = __reduce_max_sync(0xffffffffu, top);
    const float t = __uint_as_float(top);
    const bool live = t >= 4e-37f && t < INFINITY;
    const float inv = live ? 127.f / t : 0.f;
    if (lane == 0) sa[m] = live ? t / 127.f : (t < 1.f ? 0.f : __uint_as_float(0x7fc00000u));
    if (!live) {
      for (int k = k0 + lane; k < k1; k += 32) *at(m, k) = 0;
      continue;
    }
    const auto put = [&](int i, decltype(codes_of(keep[0], inv, T())) c) {
      const int k = i * V::N;
      if (i < nv && k >= k0 && k < k1) *reinterpret_cast<decltype(c)*>(at(m, k)) = c;
    };
    if (head == 0) {
#pragma unroll
      for (int i = 0; i < KEEP; ++i) put(lane + 32 * i, codes_of(keep[i], inv, T()));
      for (int i = lane + 32 * KEEP; i < nv; i += 32) put(i, codes_of(__ldg(rv + i), inv, T()));
    } else {  // read again: the kept vectors in registers would weigh on the rows above
#pragma unroll 2
      for (int i = lane; i < (nv + 31 & ~31); i += 32)
        put(i, code_word(row, rv, head, nv, i, i < nv ? __ldg(rv + i) : make_uint4(0, 0, 0, 0),
                         inv));
    }
    for (int k = nv * V::N + lane; k < K; k += 32)
      if (k >= k0 && k < k1)
        *at(m, k) = (unsigned char)(code_of(V::value(row + k), inv) & 0xffu);
  }
}

// `rows` values 128 apart in shared memory to a column of y, eight on their way at once.
template <typename T>
__device__ __forceinline__ void copy_column(T* y, int N, const T* from, int rows) {
  for (int r0 = 0; r0 < rows; r0 += 8) {
    T v[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) v[r] = from[min(r0 + r, rows - 1) * 128];
#pragma unroll
    for (int r = 0; r < 8; ++r, y += N)
      if (r0 + r < rows) *y = v[r];
  }
}

// By the multiplying thread that leaves its loop after `steps` steps: waits (with a limit
// again) for its products and for the loads of the ring of S stages, which are that far
// ahead of it at most, so that none is on its way when the CTA leaves.
__device__ __noinline__ void in_flight(uint64_t* full, uint64_t* empty, uint32_t S, uint32_t steps) {
  if (steps) tc::mbar_wait(empty + (steps - 1) % S, ((steps - 1) / S) & 1, 126);
  for (uint32_t i = steps; i < steps + S; ++i) tc::mbar_wait(full + i % S, (i / S) & 1, 127);
}

// Warps: 0 TMA, 1 MMA (and TMEM), 2..5 epilogue. split == 1: a CTA walks the (weight
// tile, token tile) pairs blockIdx.x, + gridDim.x, ..., weight tiles fastest. split
// > 1: clusters of `split` CTAs, one tile each, K dealt over the cluster. FUSE: x
// itself comes in o.x, and the epilogue warps quantise it while the weights load: one
// launch instead of two, for the few tokens of a decode step (M <= 4, K <= kFuseK).
// A wait that gives up: the loading and the multiplying thread leave their loops, the
// latter once nothing is in flight, the epilogue goes through all its barriers, and nothing
// is written from then on.
template <int BN, bool FUSE>
__global__ void __launch_bounds__(192)
i8_narrow_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tx,
                 const __grid_constant__ CUtensorMap ty, const Out o, const int split,
                 const int ytma) {
  using P = Narrow<BN, FUSE>;
  constexpr int S = P::kStages;
  extern __shared__ unsigned char raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* staging = sm + (size_t)S * P::kStage;
  unsigned char* codes = staging + kNStaging;  // FUSE: [nk][BN] rows of 128 bytes
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = split > 1 ? blockIdx.x % split : 0;
  const int wt = (o.N + 127) >> 7, tiles = wt * ((o.M + BN - 1) / BN);
  const int first = blockIdx.x / split, stride = gridDim.x / split;
  const int KT = (o.K + 127) >> 7;
  const int kt0 = split > 1 ? KT * rank / split : 0;
  const int nk = (split > 1 ? KT * (rank + 1) / split : KT) - kt0;
  float* sSa = reinterpret_cast<float*>(codes + (FUSE ? nk * P::kB : 0));  // [2][BN] token scales
  uint64_t* full = reinterpret_cast<uint64_t*>(sSa + 2 * BN);
  uint64_t* empty = full + S;
  uint64_t* acc_full = empty + S;      // [2]
  uint64_t* acc_empty = acc_full + 2;  // [2]
  uint64_t* xready = acc_empty + 2;    // FUSE: the four quantising warps
  uint32_t* tptr = reinterpret_cast<uint32_t*>(xready + 1);
  volatile int* gave_up = reinterpret_cast<volatile int*>(tptr + 1);  // an epilogue wait did
  if (tid == 0) {
    *gave_up = 0;
    tc::mbar_init(xready, 4);
    for (int s = 0; s < S; ++s) tc::mbar_init(full + s, 1), tc::mbar_init(empty + s, 1);
    for (int i = 0; i < 2; ++i) tc::mbar_init(acc_full + i, 1), tc::mbar_init(acc_empty + i, 4);
    tc::fence_mbar_init();
    tc::prefetch_tmap(&tw);
    tc::prefetch_tmap(&tx);
    tc::prefetch_tmap(&ty);
  }
  if (warp == 1) {
    tc::tmem_alloc(tptr, 2 * P::kCols);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tptr;

  if constexpr (FUSE) {
    if (warp >= 2) {
      const int k0 = kt0 * 128, k1 = min(o.K, (kt0 + nk) * 128);
      if (o.x_bf16)
        quantize_here<bf16, BN>(static_cast<const bf16*>(o.x), o.ldx, o.M, o.K, k0, k1, codes, sSa);
      else
        quantize_here<float, BN>(static_cast<const float*>(o.x), o.ldx, o.M, o.K, k0, k1, codes,
                                 sSa);
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(xready);
      tc::named_bar_sync(2, 128);  // the scales are there
    }
  }
  if (warp == 0 && lane == 0) {
    // the weights of the first stages do not depend on the launch before (the
    // quantisation of x): they load while it ends
    const int pre = min(nk, S), n0 = first % wt * 128;
    for (int i = 0; i < pre; ++i) {
      tc::mbar_expect_tx(full + i, P::kStage);
      if (i || !o.withhold)
        tma_load_2d(sm + (size_t)i * P::kStage, &tw, (kt0 + i) * 128, n0, full + i);
    }
    grid_dependency_wait();
    uint32_t it = 0;
    bool ok = true;
    for (int t = first; ok && t < tiles; t += stride) {
      const int n = t % wt * 128, m = t / wt * BN;
      for (int k = 0; k < nk; ++k, ++it) {
        const int s = it % S;
        unsigned char* st = sm + (size_t)s * P::kStage;
        if (it >= (uint32_t)pre) {
          if (it >= S && !(ok = tc::mbar_wait(empty + s, (it / S - 1) & 1, 120))) break;
          tc::mbar_expect_tx(full + s, P::kStage);
          tma_load_2d(st, &tw, (kt0 + k) * 128, n, full + s);
        }
        if constexpr (!FUSE) tma_load_2d(st + P::kA, &tx, (kt0 + k) * 128, m, full + s);
      }
    }
  } else if (warp == 1 && lane == 0) {
    constexpr uint32_t idesc = idesc_i8(128, BN);
    uint32_t it = 0, at = 0;
    bool ok = true;
    if constexpr (FUSE) ok = tc::mbar_wait(xready, 0, 125);
    for (int t = first; ok && t < tiles; t += stride, ++at) {
      const int buf = at & 1;
      if (at >= 2 && !(ok = tc::mbar_wait(acc_empty + buf, (at / 2 - 1) & 1, 123))) break;
      tc::tc_fence_after();
      for (int k = 0; k < nk; ++k, ++it) {
        const int s = it % S;
        if (!(ok = tc::mbar_wait(full + s, (it / S) & 1, 121))) break;
        tc::tc_fence_after();
        const uint32_t a0 = smem_u32(sm + (size_t)s * P::kStage);
        const uint64_t ad = tc::sdesc(a0, 0, 1024);
        const uint64_t bd =
            tc::sdesc(FUSE ? smem_u32(codes + k * P::kB) : a0 + P::kA, 0, 1024);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          mma_i8(tmem + buf * P::kCols, ad + 2 * q, bd + 2 * q, idesc, (k | q) != 0);
        tc::mma_commit(empty + s);
      }
      if (ok) tc::mma_commit(acc_full + buf);
    }
    if (!ok) in_flight(full, empty, S, it);
  } else if (warp >= 2 && split == 1) {
    const int quad = warp & 3, ch = quad * 32 + lane;  // lane = weight row n0 + ch
    const int es = o.y_bf16 ? 2 : 4, chunk = min(BN, kNStaging / (128 * es));
    grid_dependency_wait();
    uint32_t at = 0;
    for (int t = first; t < tiles; t += stride, ++at) {
      const int buf = at & 1, n0 = t % wt * 128, m0 = t / wt * BN, n = n0 + ch;
      const float sb = n < o.N ? o.sb[n] : 0.f, bias = n < o.N ? bias_at(o, n) : 0.f;
      float* sa = FUSE ? sSa : sSa + buf * BN;
      if constexpr (!FUSE)
        for (int i = tid - 64; i < BN; i += 128) sa[i] = m0 + i < o.M ? o.sa[m0 + i] : 0.f;
      if (!tc::mbar_wait(acc_full + buf, (at / 2) & 1, 122)) {
        *gave_up = 1;
        tc::mbar_wait(acc_full + buf, (at / 2) & 1, 122);  // no product is left on its way
      }
      tc::tc_fence_after();
      const int mt = min(BN, o.M - m0);
      for (int c0 = 0; c0 < mt; c0 += chunk) {
        if (tid == 64) tc::bulk_wait_read0();  // the store before has left the staging
        tc::named_bar_sync(1, 128);            // (and the scales are there)
        for (int c1 = 0; c1 < chunk; c1 += 16) {
          float v[16];
          tc::tmem_ld16(tmem + buf * P::kCols + ((uint32_t)(quad * 32) << 16) + c0 + c1, v);
          tc::tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < 16; c += 4) {
            const float4 s4 = *reinterpret_cast<const float4*>(sa + c0 + c1 + c);
            const float ss[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float y = scaled(__float_as_int(v[c + e]), ss[e], sb, bias);
              if (o.y_bf16)
                reinterpret_cast<bf16*>(staging)[(c1 + c + e) * 128 + ch] = __float2bfloat16_rn(y);
              else
                reinterpret_cast<float*>(staging)[(c1 + c + e) * 128 + ch] = y;
            }
          }
        }
        if (c0 + chunk >= mt) {  // the accumulator has been read
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(acc_empty + buf);
        }
        if (ytma) {
          tc::fence_proxy_async_smem();
          tc::named_bar_sync(1, 128);
          if (tid == 64 && !*gave_up) {
            tma_store_2d(&ty, staging, n0, m0 + c0);
            tc::bulk_commit();
          }
        } else {
          tc::named_bar_sync(1, 128);
          if (n < o.N && !*gave_up) {
            const int rows = min(chunk, mt - c0);
            const size_t at = (size_t)(m0 + c0) * o.N + n;
            if (o.y_bf16)
              copy_column(static_cast<bf16*>(o.y) + at, o.N,
                          reinterpret_cast<const bf16*>(staging) + ch, rows);
            else
              copy_column(static_cast<float*>(o.y) + at, o.N,
                          reinterpret_cast<const float*>(staging) + ch, rows);
          }
        }
      }
    }
    if (tid == 64) tc::bulk_wait0();
  }
  __syncwarp();
  if (split > 1) {  // one tile: n0, m0
    const int n0 = first % wt * 128, m0 = first / wt * BN;
    int* part = reinterpret_cast<int*>(sm);  // [BN][128], once every load has been consumed
    if (warp >= 2) {
      const int quad = warp & 3;
      grid_dependency_wait();
      const bool live = __all_sync(0xffffffffu, tc::mbar_wait(acc_full, 0, 124));
      if (!live) tc::mbar_wait(acc_full, 0, 124);
      tc::tc_fence_after();
#pragma unroll 1
      for (int c0 = 0; c0 < BN; c0 += 16) {
        float v[16];
        tc::tmem_ld16(tmem + ((uint32_t)(quad * 32) << 16) + c0, v);
        tc::tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 16; ++c)
          part[(c0 + c) * 128 + quad * 32 + lane] = live ? __float_as_int(v[c]) : kNoSum;
      }
    }
    cluster_sync();
    // the tile's token x channel elements in fours, dealt to the CTAs of the cluster
    const int mt = min(BN, o.M - m0), quads = mt * 32;
    const uint32_t base = smem_u32(part);
    for (int e = rank * 192 + tid; e < quads; e += split * 192) {
      const int c = e >> 5, q = (e & 31) * 4;
      int4 sum = make_int4(0, 0, 0, 0);
      bool lost = false;
#pragma unroll 4
      for (int r = 0; r < split; ++r) {
        const int4 p = ld_cluster_int4(map_to_rank(base + (c * 128 + q) * 4, r));
        sum.x += p.x;
        sum.y += p.y;
        sum.z += p.z;
        sum.w += p.w;
        lost = lost || p.x == kNoSum;
      }
      const float sa = FUSE ? sSa[c] : o.sa[m0 + c];
      const int v[4] = {sum.x, sum.y, sum.z, sum.w};
      const size_t at = (size_t)(m0 + c) * o.N + n0 + q;
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int nn = min(n0 + q + i, o.N - 1);
        y[i] = scaled(v[i], sa, o.sb[nn], bias_at(o, nn));
      }
      if (lost) continue;  // (here, so that nothing above waits for it)
      if (n0 + q + 4 <= o.N && (o.N & 3) == 0) {  // y is 16-byte aligned or ytma is off
        if (ytma && o.y_bf16)
          *reinterpret_cast<uint2*>(static_cast<bf16*>(o.y) + at) =
              make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
        else if (ytma)
          *reinterpret_cast<float4*>(static_cast<float*>(o.y) + at) =
              make_float4(y[0], y[1], y[2], y[3]);
      }
      if (!(ytma && n0 + q + 4 <= o.N && (o.N & 3) == 0)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (n0 + q + i >= o.N) break;
          if (o.y_bf16)
            static_cast<bf16*>(o.y)[at + i] = __float2bfloat16_rn(y[i]);
          else
            static_cast<float*>(o.y)[at + i] = y[i];
        }
      }
    }
    cluster_sync();  // peers read this CTA's partials until here
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) tc::tmem_dealloc(tmem, 2 * P::kCols);
}

// ---------------------------------------------------------------------- wide
constexpr int kWS = 5;                       // operand stages
constexpr int kWHalf = 128 * 128;            // bytes of one operand's half of a stage
constexpr int kWStage = 2 * kWHalf;          // a CTA's bytes of a stage
constexpr int kWStaging = 8 * 32 * 128;      // 32 rows x 128 bytes of y for each epilogue warp
constexpr size_t kWSmem = 1024 + (size_t)kWS * kWStage + kWStaging + 4 * 256 * 4 + 256;

__device__ __forceinline__ void store2(void* p, uint32_t w) {
  *static_cast<unsigned short*>(p) = (unsigned short)w;
}
// A warp's staging (32 rows of 128 swizzled bytes: columns cs .. of rows row0 ..) to a y
// whose rows TMA cannot store: a row at a time, 4 bytes a lane; in rows of bf16 that
// start off 4 bytes (N odd), a lane stores its upper value and its neighbour's lower one.
// (2939 tokens, K = 73, bf16: N = 92615 368 us, value by value 726; N = 92616, by TMA, 234.)
__device__ __forceinline__ void store_rows(const Out& o, const unsigned char* buf, int row0,
                                           int cs) {
  const int lane = threadIdx.x & 31, rows = min(32, o.M - row0), left = o.N - cs;
  const auto word = [&](int r) {
    return *reinterpret_cast<const uint32_t*>(buf + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) +
                                              (lane & 3) * 4);
  };
  const int es = o.y_bf16 ? 2 : 4;
  const int mine = left - lane * (4 / es);  // columns from this lane's on
  const size_t pitch = (size_t)o.N * es;
  unsigned char* y = static_cast<unsigned char*>(o.y) + ((size_t)row0 * o.N + cs) * es;
  // rows first, first + step, ..., on a multiple of 4 bytes or 2 off one
  const auto some = [&](int first, int step, bool off) {
    unsigned char* to = y + first * pitch + 4 * lane;
    const size_t by = step * pitch;
    for (int r0 = first; r0 < rows; r0 += 8 * step, to += 8 * by) {
      uint32_t w[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) w[r] = word(min(r0 + r * step, 31));
      if (!off) {
        if (4 <= mine * es) {
#pragma unroll
          for (int r = 0; r < 8; ++r)
            if (r0 + r * step < rows) *reinterpret_cast<uint32_t*>(to + r * by) = w[r];
        } else if (mine == 1) {
#pragma unroll
          for (int r = 0; r < 8; ++r)
            if (r0 + r * step < rows) store2(to + r * by, w[r]);
        }
        continue;
      }
      if (lane == 0 && mine > 0) {
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (r0 + r * step < rows) store2(to + r * by, w[r]);
      }
#pragma unroll
      for (int r = 0; r < 8; ++r)
        w[r] = __funnelshift_r(w[r], __shfl_down_sync(0xffffffffu, w[r], 1), 16);
      if (lane < 31 && mine >= 3) {
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (r0 + r * step < rows) *reinterpret_cast<uint32_t*>(to + r * by + 2) = w[r];
      } else if (mine >= 2) {
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (r0 + r * step < rows) store2(to + r * by + 2, w[r]);
      }
    }
  };
  const int odd = reinterpret_cast<uintptr_t>(y) >> 1 & 1;  // the first row's
  if (pitch % 4 == 0) {
    some(0, 1, odd);
  } else {
    some(odd, 2, false);
    some(1 - odd, 2, true);
  }
}

// Warps: 0 TMA, 1 MMA (and TMEM), 2..9 epilogue (two a lane quadrant, 128 columns each).
// YTMA: y by TMA; a kernel of its own, since the other's stores cost this one 1.5 % (518
// against 525 us at 32768 x 8192 x 2048 with the quantisation, back to back) unexecuted.
// After a wait that gives up, as the kernel above.
template <bool YTMA>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(320, 1)
i8_wide_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw,
               const __grid_constant__ CUtensorMap ty, const Out o) {
  extern __shared__ unsigned char raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* staging = sm + (size_t)kWS * kWStage;
  float* scales = reinterpret_cast<float*>(staging + kWStaging);  // [2][scale, bias][256]
  uint64_t* full = reinterpret_cast<uint64_t*>(scales + 4 * 256);  // in the leader: both CTAs' bytes
  uint64_t* empty = full + kWS;
  uint64_t* acc_full = empty + kWS;    // [2]
  uint64_t* acc_empty = acc_full + 2;  // [2], in the leader: the sixteen epilogue warps
  uint32_t* tptr = reinterpret_cast<uint32_t*>(acc_empty + 2);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_rank();
  if (tid == 0) {
    for (int s = 0; s < kWS; ++s) tc::mbar_init(full + s, 1), tc::mbar_init(empty + s, 1);
    for (int i = 0; i < 2; ++i) tc::mbar_init(acc_full + i, 1), tc::mbar_init(acc_empty + i, 16);
    tc::fence_mbar_init();
    tc::prefetch_tmap(&tx);
    tc::prefetch_tmap(&tw);
    tc::prefetch_tmap(&ty);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(
                     smem_u32(tptr)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::);
  }
  tc::tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc::tc_fence_after();
  const uint32_t tmem = *tptr;
  const int KT = (o.K + 127) >> 7;
  const int MT = (o.M + 255) >> 8, NTL = (o.N + 255) >> 8, tiles = MT * NTL;
  const int cl = blockIdx.x >> 1, ncl = gridDim.x >> 1;
  // tiles in groups of 8 channel tiles, tokens slower than the channels of a
  // group: the group's weights stay in L2 while x streams past them once
  const auto place = [&](int t, int& m, int& n) {
    const int per = 8 * MT, gidx = t / per, in = t - gidx * per;
    const int w = min(8, NTL - gidx * 8);
    m = in / w;
    n = gidx * 8 + in - m * w;
  };

  if (warp == 0 && lane == 0) {
    grid_dependency_wait();
    uint32_t it = 0;
    bool ok = true;
    const uint32_t without = o.withhold ? 0 : ~0u;  // the step whose x is not loaded (a test)
    for (int t = cl; ok && t < tiles; t += ncl) {
      int mt, nt;
      place(t, mt, nt);
      const int m = mt * 256 + rank * 128, n = nt * 256 + rank * 128;
      for (int k = 0; k < KT; ++k, ++it) {
        const int s = it % kWS;
        if (it >= kWS && !(ok = tc::mbar_wait(empty + s, (it / kWS - 1) & 1, 130))) break;
        const uint32_t bar = map_to_rank(smem_u32(full + s), 0);
        if (rank == 0) tc::mbar_expect_tx(full + s, 2 * kWStage);
        unsigned char* st = sm + (size_t)s * kWStage;
        if (it != without) tma_load_2d_pair(st, &tx, k * 128, m, bar);
        tma_load_2d_pair(st + kWHalf, &tw, k * 128, n, bar);
      }
    }
    // every stage's last release has arrived before this CTA may leave
    for (uint32_t i = it > kWS ? it - kWS : 0; i < it; ++i)
      tc::mbar_wait(empty + i % kWS, (i / kWS) & 1, 134);
  } else if (warp == 1 && lane == 0 && rank == 0) {
    constexpr uint32_t idesc = idesc_i8(256, 256);
    uint32_t it = 0, at = 0;
    bool ok = true;
    for (int t = cl; ok && t < tiles; t += ncl, ++at) {
      const int buf = at & 1;
      if (at >= 2 && !(ok = tc::mbar_wait(acc_empty + buf, (at / 2 - 1) & 1, 131))) break;
      tc::tc_fence_after();
      for (int k = 0; k < KT; ++k, ++it) {
        const int s = it % kWS;
        if (!(ok = tc::mbar_wait(full + s, (it / kWS) & 1, 132))) break;
        tc::tc_fence_after();
        const uint32_t a0 = smem_u32(sm + (size_t)s * kWStage);
        const uint64_t ad = tc::sdesc(a0, 0, 1024), bd = tc::sdesc(a0 + kWHalf, 0, 1024);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          mma_i8_pair(tmem + buf * 256, ad + 2 * q, bd + 2 * q, idesc, (k | q) != 0);
        commit_pair(empty + s);
      }
      if (ok) commit_pair(acc_full + buf);
    }
    if (!ok) in_flight(full, empty, kWS, it);  // (the loads of both CTAs)
  } else if (warp >= 2) {
    const int quad = warp & 3, col0 = (warp - 2) / 4 * 128, etid = tid - 64;
    unsigned char* buf_y = staging + (warp - 2) * 32 * 128;
    const uint32_t peer_free[2] = {map_to_rank(smem_u32(acc_empty), 0),
                                   map_to_rank(smem_u32(acc_empty + 1), 0)};
    const int per = o.y_bf16 ? 64 : 32;  // columns a 128-byte row of the staging holds
    grid_dependency_wait();
    uint32_t at = 0;
    // a tile's scales, loaded while the one before is written
    float next_sa = 0.f, next_sb = 0.f, next_bias = 0.f;
    bool live = true;  // no wait has given up
    const auto fetch = [&](int t) {
      int m, n;
      place(t, m, n);
      m = m * 256 + rank * 128 + quad * 32 + lane;
      n = n * 256 + etid;
      next_sa = m < o.M ? o.sa[m] : 0.f;
      next_sb = n < o.N ? o.sb[n] : 0.f;
      next_bias = n < o.N ? bias_at(o, n) : 0.f;
    };
    if (cl < tiles) fetch(cl);
    for (int t = cl; t < tiles; t += ncl, ++at) {
      int mt, nt;
      place(t, mt, nt);
      const int buf = at & 1, n0 = nt * 256, row0 = mt * 256 + rank * 128 + quad * 32;
      float *sSb = scales + buf * 512, *sBias = sSb + 256;
      sSb[etid] = next_sb;
      sBias[etid] = next_bias;
      const float sa = next_sa;
      tc::named_bar_sync(1, 256);  // (every warp is done with the tile before the last)
      if (t + ncl < tiles) fetch(t + ncl);
      live = __all_sync(0xffffffffu, tc::mbar_wait(acc_full + buf, (at / 2) & 1, 133)) && live;
      tc::tc_fence_after();
      const uint32_t ta = tmem + buf * 256 + col0 + ((uint32_t)(quad * 32) << 16);
      float v[2][32];
      tc::tmem_ld32(ta, v[0]);
#pragma unroll
      for (int q = 0; q < 4; ++q) {  // 32 columns at a time, the next ones loading
        tc::tmem_wait_ld();
        if (q < 3) {
          tc::tmem_ld32(ta + 32 * (q + 1), v[(q + 1) & 1]);
        } else {  // the accumulator has been read
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_remote(peer_free[buf]);
        }
        float(&x)[32] = v[q & 1];
        const int c0 = col0 + 32 * q;
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          const float4 s4 = *reinterpret_cast<const float4*>(sSb + c0 + c);
          const float ss[4] = {s4.x, s4.y, s4.z, s4.w};
          float bb[4] = {0.f, 0.f, 0.f, 0.f};
          if (o.bias) {
            const float4 b4 = *reinterpret_cast<const float4*>(sBias + c0 + c);
            bb[0] = b4.x, bb[1] = b4.y, bb[2] = b4.z, bb[3] = b4.w;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e)
            x[c + e] = scaled(__float_as_int(x[c + e]), sa, ss[e], bb[e]);
        }
        const bool starts = (32 * q) % per == 0, ends = (32 * (q + 1)) % per == 0;
        if (starts) {
          if (lane == 0) tc::bulk_wait_read0();  // the store before has left the staging
          __syncwarp();
        }
        if (o.y_bf16) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const uint4 w = make_uint4(
                pack_bf16(x[8 * u], x[8 * u + 1]), pack_bf16(x[8 * u + 2], x[8 * u + 3]),
                pack_bf16(x[8 * u + 4], x[8 * u + 5]), pack_bf16(x[8 * u + 6], x[8 * u + 7]));
            *reinterpret_cast<uint4*>(buf_y + lane * 128 +
                                      ((((q & 1) * 4 + u) ^ (lane & 7)) << 4)) = w;
          }
        } else {
#pragma unroll
          for (int u = 0; u < 8; ++u)
            *reinterpret_cast<float4*>(buf_y + lane * 128 + ((u ^ (lane & 7)) << 4)) =
                make_float4(x[4 * u], x[4 * u + 1], x[4 * u + 2], x[4 * u + 3]);
        }
        if (!ends) continue;
        const int cs = n0 + c0 + 32 - per;  // first column of the staging
        if constexpr (YTMA) {
          tc::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && row0 < o.M && cs < o.N && live) {
            tma_store_2d(&ty, buf_y, cs, row0);
            tc::bulk_commit();
          }
        } else {
          __syncwarp();
          if (live) store_rows(o, buf_y, row0, cs);
          __syncwarp();
        }
      }
    }
    if (lane == 0) tc::bulk_wait0();
  }
  __syncwarp();
  tc::tc_fence_before();
  __syncthreads();
  cluster_sync();  // no signal of the pair is still on its way
  tc::tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512));
}

// ---------------------------------------------------------------------- host
int encode(CUtensorMap* m, const char* what, CUtensorMapDataType type, const void* p, int cols,
           int rows, long long row_bytes, int box_cols, int box_rows,
           CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
  auto fn = tc::encode_tiled_fn();
  if (!fn) {
    set_error("int8: cuTensorMapEncodeTiled is not available");
    return LZ_ERR_CUDA;
  }
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)row_bytes};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  const cuuint32_t es[2] = {1, 1};
  const CUresult r = fn(m, type, 2, const_cast<void*>(p), dims, strides, box, es,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error(std::string("int8: the tensor map of ") + what + " could not be encoded, driver code " +
              std::to_string((int)r));
    return LZ_ERR_CUDA;
  }
  return LZ_OK;
}

template <typename K>
int allow_smem(K kern, size_t bytes, bool* done) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || done[dev]) return LZ_OK;
  cudaError_t e =
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e != cudaSuccess) {
    set_error(std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
    return LZ_ERR_CUDA;
  }
  done[dev] = true;
  return LZ_OK;
}

int launched(cudaError_t e, const char* what) {
  if (e != cudaSuccess) {
    set_error(std::string(what) + ": " + cudaGetErrorString(e));
    return LZ_ERR_CUDA;
  }
  count_launches(1);
  return check_launch(what);
}

struct Operand {
  const int8_t* p;
  long long ld;  // bytes, a multiple of 16
  int rows;
};

// Shares of K of the narrow kernel: K is split while the tiles leave SMs idle and
// every share keeps two steps of 128.
int k_split(long long tiles, int KT) {
  int split = 1;
  while (split < 8 && tiles * split < 148 && KT >= 4 * split) split *= 2;
  return split;
}

template <int BN, bool FUSE = false>
int launch_narrow(const Operand& x, const Operand& w, const Out& o, bool after_quantize,
                  cudaStream_t st) {
  const int es = o.y_bf16 ? 2 : 4;
  const int ytma = aligned16(o.y) && ((long long)o.N * es) % 16 == 0;
  const int wt = ceil_div(o.N, 128), mt = ceil_div(o.M, BN), KT = ceil_div(o.K, 128);
  const int split = k_split((long long)wt * mt, KT);
  CUtensorMap tw, tx, ty;
  int rc = encode(&tw, "the weight", CU_TENSOR_MAP_DATA_TYPE_UINT8, w.p, o.K, o.N, w.ld, 128, 128);
  if (!rc && !FUSE)
    rc = encode(&tx, "x", CU_TENSOR_MAP_DATA_TYPE_UINT8, x.p, o.K, o.M, x.ld, 128, BN);
  if (!rc && ytma && split == 1)
    rc = encode(&ty, "y", o.y_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32,
                o.y, o.N, o.M, (long long)o.N * es, 128, std::min(BN, kNStaging / (128 * es)),
                CU_TENSOR_MAP_SWIZZLE_NONE);
  else
    ty = tw;
  if (FUSE) tx = tw;
  if (rc) return rc;
  static bool done[64] = {false};
  using P = Narrow<BN, FUSE>;
  rc = allow_smem(i8_narrow_kernel<BN, FUSE>, P::smem(FUSE ? kFuseK / 128 : 0), done);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = split > 1 ? dim3(wt * mt * split)
                          : dim3((unsigned)std::min<long long>((long long)wt * mt, 296));
  cfg.blockDim = dim3(192);
  cfg.dynamicSmemBytes = P::smem(FUSE ? ceil_div(KT, split) : 0);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = split;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = after_quantize ? 2 : 1;
  return launched(cudaLaunchKernelEx(&cfg, i8_narrow_kernel<BN, FUSE>, tw, tx, ty, o, split, ytma),
                  "i8_narrow_kernel");
}

int launch_wide(const Operand& x, const Operand& w, const Out& o, bool after_quantize,
                cudaStream_t st) {
  const int es = o.y_bf16 ? 2 : 4;
  const int ytma = aligned16(o.y) && ((long long)o.N * es) % 16 == 0;
  CUtensorMap tx, tw, ty;
  int rc = encode(&tx, "x", CU_TENSOR_MAP_DATA_TYPE_UINT8, x.p, o.K, o.M, x.ld, 128, 128);
  if (!rc) rc = encode(&tw, "the weight", CU_TENSOR_MAP_DATA_TYPE_UINT8, w.p, o.K, o.N, w.ld, 128, 128);
  if (!rc && ytma)
    rc = encode(&ty, "y", o.y_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32,
                o.y, o.N, o.M, (long long)o.N * es, 128 / es, 32);
  if (rc) return rc;
  if (!ytma) ty = tx;
  static bool done[2][64] = {};
  const auto kernel = ytma ? i8_wide_kernel<true> : i8_wide_kernel<false>;
  rc = allow_smem(kernel, kWSmem, done[ytma]);
  if (rc) return rc;
  const long long tiles = (long long)ceil_div(o.M, 256) * ceil_div(o.N, 256);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * (unsigned)std::min<long long>(tiles, 74));
  cfg.blockDim = dim3(320);
  cfg.dynamicSmemBytes = kWSmem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = after_quantize ? 1 : 0;
  return launched(cudaLaunchKernelEx(&cfg, kernel, tx, tw, ty, o), "i8_wide_kernel");
}

template <typename T>
void launch_quantize(const void* x, long long ldx, int8_t* codes, long long ldc, float* scale,
                     int M, int K, cudaStream_t st) {
  const T* p = static_cast<const T*>(x);
  // a warp holds 8 vectors a lane: 2048 bf16 or 1024 fp32
  if (K <= 256 * Vec<T>::N)
    i8_quantize_kernel<T, 32, 8>
        <<<ceil_div(M, kQT / 32), kQT, 0, st>>>(p, ldx, codes, ldc, scale, M, K);
  else
    i8_quantize_kernel<T, kQT, 4><<<M, kQT, 0, st>>>(p, ldx, codes, ldc, scale, M, K);
}

int quantize(const void* x, int x_dtype, long long ldx, int8_t* codes, long long ldc, float* scale,
             int M, int K, cudaStream_t st) {
  if (x_dtype == LZ_DTYPE_F32)
    launch_quantize<float>(x, ldx, codes, ldc, scale, M, K, st);
  else
    launch_quantize<bf16>(x, ldx, codes, ldc, scale, M, K, st);
  count_launches(1);
  return check_launch("i8_quantize_kernel");
}

std::atomic<int> g_path{0};
std::atomic<int> g_withhold{0};  // lz_test_withhold_int8_load

// Which kernel, by an estimate of both in hundredths of a us, fitted to measured
// times (quantisation included) over M = 64 .. 2048, K = 512 .. 8192, N = 512 ..
// 128256. A step of 128 of K costs a 256 x 256 tile of a CTA pair 0.29 us and a
// 128 x 128 tile 0.5 us with two CTAs on the SM; a tile costs 2 and 2.5 us more.
// Measured, narrow / wide: M = 256, K = 8192: N = 512 11.0 / 24.7 us, N = 128256
// 337 / 214 us; M = 512, K = 8192: N = 2048 17.6 / 25.9, N = 8192 35.7 / 30.9;
// M = 256, N = 512: K = 512 10.2 / 8.2, K = 2048 8.5 / 11.5. Up to 64 tokens the
// narrow one is never slower.
bool use_wide(int M, int N, int K) {
  if (M <= 64) return false;
  const long long KT = ceil_div(K, 128);
  const long long small = (long long)ceil_div(M, 128) * ceil_div(N, 128);
  const long long large = (long long)ceil_div(M, 256) * ceil_div(N, 256);
  const int split = k_split(small, (int)KT);
  const long long narrow = 550 + (small * split + 295) / 296 * (50 * KT / split + 250);
  const long long wide = 500 + (large + 73) / 74 * (29 * KT + 200);
  return wide < narrow;
}

int product(const Operand& x, const Operand& w, const Out& o, bool after_quantize,
            cudaStream_t st) {
  const int path = g_path.load(std::memory_order_relaxed);
  if (path ? path == 2 : use_wide(o.M, o.N, o.K)) return launch_wide(x, w, o, after_quantize, st);
  if (o.M <= 16) return launch_narrow<16>(x, w, o, after_quantize, st);
  if (o.M <= 32) return launch_narrow<32>(x, w, o, after_quantize, st);
  if (o.M <= 64) return launch_narrow<64>(x, w, o, after_quantize, st);
  return launch_narrow<128>(x, w, o, after_quantize, st);
}

// Whether the product quantises x by itself: every CTA then reads all of x, a warp a
// row, so for up to four tokens of up to 4096 values, and while an SM has one weight
// tile at most (the codes' room leaves one CTA an SM, which with more tiles loads the
// weights more slowly: 50 us against 46 at K = 2048, N = 128256). One token, K = N =
// 2048: 6.3 us against 6.0 on the device, a launch less for the host.
bool fuse_quantize(int M, int N, int K) {
  return M <= 4 && K <= kFuseK && N <= 148 * 128;
}

long long row16(int K) { return ((long long)K + 15) / 16 * 16; }

// Rows of codes as the kernels take them: as they are, or repacked into *ws.
int as_operand(Operand* op, const void* p, long long ld, int rows, int K, unsigned char** ws,
               cudaStream_t st) {
  op->rows = rows;
  op->p = static_cast<const int8_t*>(p);
  if (rows == 1) ld = row16(K);  // a single row's stride is never used
  op->ld = ld;
  if (aligned16(p) && ld % 16 == 0) return LZ_OK;
  int8_t* to = reinterpret_cast<int8_t*>(*ws);
  *ws += align_up((size_t)rows * row16(K), 256);
  i8_repack_kernel<<<rows, kQT, 0, st>>>(op->p, ld, to, row16(K), K);
  count_launches(1);
  op->p = to;
  op->ld = row16(K);
  return check_launch("i8_repack_kernel");
}

int check_out(const void* bias, int bias_dtype, const void* y, int y_dtype, int M, int N, int K) {
  LZ_REQUIRE(M >= 1 && N >= 1 && K >= 1, LZ_ERR_INVALID_ARGUMENT, "sizes must be positive");
  LZ_REQUIRE(K <= kMaxK, LZ_ERR_UNSUPPORTED,
             "K above 131071 can overflow the 32-bit integer sum");
  LZ_REQUIRE(N <= (1 << 30) && M <= (1 << 30) && (N / 128 + 1ll) * (M / 16 + 1ll) < (1ll << 31),
             LZ_ERR_UNSUPPORTED, "sizes too large");
  LZ_REQUIRE(y, LZ_ERR_INVALID_ARGUMENT, "null pointer");
  LZ_REQUIRE(y_dtype == LZ_DTYPE_F32 || y_dtype == LZ_DTYPE_BF16, LZ_ERR_INVALID_ARGUMENT,
             "y must be LZ_DTYPE_F32 or LZ_DTYPE_BF16");
  LZ_REQUIRE(!bias || bias_dtype == LZ_DTYPE_F32 || bias_dtype == LZ_DTYPE_BF16,
             LZ_ERR_INVALID_ARGUMENT, "bias must be LZ_DTYPE_F32 or LZ_DTYPE_BF16");
  return LZ_OK;
}

}  // namespace
int int8_timeout_flag(unsigned int* out) { return tc::read_timeout_flag_here(out); }
int int8_timeout_clear() { return tc::clear_timeout_flag_here(); }
}  // namespace lz

extern "C" int lz_int8_set_path(int path) {
  if (path < 0 || path > 2) {
    lz::set_error("path must be 0 (chosen by size), 1 (narrow) or 2 (wide)");
    return -LZ_ERR_INVALID_ARGUMENT;
  }
  return lz::g_path.exchange(path);
}

extern "C" int lz_test_withhold_int8_load(int on) {
  return lz::g_withhold.exchange(on ? 1 : 0);
}

extern "C" int lz_int8_quantize(const void* x, int x_dtype, long long x_ld, void* codes,
                                long long codes_ld, float* scale, int M, int K, void* stream) {
  using namespace lz;
  clear_error();
  LZ_REQUIRE(M >= 1 && K >= 1, LZ_ERR_INVALID_ARGUMENT, "sizes must be positive");
  LZ_REQUIRE(x && codes && scale, LZ_ERR_INVALID_ARGUMENT, "null pointer");
  LZ_REQUIRE(x_dtype == LZ_DTYPE_F32 || x_dtype == LZ_DTYPE_BF16, LZ_ERR_INVALID_ARGUMENT,
             "x must be LZ_DTYPE_F32 or LZ_DTYPE_BF16");
  LZ_REQUIRE(codes_ld >= K && codes_ld % 16 == 0 && aligned16(codes), LZ_ERR_INVALID_ARGUMENT,
             "rows of codes must start on 16-byte boundaries");
  return quantize(x, x_dtype, x_ld, static_cast<int8_t*>(codes), codes_ld, scale, M, K,
                  static_cast<cudaStream_t>(stream));
}

extern "C" size_t lz_int8_workspace_bytes(int M, int N, int K) {
  if (M < 1 || N < 1 || K < 1) return 0;
  const size_t r = (size_t)lz::row16(K);
  return lz::align_up((size_t)M * r, 256) + lz::align_up((size_t)M * 4, 256) +
         lz::align_up((size_t)N * r, 256);
}

extern "C" size_t lz_int8_linear_workspace_bytes(int M, int N, int K) {
  if (M < 1 || N < 1 || K < 1 || lz::fuse_quantize(M, N, K)) return 0;
  return lz::align_up((size_t)M * (size_t)lz::row16(K), 256) + lz::align_up((size_t)M * 4, 256);
}

extern "C" int lz_int8_matmul(const void* a, long long a_ld, const float* a_scale, const void* b,
                              long long b_ld, const float* b_scale, const void* bias,
                              int bias_dtype, void* y, int y_dtype, void* workspace,
                              size_t workspace_bytes, int M, int N, int K, void* stream) {
  using namespace lz;
  clear_error();
  int rc = check_out(bias, bias_dtype, y, y_dtype, M, N, K);
  if (rc) return rc;
  LZ_REQUIRE(a && b && a_scale && b_scale, LZ_ERR_INVALID_ARGUMENT, "null pointer");
  LZ_REQUIRE((M == 1 || a_ld >= K) && (N == 1 || b_ld >= K), LZ_ERR_INVALID_ARGUMENT,
             "rows of codes overlap");
  const bool fits = aligned16(a) && (M == 1 || a_ld % 16 == 0) && aligned16(b) &&
                    (N == 1 || b_ld % 16 == 0);
  LZ_REQUIRE(fits || (workspace && aligned16(workspace) &&
                      workspace_bytes >= lz_int8_workspace_bytes(M, N, K)),
             LZ_ERR_WORKSPACE, "workspace too small, see lz_int8_workspace_bytes");
  auto st = static_cast<cudaStream_t>(stream);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  Operand x, w;
  rc = as_operand(&x, a, a_ld, M, K, &ws, st);
  if (!rc) rc = as_operand(&w, b, b_ld, N, K, &ws, st);
  if (rc) return rc;
  const Out o = {a_scale, b_scale, bias, y, bias_dtype == LZ_DTYPE_BF16, y_dtype == LZ_DTYPE_BF16,
                 M, N, K, nullptr, 0, 0, g_withhold.load(std::memory_order_relaxed)};
  return product(x, w, o, false, st);
}

extern "C" int lz_int8_linear(const void* x, int x_dtype, long long x_ld, const void* w,
                              long long w_ld, const float* w_scale, const void* bias,
                              int bias_dtype, void* y, int y_dtype, void* workspace,
                              size_t workspace_bytes, int M, int N, int K, void* stream) {
  using namespace lz;
  clear_error();
  int rc = check_out(bias, bias_dtype, y, y_dtype, M, N, K);
  if (rc) return rc;
  LZ_REQUIRE(x && w && w_scale, LZ_ERR_INVALID_ARGUMENT, "null pointer");
  LZ_REQUIRE(x_dtype == LZ_DTYPE_F32 || x_dtype == LZ_DTYPE_BF16, LZ_ERR_INVALID_ARGUMENT,
             "x must be LZ_DTYPE_F32 or LZ_DTYPE_BF16");
  LZ_REQUIRE(N == 1 || w_ld >= K, LZ_ERR_INVALID_ARGUMENT, "rows of codes overlap");
  const bool fits = aligned16(w) && (N == 1 || w_ld % 16 == 0);
  const size_t need =
      fits ? lz_int8_linear_workspace_bytes(M, N, K) : lz_int8_workspace_bytes(M, N, K);
  LZ_REQUIRE(!need || (workspace && aligned16(workspace) && workspace_bytes >= need),
             LZ_ERR_WORKSPACE, "workspace too small, see lz_int8_linear_workspace_bytes");
  auto st = static_cast<cudaStream_t>(stream);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  if (fits && fuse_quantize(M, N, K)) {
    const Operand wo = {static_cast<const int8_t*>(w), N == 1 ? row16(K) : w_ld, N};
    const Out o = {nullptr, w_scale, bias, y, bias_dtype == LZ_DTYPE_BF16,
                   y_dtype == LZ_DTYPE_BF16, M, N, K, x, x_ld, x_dtype == LZ_DTYPE_BF16,
                   g_withhold.load(std::memory_order_relaxed)};
    return launch_narrow<16, true>({nullptr, 0, M}, wo, o, false, st);
  }
  int8_t* codes = reinterpret_cast<int8_t*>(ws);
  ws += align_up((size_t)M * row16(K), 256);
  float* sa = reinterpret_cast<float*>(ws);
  ws += align_up((size_t)M * 4, 256);
  Operand wo;
  rc = as_operand(&wo, w, w_ld, N, K, &ws, st);
  if (!rc) rc = quantize(x, x_dtype, x_ld, codes, row16(K), sa, M, K, st);
  if (rc) return rc;
  const Operand xo = {codes, row16(K), M};
  const Out o = {sa, w_scale, bias, y, bias_dtype == LZ_DTYPE_BF16, y_dtype == LZ_DTYPE_BF16,
                 M, N, K, nullptr, 0, 0, g_withhold.load(std::memory_order_relaxed)};
  return product(xo, wo, o, true, st);
}
