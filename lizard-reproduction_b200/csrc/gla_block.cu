// A block of new tokens through the gated linear attention state, with the
// state left at the accepted prefix.
//
// Drafted decoding runs T tokens (the last accepted one and T - 1 drafted ones)
// through the model at once and learns only afterwards how many of them stand.
// The kernel therefore advances the state by the accepted tokens of the PREVIOUS
// block and reads this block's outputs from it, in one pass over the state:
//   S <- g(n) S + sum_{s < n} w_s k'_s^T v'_s,     w_s = exp(sum_{s < r < n} lg'_r)
//   z <- g(n) z + sum_{s < n} w_s k'_s,            g(n) = exp(sum_{r < n} lg'_r)
//   y_t = (d_t q_t S + sum_{s <= t} a_ts v_s) / max(d_t q_t z + sum_{s <= t} a_ts, FLT_MIN)
//   a_ts = (q_t . k_s) exp(sum_{s < r <= t} lg_r),  d_t = exp(sum_{r <= t} lg_r)
// (primes: the previous block, n = count[b] of its tokens accepted; a token-by-
// token run of lz_gla_decode over the accepted tokens and the block gives the
// same values). Every decay is the exp of a running sum over its own range, so a
// gate of zero (lg = -inf) gives 0 and not inf - inf.
//
// Bound: the state is read once and written once, 8 F D bytes a head, against
// 2 rep T F D multiply-adds: memory. A CTA takes 64 (or 32) columns of a state: TMA
// brings them into shared memory in 128-byte swizzled rows while the keys, gates
// and queries are staged, and each warp takes 16 columns by half of the F rows into
// registers, as the B fragments of mma.sync m16n8k16: thread (g, j) holds columns g
// and 8 + g of rows 2j, 2j+1, 2j+8, 2j+9 of each 16-row step (the swizzle keeps
// these reads free of bank conflicts). It updates them in fp32 (packed pairs of
// rows; k and v are bf16, their products exact), writes them back, splits them once
// into bf16 hi + lo parts (relative error 2^-17, against the 2^-8 of the bf16
// output) and contracts the queries with them 32 rows at a time; the two halves of
// F meet at the end, a row tile each. (8 columns by all of F needs no such meeting
// but reads every key and query value twice as often from shared memory, which then
// bounds the kernel.) Measured, 2048 states of 256 x 64, 32 query rows, 8 tokens: 82 us,
// 4.1 TB/s of state and operands; what is left is the chain of phases of a CTA (load,
// decays, update, products, meeting) at two CTAs an SM, since this form holds a warp's whole
// share of the state and then its bf16 parts in registers at once. A persistent form that loads the next state under this one's products
// was slower (90 us): the rows of a batch accept different numbers of tokens, and
// CTAs handed out one by one even that out.
// The scores of the block's keys are shared: a quarter of F a warp, added through
// shared memory. z rides along as two more keys (hi and lo): with M = [exp of the
// decay from key to token, 0 above the diagonal | d_t for the two z columns], a' =
// (q K^T) o M has the row sum as its own sum over all columns, and y = (d_t q S + a' V) /
// sum a' with zero rows of V for z.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "tc.cuh"

namespace lz {
namespace {

constexpr int kMaxBlock = 64;  // tokens a block

struct GlaBlockArgs {
  const bf16 *fq, *fk, *v;
  const float* lg;
  const bf16 *fk_p, *v_p;
  const float* lg_p;
  const int* count;
  float *S, *Z;
  bf16* y;
  // rep query heads a state, kvrep state heads a key/value head
  int gph, T, Tp, H, Hkv, Hs, F, D, nsl, rep, kvrep;
  int withhold;  // a test: the state's first tile is not loaded
};

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}

// rows x ncols bf16 (row stride ldg) into shared rows of ld elements, zeros to
// pad_rows x width; 16-byte copies when rows keep that alignment.
__device__ __forceinline__ void stage_rows(bf16* s, int ld, int width, int ldg, const bf16* g,
                                           int rows, int ncols, int pad_rows, int nthreads) {
  const bool vec = ((ldg | ncols) & 7) == 0 && (reinterpret_cast<uintptr_t>(g) & 15) == 0;
  if (vec) {
    const int cpr = width >> 3;
    for (int i = threadIdx.x; i < pad_rows * cpr; i += nthreads) {
      const int r = i / cpr, c = (i - r * cpr) * 8;
      const bool in = r < rows && c < ncols;
      cp_async16(s + r * ld + c, in ? g + r * ldg + c : g, in);
    }
  } else {
    for (int i = threadIdx.x; i < pad_rows * width; i += nthreads) {
      const int r = i / width, c = i - r * width;
      s[r * ld + c] = r < rows && c < ncols ? g[r * ldg + c] : __float2bfloat16_rn(0.f);
    }
  }
}

// Two fp32 values in a 64-bit register, and two operations an instruction.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float x, float y) {
  f32x2 d;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(d) : "f"(x), "f"(y));
  return d;
}
__device__ __forceinline__ void unpack2(f32x2 v, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// Gates of tokens lane and lane + 32 (x0, x1) become the sums over the tokens after
// them; returns the sum of all n. Every sum is a running one: a closed gate (-inf)
// stays -inf for the tokens before it and touches no other.
__device__ __forceinline__ float after(float& x0, float& x1, int n) {
  const int lane = threadIdx.x & 31;
  const auto scan = [&](float& x) {  // inclusive from the right; returns the total
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const float y = __shfl_down_sync(0xffffffffu, x, o);
      if (lane + o < 32) x += y;
    }
    const float all = __shfl_sync(0xffffffffu, x, 0);
    const float y = __shfl_down_sync(0xffffffffu, x, 1);
    x = lane < 31 ? y : 0.f;
    return all;
  };
  float high = 0.f;
  if (n > 32) high = scan(x1);
  const float all = scan(x0);
  x0 += high;
  return all + high;
}

constexpr int kQRows = 32;  // query rows staged at a time
constexpr int kPend = 8;    // pending tokens folded in at a time

// Shared memory, in bytes from the 1024-aligned start.
struct BlockSmem {
  int q, k, v, kw, vw, a, den, m, bar, late, total;
};
__host__ __device__ inline BlockSmem block_smem(int KS, int HALVES, int T) {
  const int LD = 64 * KS + 8, DN = 32 * HALVES, TK = (T + 2 + 15) & ~15;
  BlockSmem s;
  int n = HALVES * 64 * KS * 128;  // the state's columns
  // queries, then the halves of F on their way to each other (1 KB a warp)
  s.q = n, n += kQRows * LD * 2 > HALVES * 4096 ? kQRows * LD * 2 : HALVES * 4096;
  s.k = n, n += TK * LD * 2;
  s.v = n, n += TK * (DN + 8) * 2;
  // pending keys, then (they are done) the partial scores of the quarters of F
  const int kw = kPend * 64 * KS * 4, parts = 4 * kQRows * 16 * 4;
  s.kw = n, n += kw > parts ? kw : parts;
  s.vw = n, n += kPend * DN * 4;
  s.a = n, n += 2 * kQRows * 48;  // a' hi and lo, rows of 16 and 8 to spare
  s.den = n, n += kQRows * 8;
  s.m = n, n += (T > 0 ? T : 1) * TK * 4;
  s.bar = (n + 7) & ~7, n = s.bar + 8;
  s.late = n, n += 4;
  s.total = n + 1024;
  return s;
}

// One output by itself, from tokens 0 .. t only: y = (d q S + sum_{s <= t} a_s v_s) /
// (d q z + sum a_s). The tensor cores give masked tokens a weight of zero, and 0 * inf
// and 0 * NaN are NaN: where that may have happened (the output is NaN), a thread
// comes here. q: the row's queries; S: the state's swizzled column tile and the column
// in it; K: keys, then z hi and lo; V: this column of the values; M: the row's decays.
__device__ __forceinline__ float alone(const bf16* q, const float* S, int col, const bf16* K,
                                       int LD, const bf16* V, int LV, const float* M, int t, int T,
                                       int F) {
  float num = 0.f, den = 0.f;
#pragma unroll 1
  for (int f = 0; f < F; ++f) {
    const float x = __bfloat162float(q[f]);
    num = fmaf(x, S[f * 32 + ((((col >> 2) ^ (f & 7)) << 2) | (col & 3))], num);
    den = fmaf(x, __bfloat162float(K[T * LD + f]) + __bfloat162float(K[(T + 1) * LD + f]), den);
  }
  num *= M[T], den *= M[T];
#pragma unroll 1
  for (int s = 0; s <= t && num == num && den == den; ++s) {
    float a = 0.f;
#pragma unroll 1
    for (int f = 0; f < F; ++f)
      a = fmaf(__bfloat162float(q[f]), __bfloat162float(K[s * LD + f]), a);
    a *= M[s];
    num = fmaf(a, __bfloat162float(V[s * LV]), num);
    den += a;
  }
  return num / (den < kTiny ? kTiny : den);
}

__device__ __forceinline__ int special(int which) {
  int v;
  if (which == 0) asm volatile("mov.u32 %0, %%tid.x;\n" : "=r"(v));
  if (which == 1) asm volatile("mov.u32 %0, %%ctaid.x;\n" : "=r"(v));
  if (which == 2) asm volatile("mov.u32 %0, %%ctaid.y;\n" : "=r"(v));
  if (which == 3) asm volatile("mov.u32 %0, %%ctaid.z;\n" : "=r"(v));
  return v;
}
// A thread's outputs of rows r0 .. that are NaN, one by one. Everything is derived anew
// (the volatile reads see to it), so that nothing of this is kept in registers before;
// as a call it would cost every launch 15 %, here 1 %.
template <int KS, int HALVES>
__device__ __forceinline__ void redo(const GlaBlockArgs& a, const unsigned char* sm, int r0) {
  constexpr int FP = 64 * KS, LD = FP + 8, DN = 32 * HALVES, LV = DN + 8;
  const int T = a.T, TK = (T + 2 + 15) & ~15, R = a.rep * T;
  const BlockSmem o = block_smem(KS, HALVES, T);
  const int tid = special(0), lane = tid & 31, warp = tid >> 5;
  const int cg = warp % (2 * HALVES), fh = warp / (2 * HALVES), d0 = special(3) * DN;
  const size_t row0 = ((size_t)special(1) * a.H + special(2) * a.rep) * T;
#pragma unroll 1
  for (int e = 0; e < 8; ++e) {
    const int row = r0 + fh * 16 + (lane >> 2) + (e >> 1 & 1) * 8, t = row % T;
    const int dd = cg * 16 + (e >> 2) * 8 + 2 * (lane & 3) + (e & 1);
    if (row >= R || d0 + dd >= a.D) continue;
    bf16* yr = a.y + (row0 + row) * a.D + d0 + dd;
    if (__hisnan(*yr))
      *yr = __float2bfloat16_rn(alone(
          a.fq + (row0 + row) * a.F, reinterpret_cast<const float*>(sm + (dd >> 5) * FP * 128),
          dd & 31, reinterpret_cast<const bf16*>(sm + o.k), LD,
          reinterpret_cast<const bf16*>(sm + o.v) + dd, LV,
          reinterpret_cast<const float*>(sm + o.m) + t * TK, t, T, a.F));
  }
}

// KS: F <= 64 KS. HALVES: 32-column groups of a CTA, four warps each.
template <int KS, int HALVES>
__global__ void __launch_bounds__(128 * HALVES, 2)
gla_block_kernel(const __grid_constant__ CUtensorMap ts, const GlaBlockArgs a) {
  constexpr int NT = 128 * HALVES, FP = 64 * KS, LD = FP + 8, DN = 32 * HALVES, LV = DN + 8;
  constexpr int NH = 2 * KS;  // 16-row steps of half of F
  extern __shared__ unsigned char raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  const int T = a.T, Tp = a.Tp, F = a.F, D = a.D;
  const BlockSmem o = block_smem(KS, HALVES, T);
  const int TK = (T + 2 + 15) & ~15;
  bf16* sQ = reinterpret_cast<bf16*>(sm + o.q);       // [32][LD]
  bf16* sK = reinterpret_cast<bf16*>(sm + o.k);       // [TK][LD]: keys, z hi, z lo, zeros
  bf16* sV = reinterpret_cast<bf16*>(sm + o.v);       // [TK][LV], zero rows from T on
  float* sKw = reinterpret_cast<float*>(sm + o.kw);   // [8][FP] pending keys
  float* sVw = reinterpret_cast<float*>(sm + o.vw);   // [8][DN] pending values times their decay
  float* sP = sKw;                                    // [4][32][16]
  uint32_t* sAh = reinterpret_cast<uint32_t*>(sm + o.a);  // [32] rows of 48 bytes
  uint32_t* sAl = sAh + kQRows * 12;
  float2* sDen = reinterpret_cast<float2*>(sm + o.den);
  float* sM = reinterpret_cast<float*>(sm + o.m);     // [T][TK]
  uint64_t* bar = reinterpret_cast<uint64_t*>(sm + o.bar);
  // a thread gave up waiting for the state: nothing is written
  volatile int* late = reinterpret_cast<volatile int*>(sm + o.late);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, j = lane & 3;
  const int b = blockIdx.x, s = blockIdx.y, sl = blockIdx.z, sidx = b * a.Hs + s;
  const int rep = a.rep, R = rep * T;
  const int kvh = a.kvrep == 1 ? sidx : b * a.Hkv + s / a.kvrep;
  const int d0 = sl * DN;
  constexpr int tile = FP * 128;  // bytes of 32 columns

  if (tid == 0) {
    tc::mbar_init(bar, 1);
    *late = 0;
    tc::fence_mbar_init();
    tc::mbar_expect_tx(bar, HALVES * tile);  // rows F .. FP and columns beyond D arrive as zeros
#pragma unroll
    for (int h = 0; h < HALVES; ++h)
      if (h || !a.withhold) tc::tma_load_3d(sm + h * tile, &ts, d0 + 32 * h, 0, sidx, bar);
  }
  // small loads: they arrive while the rest is staged
  const size_t grow = a.gph ? (size_t)b * a.H + s : (size_t)b;
  // lane r of every warp holds the gates of tokens r and r + 32
  const float lg0 = lane < T ? a.lg[grow * T + lane] : 0.f;
  const float lg1 = lane + 32 < T ? a.lg[grow * T + lane + 32] : 0.f;
  float lgp0 = lane < Tp ? a.lg_p[grow * Tp + lane] : 0.f;
  float lgp1 = lane + 32 < Tp ? a.lg_p[grow * Tp + lane + 32] : 0.f;
  const int n = Tp ? (a.count ? min(max(a.count[b], 0), Tp) : Tp) : 0;
  float* Zs = a.Z + (size_t)sidx * F;
  constexpr int ZN = (FP + NT - 1) / NT;  // elements of z a thread owns
  float z[ZN];
#pragma unroll
  for (int i = 0; i < ZN; ++i) z[i] = tid + i * NT < F ? Zs[tid + i * NT] : 0.f;
  // the first pending keys and values, before it is known how many stand
  const bf16* kp = a.fk_p + (size_t)kvh * Tp * F;
  const bf16* vp = a.v_p + (size_t)kvh * Tp * D + d0;
  // (bits in whole registers: packing them in pairs would wait for the loads)
  uint32_t kk[ZN][kPend], vv[kPend * DN / NT];
  const auto bits = [](const bf16* p) {
    return (uint32_t)__ldg(reinterpret_cast<const unsigned short*>(p));
  };
  const auto fetch = [&](int t0) {
#pragma unroll
    for (int i = 0; i < ZN; ++i)
#pragma unroll
      for (int t = 0; t < kPend; ++t) {
        const int f = tid + i * NT;
        kk[i][t] = t0 + t < Tp && f < F ? bits(kp + (t0 + t) * F + f) : 0u;
      }
#pragma unroll
    for (int i = 0; i < kPend * DN / NT; ++i) {
      const int t = t0 + (tid + i * NT) / DN, d = (tid + i * NT) % DN;
      vv[i] = t < Tp && d0 + d < D ? bits(vp + t * D + d) : 0u;
    }
  };
  fetch(0);
  const bf16* fq = a.fq + (size_t)(b * a.H + s * rep) * T * F;
  if (T) {
    stage_rows(sK, LD, FP, F, a.fk + (size_t)kvh * T * F, T, F, TK, NT);
    stage_rows(sQ, LD, FP, F, fq, min(R, kQRows), F, kQRows, NT);
    stage_rows(sV, LV, DN, D, a.v + (size_t)kvh * T * D + d0, T, D - d0, TK, NT);
    cp_async_commit();
  }
  // decays: M of the block (a warp a token), w of the pending tokens (every warp)
  for (int t = warp; t < T; t += NT / 32) {
    float e0 = lane <= t ? lg0 : 0.f, e1 = lane + 32 <= t ? lg1 : 0.f;
    const float all = expf(after(e0, e1, T));
    e0 = expf(e0), e1 = expf(e1);
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const int k = lane + 32 * i;
      if (k < TK)
        sM[t * TK + k] = k <= t ? (i ? e1 : e0) : (k == T || k == T + 1 ? all : 0.f);
    }
  }
  lgp0 = lane < n ? lgp0 : 0.f;
  lgp1 = lane + 32 < n ? lgp1 : 0.f;
  const float gn = expf(after(lgp0, lgp1, n));
  const float w0 = expf(lgp0), w1 = expf(lgp1);
  const auto w_of = [&](int t) { return __shfl_sync(0xffffffffu, t < 32 ? w0 : w1, t & 31); };
  if (n && a.nsl > 1) cluster_arrive();  // every slice reads z before slice 0 writes it
#pragma unroll
  for (int i = 0; i < ZN; ++i) z[i] *= gn;
  // kPend pending tokens to shared memory: keys as they are, values times their decay
  const auto stage = [&](int t0) {
#pragma unroll
    for (int i = 0; i < ZN; ++i) {
      const int f = tid + i * NT;
      // within a step the four rows of a thread are neighbours: one 16-byte read
      const int at = (f & ~15) | (f & 6) << 1 | (f >> 2 & 2) | (f & 1);
#pragma unroll
      for (int t = 0; t < kPend; ++t)
        if (t0 + t < n) {
          const float x = bf16_lo(kk[i][t]), w = w_of(t0 + t);
          if (f < FP) sKw[t * FP + at] = x;
          z[i] += w * x;
        }
    }
#pragma unroll
    for (int i = 0; i < kPend * DN / NT; ++i) {
      const int t = t0 + (tid + i * NT) / DN;  // the same for a warp
      if (t < n) sVw[tid + i * NT] = w_of(t) * bf16_lo(vv[i]);
    }
  };
  if (n) stage(0);
  __syncthreads();

  // the state into registers: rows (2j, 2j+1) and (2j+8, 2j+9) of step ks, columns
  // g and 8 + g of this warp's 16
  f32x2 st[NH][2][2];  // [step][rows][column]
  const int cg = warp % (2 * HALVES), fh = warp / (2 * HALVES), half = cg >> 1;
  const int c = (cg & 1) * 16 + g;  // within the 32 of its tile
  cp_async_wait_all();  // here, not at their use: after the stores below it waits for those too
  if (!tc::mbar_wait(bar, 0, 95)) *late = 1;
  // (f & 7 is 2j or 2j + 1 whatever the step: two swizzled addresses and constants)
  float *even[2], *odd[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int cc = c + 8 * i, r = fh * NH * 16 + 2 * j;
    even[i] = reinterpret_cast<float*>(sm + half * tile + r * 128) +
              ((((cc >> 2) ^ (2 * j)) << 2) | (cc & 3));
    odd[i] = reinterpret_cast<float*>(sm + half * tile + (r + 1) * 128) +
             ((((cc >> 2) ^ (2 * j + 1)) << 2) | (cc & 3));
  }
#pragma unroll
  for (int ks = 0; ks < NH; ++ks)
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        st[ks][p][i] = pack2(even[i][(ks * 16 + 8 * p) * 32], odd[i][(ks * 16 + 8 * p) * 32]);
  if (n) {
    const f32x2 gg = pack2(gn, gn);
#pragma unroll
    for (int ks = 0; ks < NH; ++ks)
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int i = 0; i < 2; ++i) st[ks][p][i] = mul2(st[ks][p][i], gg);
    for (int t0 = 0; t0 < n; t0 += kPend) {
      const int nt = min(kPend, n - t0);
      if (t0) {
        fetch(t0);
        __syncthreads();  // the tokens before have been folded in
        stage(t0);
        __syncthreads();
      }
      for (int t = 0; t < nt; ++t) {
        const float v0 = sVw[t * DN + half * 32 + c], v1 = sVw[t * DN + half * 32 + c + 8];
        const f32x2 va = pack2(v0, v0), vb = pack2(v1, v1);
        const ulonglong2* kr =
            reinterpret_cast<const ulonglong2*>(sKw + t * FP + fh * NH * 16 + 4 * j);
#pragma unroll
        for (int ks = 0; ks < NH; ++ks) {
          const ulonglong2 k4 = kr[ks * 4];
          st[ks][0][0] = fma2(k4.x, va, st[ks][0][0]);
          st[ks][0][1] = fma2(k4.x, vb, st[ks][0][1]);
          st[ks][1][0] = fma2(k4.y, va, st[ks][1][0]);
          st[ks][1][1] = fma2(k4.y, vb, st[ks][1][1]);
        }
      }
    }
    // back through shared memory (each thread over its own elements) and TMA, which
    // leaves out what lies beyond F and D
#pragma unroll
    for (int ks = 0; ks < NH; ++ks)
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          unpack2(st[ks][p][i], even[i][(ks * 16 + 8 * p) * 32], odd[i][(ks * 16 + 8 * p) * 32]);
    tc::fence_proxy_async_smem();
    __syncthreads();
    if (tid == 0 && !*late) {
#pragma unroll
      for (int h = 0; h < HALVES; ++h)
        if (d0 + 32 * h < D) tc::tma_store_3d(&ts, sm + h * tile, d0 + 32 * h, 0, sidx);
      tc::bulk_commit();
    }
    if (a.nsl > 1) cluster_wait();
    if (sl == 0 && !*late)
#pragma unroll
      for (int i = 0; i < ZN; ++i)
        if (tid + i * NT < F) Zs[tid + i * NT] = z[i];
  }
  if (!T) {
    if (tid == 0) tc::bulk_wait_read0();
    if (tid == 0 && *late) tc::mbar_wait(bar, 0, 95);
    return;
  }

  // z as two more keys
  __syncthreads();  // keys and queries are there (their zero rows too)
#pragma unroll
  for (int i = 0; i < ZN; ++i) {
    const int f = tid + i * NT;
    if (f < FP) {
      const bf16 h = __float2bfloat16_rn(z[i]);
      sK[T * LD + f] = h;
      sK[(T + 1) * LD + f] = __float2bfloat16_rn(z[i] - __bfloat162float(h));
    }
  }
  // B fragments of q S: bf16 hi and lo parts of the registers
  uint32_t hi[NH][2][2], lo[NH][2][2];  // [step][column][rows]
#pragma unroll
  for (int ks = 0; ks < NH; ++ks)
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float x0, x1;
        unpack2(st[ks][p][i], x0, x1);
        const uint32_t h = pack_bf16(x0, x1);
        hi[ks][i][p] = h;
        lo[ks][i][p] = pack_bf16(x0 - bf16_lo(h), x1 - bf16_hi(h));
      }
  __syncthreads();

  // ldmatrix rows of this lane: queries (A), keys (B), a' (A)
  const uint32_t aq = smem_u32(sQ) + (lane & 15) * (LD * 2) + (lane >> 4) * 16;
  const uint32_t ak = smem_u32(sK) + ((lane & 7) + (lane >> 4) * 8) * (LD * 2) + (lane >> 3 & 1) * 16;
  const uint32_t aa = smem_u32(sAh) + (lane & 15) * 48 + (lane >> 4) * 16;
  const int vcol = cg * 16;  // this warp's columns of V and y
  const uint32_t av = smem_u32(sV) + (lane & 15) * (LV * 2) + vcol * 2 + (lane >> 4) * 16;
  const int quarter = warp & 3;  // of F, for the scores
  for (int r0 = 0; r0 < R; r0 += kQRows) {
    if (r0) {
      __syncthreads();
      stage_rows(sQ, LD, FP, F, fq + (size_t)r0 * F, min(R - r0, kQRows), F, kQRows, NT);
      cp_async_commit();
      cp_async_wait_all();
      __syncthreads();
    }
    // [row tile][column tile] of q S over this half of F, and a' V of row tile fh
    float x[2][2][4], out[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[0][i][e] = x[1][i][e] = out[i][e] = 0.f;
    float den[kQRows * 8 / NT];
#pragma unroll
    for (int i = 0; i < kQRows * 8 / NT; ++i) den[i] = 0.f;
    for (int k0 = 0; k0 < TK; k0 += 16) {
      // scores of 16 keys: each warp a quarter of F, for one row tile (or, with four warps, both)
#pragma unroll
      for (int rt = warp >> 2; rt < 2; rt += HALVES) {
        float sc[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[i][e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          uint32_t qa[4], kb[4];
          ldsm_x4(qa, aq + rt * (16 * LD * 2) + (quarter * KS + ks) * 32);
          ldsm_x4(kb, ak + k0 * (LD * 2) + (quarter * KS + ks) * 32);
          mma16816(sc[0], qa, kb[0], kb[1]);
          mma16816(sc[1], qa, kb[2], kb[3]);
        }
        float* p = sP + (quarter * kQRows + rt * 16 + g) * 16 + 2 * j;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          *reinterpret_cast<float2*>(p + 8 * i) = make_float2(sc[i][0], sc[i][1]);
          *reinterpret_cast<float2*>(p + 128 + 8 * i) = make_float2(sc[i][2], sc[i][3]);
        }
      }
      if (k0 == 0) {
#pragma unroll
        for (int ks = 0; ks < NH; ++ks)
#pragma unroll
          for (int rt = 0; rt < 2; ++rt) {
            uint32_t qa[4];
            ldsm_x4(qa, aq + rt * (16 * LD * 2) + (fh * NH + ks) * 32);
#pragma unroll
            for (int i = 0; i < 2; ++i) mma16816(x[rt][i], qa, hi[ks][i][0], hi[ks][i][1]);
#pragma unroll
            for (int i = 0; i < 2; ++i) mma16816(x[rt][i], qa, lo[ks][i][0], lo[ks][i][1]);
          }
      }
      __syncthreads();
      // a' = (q k^T) o M, two keys a thread, and its row sum
#pragma unroll
      for (int i = 0; i < kQRows * 8 / NT; ++i) {
        const int r = (tid + i * NT) >> 3, k = (tid & 7) * 2;
        float2 p = make_float2(0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float2 v = *reinterpret_cast<const float2*>(sP + (w * kQRows + r) * 16 + k);
          p.x += v.x;
          p.y += v.y;
        }
        const float2 m = *reinterpret_cast<const float2*>(sM + (r0 + r) % T * TK + k0 + k);
        p.x *= m.x;
        p.y *= m.y;
        den[i] += p.x + p.y;
        const uint32_t h = pack_bf16(p.x, p.y);
        sAh[(r * 48 + k * 2) / 4] = h;
        sAl[(r * 48 + k * 2) / 4] = pack_bf16(p.x - bf16_lo(h), p.y - bf16_hi(h));
      }
      __syncthreads();
      uint32_t vb[4], ph[4], pl[4];  // vb: 16 keys by this warp's two column tiles
      ldsm_x4_t(vb, av + k0 * (LV * 2));
      ldsm_x4(ph, aa + fh * (16 * 48));
      ldsm_x4(pl, aa + kQRows * 48 + fh * (16 * 48));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mma16816(out[i], ph, vb[2 * i], vb[2 * i + 1]);
        mma16816(out[i], pl, vb[2 * i], vb[2 * i + 1]);
      }
    }
#pragma unroll
    for (int i = 0; i < kQRows * 8 / NT; ++i) {
#pragma unroll
      for (int w = 1; w < 8; w <<= 1) den[i] += __shfl_xor_sync(0xffffffffu, den[i], w);
      const int r = (tid + i * NT) >> 3;
      if ((tid & 7) == 0)  // d_t / den and 1 / den
        sDen[r] = make_float2(sM[(r0 + r) % T * TK + T], 1.f / fmaxf(den[i], kTiny));
    }
    // the other half's sums of this warp's row tile, over the queries (they are done)
    float4* sX = reinterpret_cast<float4*>(sQ);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      sX[(warp * 2 + i) * 32 + lane] = make_float4(fh ? x[0][i][0] : x[1][i][0],
                                                   fh ? x[0][i][1] : x[1][i][1],
                                                   fh ? x[0][i][2] : x[1][i][2],
                                                   fh ? x[0][i][3] : x[1][i][3]);
    __syncthreads();
    const bool live = !*late;
    float probe = 0.f;  // NaN once an output is not finite
    const int other = fh ? warp - 2 * HALVES : warp + 2 * HALVES, row = r0 + fh * 16 + g;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 o4 = sX[(other * 2 + i) * 32 + lane];
      const float q[4] = {o4.x, o4.y, o4.z, o4.w};
      const int dd = d0 + vcol + 8 * i + 2 * j;
      bf16* yr = a.y + ((size_t)(b * a.H + s * rep) * T + row) * D + dd;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (row + 8 * h < R && dd < D && live) {  // D is a multiple of 4
          const float2 f = sDen[fh * 16 + g + 8 * h];
          float y[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float mine = fh ? x[1][i][2 * h + e] : x[0][i][2 * h + e];
            y[e] = (f.x * (mine + q[2 * h + e]) + out[i][2 * h + e]) * f.y;
            probe = fmaf(y[e], 0.f, probe);
          }
          *reinterpret_cast<uint32_t*>(yr + 8 * h * D) = pack_bf16(y[0], y[1]);
        }
    }
    if (probe != 0.f) redo<KS, HALVES>(a, sm, r0);
  }
  if (tid == 0) tc::bulk_wait_read0();  // the state has left shared memory
  // once more for a load that may still be on its way
  if (tid == 0 && *late) tc::mbar_wait(bar, 0, 95);
}

template <int KS, int HALVES>
int launch_gla_block(const GlaBlockArgs& a, int B, cudaStream_t stream) {
  auto fn = tc::encode_tiled_fn();
  if (!fn) {
    set_error("lz_gla_decode_block: cuTensorMapEncodeTiled is not available");
    return LZ_ERR_CUDA;
  }
  CUtensorMap ts;
  const cuuint64_t dims[3] = {(cuuint64_t)a.D, (cuuint64_t)a.F, (cuuint64_t)B * a.Hs};
  const cuuint64_t strides[2] = {(cuuint64_t)a.D * 4, (cuuint64_t)a.F * a.D * 4};
  const cuuint32_t box[3] = {32, 64 * KS, 1}, es[3] = {1, 1, 1};
  const CUresult r = fn(&ts, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, a.S, dims, strides, box, es,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("lz_gla_decode_block: the tensor map of the state could not be encoded, driver code " +
              std::to_string((int)r));
    return LZ_ERR_CUDA;
  }
  static bool done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 64 && !done[dev]) {
    const int most = block_smem(KS, HALVES, kMaxBlock).total;
    cudaError_t e = cudaFuncSetAttribute(gla_block_kernel<KS, HALVES>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e != cudaSuccess) {
      set_error(std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
      return LZ_ERR_CUDA;
    }
    done[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(B, a.Hs, a.nsl);
  cfg.blockDim = dim3(128 * HALVES);
  cfg.dynamicSmemBytes = block_smem(KS, HALVES, a.T).total;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = a.nsl;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, gla_block_kernel<KS, HALVES>, ts, a);
  if (e != cudaSuccess) {
    set_error(std::string("gla_block_kernel: ") + cudaGetErrorString(e));
    return LZ_ERR_CUDA;
  }
  count_launches(1);
  return check_launch("gla_block_kernel");
}

}  // namespace
std::atomic<int> g_withhold_block{0};  // lz_test_withhold_block_load
int gla_block_timeout_flag(unsigned int* out) { return tc::read_timeout_flag_here(out); }
int gla_block_timeout_clear() { return tc::clear_timeout_flag_here(); }
}  // namespace lz

extern "C" int lz_test_withhold_block_load(int on) {
  return lz::g_withhold_block.exchange(on ? 1 : 0);
}

extern "C" int lz_gla_decode_block(const void* fq, const void* fk, const void* v,
                                   const float* log_gamma, int gate_per_head, const void* fk_prev,
                                   const void* v_prev, const float* log_gamma_prev,
                                   const int* count, float* state, float* zstate, void* y, int B,
                                   int H, int Hkv, int Hs, int T, int T_prev, int F, int D,
                                   void* stream) {
  using namespace lz;
  clear_error();
  LZ_REQUIRE(B >= 1 && H >= 1 && Hkv >= 1 && F >= 1 && D >= 1 && T >= 0 && T_prev >= 0,
             LZ_ERR_INVALID_ARGUMENT, "sizes must be positive");
  LZ_REQUIRE(T + T_prev >= 1, LZ_ERR_INVALID_ARGUMENT, "no tokens: T and T_prev are both 0");
  LZ_REQUIRE(H % Hkv == 0, LZ_ERR_INVALID_ARGUMENT,
             "the key/value head count must divide the query head count");
  LZ_REQUIRE(Hs == H || (Hs == Hkv && !gate_per_head), LZ_ERR_INVALID_ARGUMENT,
             "state heads must be H, or Hkv when the gate is shared by the heads");
  LZ_REQUIRE(T <= kMaxBlock && T_prev <= kMaxBlock, LZ_ERR_UNSUPPORTED,
             "a block holds at most 64 tokens");
  LZ_REQUIRE(F <= 256 && D % 4 == 0 && D <= 256, LZ_ERR_UNSUPPORTED,
             "decode supports F <= 256 and D a multiple of 4 up to 256");
  LZ_REQUIRE((long long)B * H * std::max({T, T_prev, 1}) < (1ll << 31) && Hs <= 65535,
             LZ_ERR_UNSUPPORTED, "too many sequences or heads");
  LZ_REQUIRE(state && zstate, LZ_ERR_INVALID_ARGUMENT, "null pointer");
  LZ_REQUIRE(!T || (fq && fk && v && log_gamma && y), LZ_ERR_INVALID_ARGUMENT, "null pointer");
  LZ_REQUIRE(!T_prev || (fk_prev && v_prev && log_gamma_prev), LZ_ERR_INVALID_ARGUMENT,
             "null pointer in the previous block");
  LZ_REQUIRE(aligned16(state), LZ_ERR_INVALID_ARGUMENT, "state must be 16-byte aligned");
  LZ_REQUIRE(!T || (reinterpret_cast<uintptr_t>(y) & 3) == 0, LZ_ERR_INVALID_ARGUMENT,
             "y must be 4-byte aligned");
  GlaBlockArgs a;
  a.fq = static_cast<const bf16*>(fq);
  a.fk = static_cast<const bf16*>(fk);
  a.v = static_cast<const bf16*>(v);
  a.lg = log_gamma;
  a.fk_p = static_cast<const bf16*>(fk_prev);
  a.v_p = static_cast<const bf16*>(v_prev);
  a.lg_p = log_gamma_prev;
  a.count = count;
  a.S = state;
  a.Z = zstate;
  a.y = static_cast<bf16*>(y);
  a.gph = gate_per_head ? 1 : 0;
  a.T = T;
  a.Tp = T_prev;
  a.H = H;
  a.Hkv = Hkv;
  a.Hs = Hs;
  a.F = F;
  a.D = D;
  auto st = static_cast<cudaStream_t>(stream);
  const int ks = ceil_div(F, 64), halves = D > 32 ? 2 : 1;
  a.nsl = ceil_div(D, 32 * halves);
  a.rep = H / Hs;
  a.kvrep = Hs / Hkv;
  a.withhold = g_withhold_block.load(std::memory_order_relaxed);
#define LZ_GB(K_)                                                      \
  case K_:                                                             \
    return halves == 2 ? launch_gla_block<K_, 2>(a, B, st) \
                       : launch_gla_block<K_, 1>(a, B, st);
  switch (ks) {
    LZ_GB(1) LZ_GB(2) LZ_GB(3) LZ_GB(4)
  }
#undef LZ_GB
  set_error("lz_gla_decode_block: unreachable feature size");
  return LZ_ERR_UNSUPPORTED;
}
