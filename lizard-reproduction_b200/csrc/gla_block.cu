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
// 2 rep T F D multiply-adds: memory. One CTA holds F x 64 (or 32) of a state in
// registers, laid out as the B fragments of mma.sync m16n8k16: thread (g, j) of
// a warp holds rows 2j, 2j+1, 2j+8, 2j+9 of each 16-row step and columns
// 4g..4g+3 of a 32-column group, so a load is one float4 and a warp's load
// covers four whole 128-byte lines, and tile i of the group stands for columns
// 4n + i. The update runs in fp32 in those registers (k and v are bf16, their
// products exact); for q S the registers are split once into bf16 hi + lo parts
// (relative error 2^-17, against the 2^-9 of the bf16 output). The four warps
// of a column half each contract a quarter of F and are added through shared
// memory in a fixed order.
#include <algorithm>

#include "common.cuh"

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
  int gph, T, Tp, H, Hkv, Hs, F, D, nsl;
};

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}

// rows x ncols bf16 (row stride ncols) into shared rows of ld elements, columns
// ncols..width zeroed; 16-byte loads when rows keep that alignment.
__device__ __forceinline__ void stage_rows(bf16* s, int ld, int width, const bf16* g, int rows,
                                           int ncols, int pad_rows, int nthreads) {
  const bool vec = (ncols & 7) == 0 && (reinterpret_cast<uintptr_t>(g) & 15) == 0;
  if (vec) {
    const int cpr = width >> 3;
    for (int i = threadIdx.x; i < pad_rows * cpr; i += nthreads) {
      const int r = i / cpr, c = (i - r * cpr) * 8;
      cp_async16(s + r * ld + c, r < rows && c < ncols ? g + (size_t)r * ncols + c : g,
                 r < rows && c < ncols);
    }
  } else {
    for (int i = threadIdx.x; i < pad_rows * width; i += nthreads) {
      const int r = i / width, c = i - r * width;
      s[r * ld + c] = r < rows && c < ncols ? g[(size_t)r * ncols + c] : __float2bfloat16_rn(0.f);
    }
  }
}

// KS: 16-row steps of F a warp owns (F <= 64 KS). HALVES: 32-column groups a CTA.
template <int KS, int HALVES>
__global__ void __launch_bounds__(128 * HALVES)
gla_block_kernel(const GlaBlockArgs a) {
  constexpr int NT = 128 * HALVES, FP = 64 * KS, LD = FP + 8, DN = 32 * HALVES;
  extern __shared__ __align__(16) unsigned char smraw[];
  const int T = a.T, Tp = a.Tp, F = a.F, D = a.D;
  const int TK = (T + 7) & ~7;  // block keys, padded to mma columns
  const int LDR = DN + TK + 4;  // row of a partial: DN values, TK scores
  bf16* sQ = reinterpret_cast<bf16*>(smraw);      // [16][LD]
  bf16* sK = sQ + 16 * LD;                        // [TK][LD] block keys
  bf16* sKp = sK + TK * LD;                       // [Tp][LD] pending keys
  float* sV = reinterpret_cast<float*>(sKp + ((Tp + 1) & ~1) * LD);  // [T][DN]
  float* sVp = sV + T * DN;                       // [Tp][DN], then the partials
  float* sRed = sVp + Tp * DN;                    // [4][16][LDR]
  float* sA = sRed + 4 * 16 * LDR;                // [16][TK + 1]
  float* sM = sA + 16 * (TK + 1);                 // [T][T] decay of key s at token t
  float* sDec = sM + T * T;                       // [T]
  float* sW = sDec + T;                           // [Tp]
  float* sZ = sW + Tp;                            // [FP]
  float* sQz = sZ + FP;                           // [16]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int wf = warp & 3, wd = warp >> 2, g = lane >> 2, j = lane & 3;
  const int sidx = blockIdx.x / a.nsl, sl = blockIdx.x - sidx * a.nsl;
  const int b = sidx / a.Hs, s = sidx - b * a.Hs;
  const int rep = a.H / a.Hs, R = rep * T;
  const int kvh = a.Hs == a.Hkv ? sidx : kv_head(b * a.H + s, a.H, a.H / a.Hkv);
  const int d0 = sl * DN, dcol = d0 + wd * 32 + 4 * g;
  const bool dok = dcol < D;
  const int n = Tp ? (a.count ? min(max(a.count[b], 0), Tp) : Tp) : 0;

  // the state first: every load is in flight before anything waits
  float4 st[KS][4];
  float* Sb = a.S + (size_t)sidx * F * D + dcol;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int f = (wf * KS + ks) * 16 + 2 * j + (u & 1) + (u >> 1) * 8;
      st[ks][u] = dok && f < F ? *reinterpret_cast<const float4*>(Sb + (size_t)f * D)
                               : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  // block and pending keys, values and gates
  if (T) stage_rows(sK, LD, FP, a.fk + (size_t)kvh * T * F, T, F, TK, NT);
  if (n) stage_rows(sKp, LD, FP, a.fk_p + (size_t)kvh * Tp * F, n, F, n, NT);
  const bf16* fq = a.fq + (size_t)(b * a.H + s * rep) * T * F;
  if (T) stage_rows(sQ, LD, FP, fq, min(R, 16), F, 16, NT);
  cp_async_commit();
  for (int i = tid; i < T * DN; i += NT) {
    const int t = i / DN, d = d0 + i - t * DN;
    sV[i] = d < D ? __bfloat162float(a.v[((size_t)kvh * T + t) * D + d]) : 0.f;
  }
  for (int i = tid; i < n * DN; i += NT) {
    const int t = i / DN, d = d0 + i - t * DN;
    sVp[i] = d < D ? __bfloat162float(a.v_p[((size_t)kvh * Tp + t) * D + d]) : 0.f;
  }
  const size_t grow = a.gph ? (size_t)b * a.H + s : (size_t)b;
  if (tid < T) {  // column tid of the block's decays: running sums from its own key on
    const float* lg = a.lg + grow * T;
    float acc = 0.f;
    for (int t = 0; t < tid; ++t) sM[t * T + tid] = 0.f;
    sM[tid * T + tid] = 1.f;
    for (int t = tid + 1; t < T; ++t) {
      acc += lg[t];
      sM[t * T + tid] = expf(acc);
    }
  }
  const int tp = NT - 1 - tid;  // from the other end: other warps
  if (tp < T) {
    float acc = 0.f;
    for (int t = 0; t <= tp; ++t) acc += a.lg[grow * T + t];
    sDec[tp] = expf(acc);
  }
  float gn = 1.f;
  if (n) {
    const float* lg = a.lg_p + grow * Tp;
    float acc = 0.f;
    for (int t = 0; t < n; ++t) acc += lg[t];
    gn = expf(acc);
    if (tid < n) {
      acc = 0.f;
      for (int t = tid + 1; t < n; ++t) acc += lg[t];
      sW[tid] = expf(acc);
    }
  }
  cp_async_wait_all();
  __syncthreads();

  // the normaliser (every slice's CTA needs it; slice 0 writes it once all have read it)
  float* Zs = a.Z + (size_t)sidx * F;
  for (int f = tid; f < FP; f += NT) {
    float z = f < F ? Zs[f] : 0.f;
    if (n) {
      z *= gn;
      for (int t = 0; t < n; ++t) z += sW[t] * __bfloat162float(sKp[t * LD + f]);
    }
    sZ[f] = z;
  }
  if (n && a.nsl > 1) cluster_arrive();

  // the state: S <- g S + sum w_t k_t^T v_t, in fp32
  if (n) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        st[ks][u].x *= gn;
        st[ks][u].y *= gn;
        st[ks][u].z *= gn;
        st[ks][u].w *= gn;
      }
    for (int t = 0; t < n; ++t) {
      const float w = sW[t];
      const float4 vv = *reinterpret_cast<const float4*>(sVp + t * DN + wd * 32 + 4 * g);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const bf16* kr = sKp + t * LD + (wf * KS + ks) * 16 + 2 * j;
        const uint32_t k01 = *reinterpret_cast<const uint32_t*>(kr);
        const uint32_t k89 = *reinterpret_cast<const uint32_t*>(kr + 8);
        const float kf[4] = {w * bf16_lo(k01), w * bf16_hi(k01), w * bf16_lo(k89),
                             w * bf16_hi(k89)};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          st[ks][u].x += kf[u] * vv.x;
          st[ks][u].y += kf[u] * vv.y;
          st[ks][u].z += kf[u] * vv.z;
          st[ks][u].w += kf[u] * vv.w;
        }
      }
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int f = (wf * KS + ks) * 16 + 2 * j + (u & 1) + (u >> 1) * 8;
        if (dok && f < F) *reinterpret_cast<float4*>(Sb + (size_t)f * D) = st[ks][u];
      }
  }
  if (n && a.nsl > 1) cluster_wait();
  __syncthreads();
  if (n && sl == 0)
    for (int f = tid; f < F; f += NT) Zs[f] = sZ[f];
  if (!T) return;

  // B fragments of q S: bf16 hi and lo parts of the registers
  uint32_t hi[KS][4][2], lo[KS][4][2];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const float x0 = reinterpret_cast<const float*>(&st[ks][2 * p])[i];
        const float x1 = reinterpret_cast<const float*>(&st[ks][2 * p + 1])[i];
        const uint32_t h = pack_bf16(x0, x1);
        hi[ks][i][p] = h;
        lo[ks][i][p] = pack_bf16(x0 - bf16_lo(h), x1 - bf16_hi(h));
      }

  for (int r0 = 0; r0 < R; r0 += 16) {
    if (r0) {
      stage_rows(sQ, LD, FP, fq + (size_t)r0 * F, min(R - r0, 16), F, 16, NT);
      cp_async_commit();
      cp_async_wait_all();
      __syncthreads();
    }
    float acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[i][c] = 0.f;
    uint32_t qa[KS][4];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      lda_rm(qa[ks], sQ, LD, 0, (wf * KS + ks) * 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mma16816(acc[i], qa[ks], hi[ks][i][0], hi[ks][i][1]);
        mma16816(acc[i], qa[ks], lo[ks][i][0], lo[ks][i][1]);
      }
    }
    // thread (g, j): rows g, g + 8; tile i's columns 2j, 2j+1 are 4 (2j) + i, 4 (2j+1) + i
    float* red = sRed + wf * 16 * LDR;
    const int c0 = wd * 32 + 8 * j;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float* row = red + (g + 8 * h) * LDR + c0;
      *reinterpret_cast<float4*>(row) =
          make_float4(acc[0][2 * h], acc[1][2 * h], acc[2][2 * h], acc[3][2 * h]);
      *reinterpret_cast<float4*>(row + 4) =
          make_float4(acc[0][2 * h + 1], acc[1][2 * h + 1], acc[2][2 * h + 1], acc[3][2 * h + 1]);
    }
    // scores of the block's own keys, eight at a time, dealt to the column halves
    for (int k0 = wd * 8; k0 < TK; k0 += 8 * HALVES) {
      float sc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const bf16* kr = sK + (k0 + g) * LD + (wf * KS + ks) * 16 + 2 * j;
        mma16816(sc, qa[ks], *reinterpret_cast<const uint32_t*>(kr),
                 *reinterpret_cast<const uint32_t*>(kr + 8));
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<float2*>(red + (g + 8 * h) * LDR + DN + k0 + 2 * j) =
            make_float2(sc[2 * h], sc[2 * h + 1]);
    }
    // q . z, a warp per row
    for (int r = warp; r < 16; r += NT / 32) {
      float x = 0.f;
#pragma unroll
      for (int f = 0; f < FP / 32; ++f)
        x += __bfloat162float(sQ[r * LD + lane + 32 * f]) * sZ[lane + 32 * f];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      if (lane == 0) sQz[r] = x;
    }
    __syncthreads();
    for (int e = tid; e < 16 * T; e += NT) {
      const int r = e / T, k = e - r * T, t = (r0 + r) % T;
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) x += sRed[(w * 16 + r) * LDR + DN + k];
      sA[r * (TK + 1) + k] = k <= t ? x * sM[t * T + k] : 0.f;
    }
    __syncthreads();
    for (int e = tid; e < 16 * (DN / 4); e += NT) {
      const int r = e / (DN / 4), c = (e - r * (DN / 4)) * 4, d = d0 + c;
      if (r0 + r >= R || d >= D) continue;
      const int t = (r0 + r) % T;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float4 p = *reinterpret_cast<const float4*>(sRed + (w * 16 + r) * LDR + c);
        x.x += p.x;
        x.y += p.y;
        x.z += p.z;
        x.w += p.w;
      }
      const float dec = sDec[t];
      float den = dec * sQz[r];
      x.x *= dec;
      x.y *= dec;
      x.z *= dec;
      x.w *= dec;
      for (int k = 0; k <= t; ++k) {
        const float w = sA[r * (TK + 1) + k];
        const float4 vv = *reinterpret_cast<const float4*>(sV + k * DN + c);
        den += w;
        x.x += w * vv.x;
        x.y += w * vv.y;
        x.z += w * vv.z;
        x.w += w * vv.w;
      }
      const float inv = 1.f / fmaxf(den, kTiny);
      bf16* yr = a.y + ((size_t)(b * a.H + s * rep) * T + r0 + r) * D + d;
      *reinterpret_cast<uint2*>(yr) =
          make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
    }
    __syncthreads();
  }
}

size_t block_smem(int KS, int HALVES, int T, int Tp) {
  const int LD = 64 * KS + 8, DN = 32 * HALVES, TK = (T + 7) & ~7, LDR = DN + TK + 4;
  size_t n = (size_t)(16 + TK + ((Tp + 1) & ~1)) * LD * 2;
  n += ((size_t)(T + Tp) * DN + 4 * 16 * LDR + 16 * (TK + 1) + (size_t)T * T + T + Tp + 64 * KS +
        16) * 4;
  return n;
}

template <int KS, int HALVES>
int launch_gla_block(const GlaBlockArgs& a, unsigned states, cudaStream_t stream) {
  const size_t smem = block_smem(KS, HALVES, a.T, a.Tp);
  // the largest block (64 pending and 64 new tokens) needs under the 227 KB limit
  static bool done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 64 && !done[dev]) {
    cudaError_t e = cudaFuncSetAttribute(gla_block_kernel<KS, HALVES>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)block_smem(KS, HALVES, kMaxBlock, kMaxBlock));
    if (e != cudaSuccess) {
      set_error(std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
      return LZ_ERR_CUDA;
    }
    done[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(states * a.nsl);
  cfg.blockDim = dim3(128 * HALVES);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = a.nsl;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, gla_block_kernel<KS, HALVES>, a);
  if (e != cudaSuccess) {
    set_error(std::string("gla_block_kernel: ") + cudaGetErrorString(e));
    return LZ_ERR_CUDA;
  }
  count_launches(1);
  return check_launch("gla_block_kernel");
}

}  // namespace
}  // namespace lz

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
  LZ_REQUIRE((long long)B * Hs * 8 < (1ll << 31), LZ_ERR_UNSUPPORTED, "too many state heads");
  LZ_REQUIRE(state && zstate, LZ_ERR_INVALID_ARGUMENT, "null pointer");
  LZ_REQUIRE(!T || (fq && fk && v && log_gamma && y), LZ_ERR_INVALID_ARGUMENT, "null pointer");
  LZ_REQUIRE(!T_prev || (fk_prev && v_prev && log_gamma_prev), LZ_ERR_INVALID_ARGUMENT,
             "null pointer in the previous block");
  LZ_REQUIRE(aligned16(state), LZ_ERR_INVALID_ARGUMENT, "state must be 16-byte aligned");
  LZ_REQUIRE(!T || (reinterpret_cast<uintptr_t>(y) & 7) == 0, LZ_ERR_INVALID_ARGUMENT,
             "y must be 8-byte aligned");
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
  const unsigned states = (unsigned)(B * Hs);
  const int ks = ceil_div(F, 64), halves = D > 32 ? 2 : 1;
  a.nsl = ceil_div(D, 32 * halves);
#define LZ_GB(K_)                                                      \
  case K_:                                                             \
    return halves == 2 ? launch_gla_block<K_, 2>(a, states, st) \
                       : launch_gla_block<K_, 1>(a, states, st);
  switch (ks) {
    LZ_GB(1) LZ_GB(2) LZ_GB(3) LZ_GB(4)
  }
#undef LZ_GB
  set_error("lz_gla_decode_block: unreachable feature size");
  return LZ_ERR_UNSUPPORTED;
}
