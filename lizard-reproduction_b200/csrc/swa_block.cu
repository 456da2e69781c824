// A block of new tokens through the sliding-window ring, with the ring left at
// the accepted prefix.
//
// As in the GLA block step, the call first writes the accepted tokens of the
// PREVIOUS block (n = count[b] of them: rotated keys and values, into slots
// (pos + t) % W) and then attends this block's T tokens, at positions base =
// pos + n and on, to the ring and to the block's earlier tokens:
//   y_t = sum_i p_ti v_i / (sum_i p_ti + sum_m exp(meta_m)),  p_ti = exp(q_t . k_i / sqrt(D))
// over the keys at positions base + t - W < position <= base + t. The block's
// own keys never enter the ring here, so a refused token leaves no trace.
//
// One CTA per (batch row, key/value head): the ring is read once for all rep T
// query rows of the group. 64 keys at a time are staged in shared memory as
// bf16 hi + lo parts (the ring is fp32; hi hi + hi lo + lo hi keeps 2^-17 of
// the product, well under the bf16 output) and contracted with mma.sync
// m16n8k16; each of the four warps of a 16-row tile takes 16 of the 64 keys
// with its own running maximum and sum, and the four are merged at the end, so
// a block of few rows still keeps every warp busy. Bound: 8 (W + T) D bytes of
// ring a head against 4 rep T (W + T) D operations: memory.
#include <algorithm>

#include "common.cuh"
#include "tc.cuh"

namespace lz {
namespace {

constexpr int kMaxBlock = 64;    // tokens a block
constexpr int kMaxWindow = 1024;  // as the single-token step
constexpr int kKeys = 64;        // keys a staged tile

struct Heads {  // [B, heads, T, D] in place: strides in elements, last dimension contiguous
  const void* p;
  long long sb, sh, st;
};
struct Rotary {  // [B or 1, T, D] contiguous, sb = 0 for one table for all rows
  const void *cos, *sin;
  long long sb;
  int bf16_;
};
struct SwaBlockArgs {
  Heads q, k, v, kp, vp;
  Rotary rot, rot_p;
  const int *pos, *count;
  const float* meta;
  float *kr, *vr;
  bf16* y;
  int n_meta, T, Tp, H, Hkv, W, D;
};

template <typename T>
__device__ __forceinline__ float ldx(const void* p, long long i);
template <>
__device__ __forceinline__ float ldx<float>(const void* p, long long i) {
  return static_cast<const float*>(p)[i];
}
template <>
__device__ __forceinline__ float ldx<bf16>(const void* p, long long i) {
  return __bfloat162float(static_cast<const bf16*>(p)[i]);
}
__device__ __forceinline__ float ldr(const void* p, long long i, int is_bf16) {
  return is_bf16 ? ldx<bf16>(p, i) : ldx<float>(p, i);
}

// The rotated pair (d, d + D / 2) of a row, each product and sum rounded once,
// as the single-token step rounds them.
template <typename XT>
__device__ __forceinline__ float2 rotated(const void* x, long long row, const Rotary& r,
                                          long long crow, int d, int half) {
  const float x1 = ldx<XT>(x, row + d), x2 = ldx<XT>(x, row + d + half);
  const float c1 = ldr(r.cos, crow + d, r.bf16_), s1 = ldr(r.sin, crow + d, r.bf16_);
  const float c2 = ldr(r.cos, crow + d + half, r.bf16_), s2 = ldr(r.sin, crow + d + half, r.bf16_);
  return make_float2(__fadd_rn(__fmul_rn(x1, c1), -__fmul_rn(x2, s1)),
                     __fadd_rn(__fmul_rn(x2, c2), __fmul_rn(x1, s2)));
}

__device__ __forceinline__ void put(bf16* hi, bf16* lo, int at, float x) {
  const bf16 h = __float2bfloat16_rn(x);
  hi[at] = h;
  lo[at] = __float2bfloat16_rn(x - __bfloat162float(h));
}
__device__ __forceinline__ void put4(bf16* hi, bf16* lo, int at, float4 x) {
  const uint32_t h0 = pack_bf16(x.x, x.y), h1 = pack_bf16(x.z, x.w);
  *reinterpret_cast<uint2*>(hi + at) = make_uint2(h0, h1);
  *reinterpret_cast<uint2*>(lo + at) =
      make_uint2(pack_bf16(x.x - bf16_lo(h0), x.y - bf16_hi(h0)),
                 pack_bf16(x.z - bf16_lo(h1), x.w - bf16_hi(h1)));
}

constexpr size_t swa_block_smem(int DP, int RT) {
  return (size_t)(4 * kKeys + 2 * 16 * RT) * (DP + 8) * 2 + (kKeys + 2 * 64 * RT) * 4;
}

// DP: D padded to whole mma steps. RT: 16-row tiles of queries at once.
template <typename XT, int DP, int RT>
__global__ void __launch_bounds__(128 * RT)
swa_block_kernel(const SwaBlockArgs a) {
  constexpr int NT = 128 * RT, LD = DP + 8, NS = DP / 16;
  extern __shared__ __align__(16) unsigned char smraw[];
  bf16* sKh = reinterpret_cast<bf16*>(smraw);
  bf16* sKl = sKh + kKeys * LD;
  bf16* sVh = sKl + kKeys * LD;
  bf16* sVl = sVh + kKeys * LD;
  bf16* sQh = sVl + kKeys * LD;
  bf16* sQl = sQh + 16 * RT * LD;
  int* sRel = reinterpret_cast<int*>(sQl + 16 * RT * LD);  // [64] position - base
  float* sMax = reinterpret_cast<float*>(sRel + kKeys);    // [RT][4][16]
  float* sSum = sMax + 64 * RT;
  float* sO = reinterpret_cast<float*>(smraw);             // [RT][4][16][DP], after the last tile
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int wk = warp & 3, rt = warp >> 2, g = lane >> 2, j = lane & 3;
  const int T = a.T, W = a.W, D = a.D, half = D / 2;
  const int bk = blockIdx.x, b = bk / a.Hkv, hk = bk - b * a.Hkv;
  const int rep = a.H / a.Hkv, R = rep * T;
  const int pos = a.pos[b];
  const int n = a.Tp ? (a.count ? min(max(a.count[b], 0), a.Tp) : a.Tp) : 0;
  float* kring = a.kr + (size_t)bk * W * D;
  float* vring = a.vr + (size_t)bk * W * D;

  // accepted tokens of the previous block (of more than W, the last W)
  const int t0 = max(0, n - W);
  for (int e = tid; e < (n - t0) * half; e += NT) {
    const int t = t0 + e / half, d = e % half, slot = (int)(((long long)pos + t) % W);
    const float2 kk = rotated<XT>(a.kp.p, b * a.kp.sb + hk * a.kp.sh + t * a.kp.st, a.rot_p,
                                  b * a.rot_p.sb + (long long)t * D, d, half);
    kring[(size_t)slot * D + d] = kk.x;
    kring[(size_t)slot * D + d + half] = kk.y;
    const long long vrow = b * a.vp.sb + hk * a.vp.sh + t * a.vp.st;
    vring[(size_t)slot * D + d] = ldx<XT>(a.vp.p, vrow + d);
    vring[(size_t)slot * D + d + half] = ldx<XT>(a.vp.p, vrow + d + half);
  }
  if (!T) return;
  const long long base = (long long)pos + n;
  const int nr = base < W ? (int)base : W;  // ring rows that hold a token
  const int last = (int)((base - 1 + W) % W);  // slot of the newest (W >= 1)
  const int N = nr + T;
  const float scale = rsqrtf((float)D) * kLog2e;
  const bool vec = (D & 3) == 0 && ((reinterpret_cast<uintptr_t>(a.kr) |
                                     reinterpret_cast<uintptr_t>(a.vr)) & 15) == 0;

  for (int r0 = 0; r0 < R; r0 += 16 * RT) {
    __syncthreads();  // the ring writes above; the merge of the rows before
    for (int e = tid; e < 16 * RT * (DP / 2); e += NT) {
      const int r = e / (DP / 2), d = e - r * (DP / 2), row = r0 + r;
      if (row < R && d < half) {
        const int h = row / T, t = row - h * T;
        const float2 x =
            rotated<XT>(a.q.p, b * a.q.sb + (hk * rep + h) * a.q.sh + t * a.q.st, a.rot,
                        b * a.rot.sb + (long long)t * D, d, half);
        put(sQh, sQl, r * LD + d, x.x);
        put(sQh, sQl, r * LD + d + half, x.y);
      } else if (row >= R) {
        put(sQh, sQl, r * LD + 2 * d, 0.f);
        put(sQh, sQl, r * LD + 2 * d + 1, 0.f);
      } else {  // the padding columns D .. DP
        put(sQh, sQl, r * LD + 2 * d, 0.f);
        put(sQh, sQl, r * LD + 2 * d + 1, 0.f);
      }
    }
    float m[2] = {-1e30f, -1e30f}, l[2] = {0.f, 0.f};
    float o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[i][c] = 0.f;
    // this thread's two rows: their token within the block
    const int rowa = r0 + rt * 16 + g;
    const int ta = rowa % T, tb = (rowa + 8) % T;

    for (int k0 = 0; k0 < N; k0 += kKeys) {
      if (k0) __syncthreads();  // the tile before has been used
      const int nring = min(max(nr - k0, 0), kKeys);  // ring rows of this tile
      for (int e = tid; e < kKeys * (DP / 4); e += NT) {
        const int r = e / (DP / 4), c = (e - r * (DP / 4)) * 4;
        float4 kk = make_float4(0.f, 0.f, 0.f, 0.f), vv = kk;
        if (r < nring) {
          const size_t at = (size_t)(k0 + r) * D + c;
          if (vec) {
            if (c < D) {
              kk = *reinterpret_cast<const float4*>(kring + at);
              vv = *reinterpret_cast<const float4*>(vring + at);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (c + i < D) {
                reinterpret_cast<float*>(&kk)[i] = kring[at + i];
                reinterpret_cast<float*>(&vv)[i] = vring[at + i];
              }
          }
        }
        put4(sKh, sKl, r * LD + c, kk);
        put4(sVh, sVl, r * LD + c, vv);
      }
      for (int r = tid; r < kKeys; r += NT) {
        const int i = k0 + r;
        // a ring slot holds the last position before base that falls on it
        const int back = last - i;
        sRel[r] = i < nr ? -1 - (back < 0 ? back + W : back) : (i < N ? i - nr : 1 << 30);
      }
      if (nring < kKeys) {  // the block's own keys follow the ring's
        __syncthreads();    // over the zeros written above
        const int s0 = k0 + nring - nr, ns = min(kKeys - nring, T - s0);
        for (int e = tid; e < ns * half; e += NT) {
          const int i = e / half, d = e - i * half, s = s0 + i, at = (nring + i) * LD + d;
          const float2 kk = rotated<XT>(a.k.p, b * a.k.sb + hk * a.k.sh + s * a.k.st, a.rot,
                                        b * a.rot.sb + (long long)s * D, d, half);
          put(sKh, sKl, at, kk.x);
          put(sKh, sKl, at + half, kk.y);
          const long long vrow = b * a.v.sb + hk * a.v.sh + s * a.v.st;
          put(sVh, sVl, at, ldx<XT>(a.v.p, vrow + d));
          put(sVh, sVl, at + half, ldx<XT>(a.v.p, vrow + d + half));
        }
      }
      __syncthreads();
      // scores of this warp's 16 keys
      float sc[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) sc[i][c] = 0.f;
#pragma unroll
      for (int ks = 0; ks < NS; ++ks) {
        uint32_t qh[4], ql[4], kh[4], kl[4];
        lda_rm(qh, sQh, LD, rt * 16, ks * 16);
        lda_rm(ql, sQl, LD, rt * 16, ks * 16);
        ldb_nk(kh, sKh, LD, wk * 16, ks * 16);
        ldb_nk(kl, sKl, LD, wk * 16, ks * 16);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          mma16816(sc[i], qh, kh[2 * i], kh[2 * i + 1]);
          mma16816(sc[i], qh, kl[2 * i], kl[2 * i + 1]);
          mma16816(sc[i], ql, kh[2 * i], kh[2 * i + 1]);
        }
      }
      float mx[2] = {m[0], m[1]};
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int rel = sRel[wk * 16 + i * 8 + 2 * j + (c & 1)], t = c < 2 ? ta : tb;
          sc[i][c] = rel <= t && rel > t - W ? sc[i][c] * scale : -INFINITY;
          mx[c >> 1] = fmaxf(mx[c >> 1], sc[i][c]);
        }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
        const float f = tc::ex2(m[h] - mx[h]);
        m[h] = mx[h];
        l[h] *= f;
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
          o[i][2 * h] *= f;
          o[i][2 * h + 1] *= f;
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          sc[i][c] = tc::ex2(sc[i][c] - m[c >> 1]);
          l[c >> 1] += sc[i][c];
        }
      uint32_t ph[4], pl[4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float x0 = sc[i][2 * h], x1 = sc[i][2 * h + 1];
          const uint32_t p = pack_bf16(x0, x1);
          ph[2 * i + h] = p;
          pl[2 * i + h] = pack_bf16(x0 - bf16_lo(p), x1 - bf16_hi(p));
        }
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        uint32_t vh[4], vl[4];
        ldb_kn(vh, sVh, LD, wk * 16, i * 16);
        ldb_kn(vl, sVl, LD, wk * 16, i * 16);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          mma16816(o[2 * i + u], ph, vh[2 * u], vh[2 * u + 1]);
          mma16816(o[2 * i + u], ph, vl[2 * u], vl[2 * u + 1]);
          mma16816(o[2 * i + u], pl, vh[2 * u], vh[2 * u + 1]);
        }
      }
    }
    __syncthreads();
    // merge the four key quarters and the sinks
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      if (j == 0) {
        sMax[(rt * 4 + wk) * 16 + g + 8 * h] = m[h];
        sSum[(rt * 4 + wk) * 16 + g + 8 * h] = l[h];
      }
#pragma unroll
      for (int i = 0; i < DP / 8; ++i)
        *reinterpret_cast<float2*>(sO + ((rt * 4 + wk) * 16 + g + 8 * h) * DP + i * 8 + 2 * j) =
            make_float2(o[i][2 * h], o[i][2 * h + 1]);
    }
    __syncthreads();
    for (int e = tid; e < 16 * RT * half; e += NT) {
      const int r = e / half, d = (e - r * half) * 2, row = r0 + r;
      if (row >= R) continue;
      const int q4 = (r >> 4) * 4, rr = r & 15;
      float mm = -1e30f;
#pragma unroll
      for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sMax[(q4 + w) * 16 + rr]);
      for (int i = 0; i < a.n_meta; ++i) mm = fmaxf(mm, a.meta[i] * kLog2e);
      float sum = 0.f, x = 0.f, y = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = tc::ex2(sMax[(q4 + w) * 16 + rr] - mm);
        const float2 v = *reinterpret_cast<const float2*>(sO + ((q4 + w) * 16 + rr) * DP + d);
        sum += f * sSum[(q4 + w) * 16 + rr];
        x += f * v.x;
        y += f * v.y;
      }
      for (int i = 0; i < a.n_meta; ++i) sum += tc::ex2(a.meta[i] * kLog2e - mm);
      const float inv = 1.f / sum;
      *reinterpret_cast<uint32_t*>(
          a.y + ((size_t)(b * a.H + hk * rep) * T + row) * D + d) = pack_bf16(x * inv, y * inv);
    }
  }
}

template <typename XT, int DP, int RT>
int launch_swa_block(const SwaBlockArgs& a, int grid, cudaStream_t st) {
  constexpr size_t smem = swa_block_smem(DP, RT);
  static bool done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (smem > 48 * 1024 && dev < 64 && !done[dev]) {
    cudaError_t e = cudaFuncSetAttribute(swa_block_kernel<XT, DP, RT>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) {
      set_error(std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
      return LZ_ERR_CUDA;
    }
    done[dev] = true;
  }
  swa_block_kernel<XT, DP, RT><<<grid, 128 * RT, smem, st>>>(a);
  count_launches(1);
  return check_launch("swa_block_kernel");
}

template <typename XT>
int pick_swa_block(const SwaBlockArgs& a, int grid, cudaStream_t st) {
  const bool one = a.H / a.Hkv * a.T <= 16;
#define LZ_SB(DP_) \
  return one ? launch_swa_block<XT, DP_, 1>(a, grid, st) : launch_swa_block<XT, DP_, 2>(a, grid, st)
  if (a.D <= 32) LZ_SB(32);
  if (a.D <= 64) LZ_SB(64);
  if (a.D <= 128) LZ_SB(128);
  LZ_SB(256);
#undef LZ_SB
}

}  // namespace
}  // namespace lz

extern "C" int lz_swa_decode_block(const void* q, const void* k, const void* v, int x_dtype,
                                   const long long* strides, const void* cos, const void* sin,
                                   int cs_dtype, long long cs_sb, const void* k_prev,
                                   const void* v_prev, const long long* strides_prev,
                                   const void* cos_prev, const void* sin_prev, long long cs_prev_sb,
                                   const int* count, float* k_ring, float* v_ring, const int* pos,
                                   const float* meta, int n_meta, void* y, int B, int H, int Hkv,
                                   int T, int T_prev, int window, int D, void* stream) {
  using namespace lz;
  clear_error();
  LZ_REQUIRE(B >= 1 && H >= 1 && Hkv >= 1 && D >= 2 && window >= 1 && T >= 0 && T_prev >= 0,
             LZ_ERR_INVALID_ARGUMENT, "sizes must be positive");
  LZ_REQUIRE(T + T_prev >= 1, LZ_ERR_INVALID_ARGUMENT, "no tokens: T and T_prev are both 0");
  LZ_REQUIRE(H % Hkv == 0, LZ_ERR_INVALID_ARGUMENT,
             "the key/value head count must divide the query head count");
  LZ_REQUIRE(D % 2 == 0, LZ_ERR_INVALID_ARGUMENT, "the rotated head dim must be even");
  LZ_REQUIRE(T <= kMaxBlock && T_prev <= kMaxBlock, LZ_ERR_UNSUPPORTED,
             "a block holds at most 64 tokens");
  LZ_REQUIRE(D <= 256 && window <= kMaxWindow, LZ_ERR_UNSUPPORTED,
             "decode supports D <= 256 and windows up to 1024");
  LZ_REQUIRE((long long)B * Hkv < (1ll << 31) && (long long)H / Hkv * T < (1ll << 30),
             LZ_ERR_UNSUPPORTED, "too many heads");
  LZ_REQUIRE(n_meta >= 0 && n_meta <= 32 && (n_meta == 0 || meta), LZ_ERR_INVALID_ARGUMENT,
             "meta must hold n_meta (<= 32) values");
  LZ_REQUIRE((x_dtype == LZ_DTYPE_F32 || x_dtype == LZ_DTYPE_BF16) &&
                 (cs_dtype == LZ_DTYPE_F32 || cs_dtype == LZ_DTYPE_BF16),
             LZ_ERR_INVALID_ARGUMENT, "dtypes must be LZ_DTYPE_F32 or LZ_DTYPE_BF16");
  LZ_REQUIRE(k_ring && v_ring && pos, LZ_ERR_INVALID_ARGUMENT, "null pointer");
  LZ_REQUIRE(!T || (q && k && v && strides && cos && sin && y), LZ_ERR_INVALID_ARGUMENT,
             "null pointer");
  LZ_REQUIRE(!T_prev || (k_prev && v_prev && strides_prev && cos_prev && sin_prev),
             LZ_ERR_INVALID_ARGUMENT, "null pointer in the previous block");
  LZ_REQUIRE(!T || (reinterpret_cast<uintptr_t>(y) & 3) == 0, LZ_ERR_INVALID_ARGUMENT,
             "y must be 4-byte aligned");
  SwaBlockArgs a = {};
  if (T) {
    a.q = {q, strides[0], strides[1], strides[2]};
    a.k = {k, strides[3], strides[4], strides[5]};
    a.v = {v, strides[6], strides[7], strides[8]};
  }
  if (T_prev) {
    a.kp = {k_prev, strides_prev[0], strides_prev[1], strides_prev[2]};
    a.vp = {v_prev, strides_prev[3], strides_prev[4], strides_prev[5]};
  }
  const int cb = cs_dtype == LZ_DTYPE_BF16;
  a.rot = {cos, sin, cs_sb, cb};
  a.rot_p = {cos_prev, sin_prev, cs_prev_sb, cb};
  a.pos = pos;
  a.count = count;
  a.meta = meta;
  a.kr = k_ring;
  a.vr = v_ring;
  a.y = static_cast<bf16*>(y);
  a.n_meta = n_meta;
  a.T = T;
  a.Tp = T_prev;
  a.H = H;
  a.Hkv = Hkv;
  a.W = window;
  a.D = D;
  auto st = static_cast<cudaStream_t>(stream);
  return x_dtype == LZ_DTYPE_F32 ? pick_swa_block<float>(a, B * Hkv, st)
                                 : pick_swa_block<bf16>(a, B * Hkv, st);
}
