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
// Two kernels. The first rotates: the accepted keys and their values go into the
// ring, the block's queries (split into bf16 hi + lo) and keys into a workspace, laid
// out as the second wants them in shared memory; a thread takes the same columns of
// all heads of a token, so cos and sin are read once. The second, launched under
// the first, attends: one CTA per (batch row, key/value head) for all rep T query
// rows of the group. Bound: 8 (W + T) D bytes of ring a head against 4 rep T (W + T) D
// operations: memory. Everything it reads arrives by TMA and bulk copies, the ring
// as it is, fp32 in 128-byte swizzled rows (of a long window, a part at a time).
// A warp takes a 16-row tile of queries over 16 keys at a time: it
// reads the keys as the B fragments of mma.sync m16n8k16, splits them into bf16 hi + lo
// in registers (hi hi + hi lo + lo hi keeps 2^-17 of a product, well under the bf16
// output) and keeps its own maximum and sum; the warps' outputs meet at the end,
// scaled to the common maximum, so a block of few rows keeps every warp busy. Nothing
// converted is written back to shared memory. (A warp on two row tiles converts a
// key once instead of twice, but its registers leave 16 warps an SM for 20, and
// the nine 16-key tiles of a window of 128 and its block do not divide over eight.)
// Measured, 128 sequences of 8 key / value heads of 64, window 128, 32 query heads, 8
// tokens: 47 us (85 MB, 1.8 TB/s). Nothing is full (issue 47 %, DRAM 25 %, tensor cores
// 16 %): a CTA waits for its ring, computes and merges, two an SM do not hide that, and 1024
// CTAs leave the fullest SM 8 for a mean of 6.9; a fifth of the instructions are the
// conversions. The ring in smaller parts (16, 32, 64 KB) or fewer warps a CTA (4 .. 8), so
// that more CTAs fit an SM, took 47 to 55 us where this took 48: a long window is cut at 64 KB.
//
// Fragments. Within a step of 16 columns thread j takes d = 4j .. 4j+3 (the
// queries are stored in that order), so a key is one 16-byte read; column tile i
// of 32 stands for d = 4n + i, so a value is one 16-byte read too. The keys of an
// 8-tile sit in rows 0 5 2 7 4 1 6 3: with the swizzle (16-byte chunk ^ row & 7)
// both reads are then free of bank conflicts.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "tc.cuh"

namespace lz {
extern std::atomic<int> g_withhold_block;  // gla_block.cu
namespace {

constexpr int kMaxBlock = 64;    // tokens a block
constexpr int kMaxWindow = 1024;  // as the single-token step
constexpr int kWarps = 10;        // most warps a CTA
constexpr int kSmem = 227 * 1024;  // shared memory that a CTA can have

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
  unsigned char* ws;  // SwaWork a (batch row, key/value head)
  int n_meta, T, Tp, H, Hkv, W, D;
  int rep;    // query heads a key/value head
  int part;   // ring rows in shared memory at a time, a multiple of 16
  int tma;    // the rings can be read by TMA
  int withhold;  // a test: the first keys are not loaded
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
// N (1 or 2) neighbouring values.
template <typename XT, int N>
__device__ __forceinline__ float2 ldn(const XT* p) {
  if constexpr (N == 1) {
    return make_float2(ldx<XT>(p, 0), 0.f);
  } else if constexpr (sizeof(XT) == 4) {
    return *reinterpret_cast<const float2*>(p);
  } else {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
    return make_float2(bf16_lo(w), bf16_hi(w));
  }
}
// cos and sin at columns d .. d + N - 1 and the same plus D / 2 of one token.
struct Angle {
  float2 c1, c2, s1, s2;
};
template <int N>
__device__ __forceinline__ Angle angle(const Rotary& r, long long at, int half) {
  if (r.bf16_) {
    const bf16 *c = static_cast<const bf16*>(r.cos) + at, *s = static_cast<const bf16*>(r.sin) + at;
    return {ldn<bf16, N>(c), ldn<bf16, N>(c + half), ldn<bf16, N>(s), ldn<bf16, N>(s + half)};
  }
  const float *c = static_cast<const float*>(r.cos) + at, *s = static_cast<const float*>(r.sin) + at;
  return {ldn<float, N>(c), ldn<float, N>(c + half), ldn<float, N>(s), ldn<float, N>(s + half)};
}
// The rotated columns of a row's x1 (d ..) and x2 (d + D / 2 ..), each product and
// sum rounded once, as the single-token step rounds them.
__device__ __forceinline__ void rotate(float2& x1, float2& x2, const Angle& a) {
  const float2 y1 = x1, y2 = x2;
  x1.x = __fadd_rn(__fmul_rn(y1.x, a.c1.x), -__fmul_rn(y2.x, a.s1.x));
  x1.y = __fadd_rn(__fmul_rn(y1.y, a.c1.y), -__fmul_rn(y2.y, a.s1.y));
  x2.x = __fadd_rn(__fmul_rn(y2.x, a.c2.x), __fmul_rn(y1.x, a.s2.x));
  x2.y = __fadd_rn(__fmul_rn(y2.y, a.c2.y), __fmul_rn(y1.y, a.s2.y));
}

// The place of column d of row r in a tile of DP / 32 boxes of `rows` swizzled
// 128-byte rows each, in floats.
__device__ __forceinline__ int spot(int rows, int r, int d) {
  return ((d >> 5) * rows + r) * 32 + ((((d >> 2) & 7) ^ (r & 7)) << 2) + (d & 3);
}
// The place of query column d in its row: thread j's four columns of a step are
// the mma's k slots 2j, 2j + 1, 2j + 8, 2j + 9.
__device__ __forceinline__ int slot_of(int d) {
  return (d & ~15) + ((d >> 2) & 3) * 2 + (d & 1) + ((d >> 1) & 1) * 8;
}
// The row of an 8-tile that holds key n of the mma.
__device__ __forceinline__ int key_row(int n) { return n ^ ((n & 1) << 2); }

__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = pack_bf16(x, y);
  lo = pack_bf16(x - bf16_lo(hi), y - bf16_hi(hi));
}
// N columns to their places (neighbours stay neighbours).
template <int N>
__device__ __forceinline__ void put(float* p, float2 x) {
  if constexpr (N == 2)
    *reinterpret_cast<float2*>(p) = x;
  else
    *p = x.x;
}
template <int N>
__device__ __forceinline__ void put_split(bf16* hi, bf16* lo, int at, float2 x) {
  uint32_t h, l;
  split2(x.x, x.y, h, l);
  if constexpr (N == 2) {
    *reinterpret_cast<uint32_t*>(hi + at) = h;
    *reinterpret_cast<uint32_t*>(lo + at) = l;
  } else {
    hi[at] = __ushort_as_bfloat16((unsigned short)h);
    lo[at] = __ushort_as_bfloat16((unsigned short)l);
  }
}

// Workspace of a (batch row, key/value head), in bytes: queries hi and lo, a pass of
// 16 QT rows after another ([hi | lo][16 QT][DP + 8]), then the new keys and values
// ([DP / 32 boxes][T rounded up to 16][32], swizzled).
struct SwaWork {
  int q, k, v, total;
};
__host__ __device__ inline SwaWork swa_work(int DP, int QT, int R, int T) {
  const int passes = (R + 16 * QT - 1) / (16 * QT), rows = (T + 15) & ~15;
  SwaWork w;
  w.q = 0;
  w.k = passes * 2 * 16 * QT * (DP + 8) * 2;
  w.v = w.k + rows * DP * 4;
  w.total = w.v + rows * DP * 4;
  return w;
}

// The first kernel. blockIdx = (256 threads over (token, columns), key/value head,
// batch row); tokens 0 .. T are the block's, the rest the pending ones. Rows beyond
// the last token or query stay as they are: the second kernel masks such keys, zeroes
// such values and writes no such output. N: columns a thread takes (2 where alignment
// allows).
template <typename XT, int DP, int QT, int N>
__global__ void __launch_bounds__(256) swa_rotate_kernel(const SwaBlockArgs a) {
  constexpr int LQ = DP + 8, RQ = 16 * QT, PER = DP / 2 / N;  // threads a token
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  const int i = blockIdx.x * 256 + threadIdx.x, row = i / PER, d = i % PER * N;
  const int b = blockIdx.z, hk = blockIdx.y, T = a.T, D = a.D, half = D / 2;
  const int TN = (T + 15) & ~15, rep = a.rep, R = rep * T;
  if (row < T) {
    const SwaWork o = swa_work(DP, QT, R, T);
    unsigned char* ws = a.ws + (size_t)(b * a.Hkv + hk) * o.total;
    float* wk = reinterpret_cast<float*>(ws + o.k);
    float* wv = reinterpret_cast<float*>(ws + o.v);
    const int t = row;
    const bool in = d < half;
    const XT* kp = static_cast<const XT*>(a.k.p) + b * a.k.sb + hk * a.k.sh + t * a.k.st + d;
    const XT* vp = static_cast<const XT*>(a.v.p) + b * a.v.sb + hk * a.v.sh + t * a.v.st + d;
    const XT* qp = static_cast<const XT*>(a.q.p) + b * a.q.sb + hk * rep * a.q.sh + t * a.q.st + d;
    // columns d .. and half + d .. of the rotation; beyond D, the zeros of the padding
    const int e1 = d < half ? d : 2 * d, e2 = d < half ? d + half : 2 * d + N;
    Angle ang = {};
    float2 x1 = {}, x2 = {}, v1 = {}, v2 = {};
    if (in) {
      ang = angle<N>(a.rot, b * a.rot.sb + (long long)t * D + d, half);
      x1 = ldn<XT, N>(kp), x2 = ldn<XT, N>(kp + half);
      v1 = ldn<XT, N>(vp), v2 = ldn<XT, N>(vp + half);
      rotate(x1, x2, ang);
    }
    put<N>(wk + spot(TN, t, e1), x1);
    put<N>(wk + spot(TN, t, e2), x2);
    put<N>(wv + spot(TN, t, e1), v1);
    put<N>(wv + spot(TN, t, e2), v2);
    const int c1 = slot_of(e1), c2 = slot_of(e2);
#pragma unroll 4
    for (int h = 0; h < rep; ++h) {
      float2 q1 = {}, q2 = {};
      if (in) {
        q1 = ldn<XT, N>(qp + h * a.q.sh), q2 = ldn<XT, N>(qp + h * a.q.sh + half);
        rotate(q1, q2, ang);
      }
      const int r = h * T + t;
      bf16* hi = reinterpret_cast<bf16*>(ws) + (r / RQ) * (2 * RQ * LQ) + (r % RQ) * LQ;
      put_split<N>(hi, hi + RQ * LQ, c1, q1);
      put_split<N>(hi, hi + RQ * LQ, c2, q2);
    }
  } else if (row < T + a.Tp && d < half) {
    const int t = row - T, W = a.W;
    const int n = a.count ? min(max(a.count[b], 0), a.Tp) : a.Tp;
    if (t >= n || t < n - W) return;  // of more accepted tokens than the window, the last W
    const XT* kp = static_cast<const XT*>(a.kp.p) + b * a.kp.sb + hk * a.kp.sh + t * a.kp.st + d;
    const XT* vp = static_cast<const XT*>(a.vp.p) + b * a.vp.sb + hk * a.vp.sh + t * a.vp.st + d;
    float2 x1 = ldn<XT, N>(kp), x2 = ldn<XT, N>(kp + half);
    rotate(x1, x2, angle<N>(a.rot_p, b * a.rot_p.sb + (long long)t * D + d, half));
    const int slot = (max(a.pos[b], 0) % W + t) % W;
    const size_t at = ((size_t)(b * a.Hkv + hk) * W + slot) * D + d;
    put<N>(a.kr + at, x1);
    put<N>(a.kr + at + half, x2);
    put<N>(a.vr + at, ldn<XT, N>(vp));
    put<N>(a.vr + at + half, ldn<XT, N>(vp + half));
  }
}

// Shared memory of the second kernel, in bytes from the 1024-aligned start.
struct SwaSmem {
  int k = 0, v = 0, nk = 0, nv = 0, q = 0, stat = 0, bar = 0, total = 0;
};
__host__ __device__ constexpr SwaSmem swa_smem(int DP, int QT, int part, int T, int warps) {
  SwaSmem s;
  const int new_rows = (T + 15) & ~15;
  int n = 0;
  s.k = n, n += part * DP * 4;
  s.v = n, n += part * DP * 4;
  s.nk = n, n += new_rows * DP * 4;
  s.nv = n, n += new_rows * DP * 4;
  const int merge = warps * 16 * (DP + 4) * 4;  // the warps' outputs, over the keys
  if (n < merge) n = (merge + 1023) & ~1023;
  s.q = n, n += 2 * 16 * QT * (DP + 8) * 2;
  s.stat = n, n += 3 * warps * 16 * 4;
  s.bar = n, n += 8;
  s.total = n + 1024;
  return s;
}

// Four outputs by themselves, from the keys that their row sees only. The tensor cores
// give masked values a weight of zero, and 0 * inf and 0 * NaN are NaN: where that may
// have happened (an output is NaN), a thread comes here. q: the row's queries, hi, with
// lo after `lo`; kr, vr: the ring, `nr` of its W rows in use, the newest in slot `last`;
// nk, nv: the block's keys and values in swizzled tiles of TN rows.
__device__ __noinline__ float4 alone(const bf16* q, int lo, const float* kr, const float* vr,
                                     int nr, int last, int W, const float* nk, const float* nv,
                                     int TN, int t, int D, int d, const float* meta, int n_meta) {
  const float scale = rsqrtf((float)D) * kLog2e;
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < n_meta; ++i) m = fmaxf(m, meta[i] * kLog2e);
  for (int i = 0; i < n_meta; ++i)  // (sinks of -inf only: m is -inf too, and they weigh nothing)
    if (meta[i] != -INFINITY) l += tc::ex2(meta[i] * kLog2e - m);
  for (int i = 0; i < nr + t + 1 && l == l; ++i) {
    const bool own = i >= nr;
    const int back = last - i, k = own ? i - nr : i;
    const int rel = own ? k : -1 - (back < 0 ? back + W : back);
    if (rel <= t - W) continue;
    float s = 0.f;
    for (int e = 0; e < D; ++e) {
      const int at = slot_of(e);
      s = fmaf(__bfloat162float(q[at]) + __bfloat162float(q[lo + at]),
               own ? nk[spot(TN, k, e)] : kr[(size_t)k * D + e], s);
    }
    s *= scale;
    if (s == -INFINITY) continue;
    const float mx = fmaxf(m, s), f = m > -INFINITY ? tc::ex2(m - mx) : 0.f, x = tc::ex2(s - mx);
    m = mx;
    l = l * f + x;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int at = d + c < D ? d + c : d;
      o[c] = o[c] * f + x * (own ? nv[spot(TN, k, at)] : vr[(size_t)k * D + at]);
    }
  }
  return make_float4(o[0] / l, o[1] / l, o[2] / l, o[3] / l);
}

// DP: D padded to whole 32s. QT: 16-row tiles of queries at once, one a warp.
template <int DP, int QT>
__global__ void __launch_bounds__(32 * kWarps, DP <= 64 ? 2 : 1)
swa_block_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                 const SwaBlockArgs a) {
  constexpr int LQ = DP + 8, NS = DP / 16, NG = DP / 32, LO = DP + 4, RQ = 16 * QT;
  extern __shared__ unsigned char raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5, nw = nt >> 5;
  const int g = lane >> 2, j = lane & 3;
  const int T = a.T, W = a.W, D = a.D, part = a.part;
  const int TN = (T + 15) & ~15;  // rows of the new tokens' tile
  const SwaSmem o = swa_smem(DP, QT, part, T, nw);
  float* sK = reinterpret_cast<float*>(sm + o.k);
  float* sV = reinterpret_cast<float*>(sm + o.v);
  float* sNK = reinterpret_cast<float*>(sm + o.nk);
  float* sNV = reinterpret_cast<float*>(sm + o.nv);
  float* sO = reinterpret_cast<float*>(sm);             // [warp][16][LO], after the last key
  bf16* sQh = reinterpret_cast<bf16*>(sm + o.q);        // [hi | lo][RQ][LQ]
  float* sMax = reinterpret_cast<float*>(sm + o.stat);  // [warp][16]
  float* sSum = sMax + nw * 16;
  float* sCof = sSum + nw * 16;
  uint64_t* bar = reinterpret_cast<uint64_t*>(sm + o.bar);
  const int pass = blockIdx.x, b = blockIdx.y, hk = blockIdx.z, bk = b * a.Hkv + hk;
  const int rep = a.rep, R = rep * T, r0 = pass * RQ;
  const float* kring = a.kr + (size_t)bk * W * D;
  const float* vring = a.vr + (size_t)bk * W * D;
  const int parts = (W + part - 1) / part;
  const SwaWork wo = swa_work(DP, QT, R, T);
  const unsigned char* ws = a.ws + (size_t)bk * wo.total;
  constexpr int kQBytes = 2 * RQ * LQ * 2;
  uint32_t phase = 0;
  bool live = true;  // after a timeout (of any thread) nothing is written

  // ring rows [p part, (p + 1) part) into sK / sV; with the first part, the queries and
  // the new keys and values
  const auto load = [&](int p) {
    if (tid == 0 && (a.tma || !p) && live) {  // (a phase that has not ended takes no other load)
      const int nb = TN * DP * 4;
      tc::mbar_expect_tx(bar, (a.tma ? 2 * part * DP * 4 : 0) + (p ? 0 : kQBytes + 2 * nb));
      if (a.tma) {
#pragma unroll
        for (int i = 0; i < NG; ++i) {  // rows and columns beyond the ring arrive as zeros
          if (i || p || !a.withhold)
            tc::tma_load_3d(sK + i * part * 32, &tk, 32 * i, p * part, bk, bar);
          tc::tma_load_3d(sV + i * part * 32, &tv, 32 * i, p * part, bk, bar);
        }
      }
      if (!p) {
        tc::bulk_load(sQh, ws + wo.q + pass * kQBytes, kQBytes, bar);
        tc::bulk_load(sNK, ws + wo.k, nb, bar);
        tc::bulk_load(sNV, ws + wo.v, nb, bar);
      }
    }
    if (!a.tma)
      for (int e = tid; e < part * DP; e += nt) {
        const int r = e / DP, d = e - r * DP, slot = p * part + r;
        const bool in = slot < W && d < D;
        sK[spot(part, r, d)] = in ? kring[(size_t)slot * D + d] : 0.f;
        sV[spot(part, r, d)] = in ? vring[(size_t)slot * D + d] : 0.f;
      }
  };
  const int pos = max(a.pos[b], 0);
  const int n = a.Tp ? (a.count ? min(max(a.count[b], 0), a.Tp) : a.Tp) : 0;
  if (tid == 0) {
    tc::mbar_init(bar, 1);
    tc::fence_mbar_init();
    tc::prefetch_tmap(&tk);
    tc::prefetch_tmap(&tv);
  }
  // the sinks of lane16 and lane16 + 16, in the exponent's base
  const int lane16 = tid & 15;
  const float sink0 = lane16 < a.n_meta ? a.meta[lane16] * kLog2e : -INFINITY;
  const float sink1 = lane16 + 16 < a.n_meta ? a.meta[lane16 + 16] * kLog2e : -INFINITY;
  asm volatile("griddepcontrol.wait;\n" ::: "memory");  // the ring and the workspace are written
  if (tid == 0) asm volatile("fence.proxy.async;\n" ::: "memory");
  load(0);
  __syncthreads();  // the barrier is initialised

  const int nr = (int)min((long long)pos + n, (long long)W);  // ring rows that hold a token
  const int last = (pos % W + n - 1 + W) % W;                 // slot of the newest (W >= 1)
  const float scale = rsqrtf((float)D) * kLog2e;
  const int krow = key_row(g), vrow0 = key_row(2 * j), vrow1 = key_row(2 * j + 1);
  const int eight = 8 % T;
  const int rt = QT == 1 ? 0 : warp % QT;                     // this warp's row tile
  const int kw = QT == 1 ? warp : warp / QT, kws = nw / QT;   // and its turn among the keys
  // ldmatrix rows of this lane's queries, hi and lo
  const uint32_t aqh = smem_u32(sQh) + (rt * 16 + (lane & 15)) * (LQ * 2) + (lane >> 4) * 16;
  const uint32_t aql = aqh + RQ * LQ * 2;

  float m[2] = {-1e30f, -1e30f}, l[2] = {0.f, 0.f}, acc[4 * NG][4];
#pragma unroll
  for (int i = 0; i < 4 * NG; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[i][c] = 0.f;
  int tq[2];  // the tokens of this thread's rows
  tq[0] = (r0 + rt * 16 + g) % T;
  tq[1] = tq[0] + eight;
  if (tq[1] >= T) tq[1] -= T;

  for (int p = 0; p < parts; ++p) {
    if (p) {
      tc::fence_proxy_async_smem();
      __syncthreads();  // the part before has been used
      load(p);
    }
    if (a.tma || !p) {
      if (tc::mbar_wait(bar, phase, 96))
        phase ^= 1;
      else
        live = false;
    }
    if (!a.tma) __syncthreads();
    const int held = min(max(nr - p * part, 0), part);  // rows of this part that hold a token
    const int ring_tiles = (held + 15) >> 4;
    const int tiles = ring_tiles + (p + 1 == parts ? TN >> 4 : 0);
    for (int tl = kw; tl < tiles; tl += kws) {
      const bool own = tl >= ring_tiles;
      const int rows = own ? TN : part, row0 = (own ? tl - ring_tiles : tl) * 16;
      const int lim = own ? T : held;  // rows beyond hold nothing (perhaps not numbers)
      // this lane's places: key row krow, value rows of keys 2j and 2j + 1 (8 rows on
      // and 16 columns on keep the swizzle's row and flip one bit of its chunk)
      const float* kg = (own ? sNK : sK) + (row0 + krow) * 32;
      const float *k0 = kg + ((j ^ krow) << 2), *k1 = kg + (((4 + j) ^ krow) << 2);
      const float* vt = own ? sNV : sV;
      const float* v0 = vt + (row0 + vrow0) * 32 + ((g ^ vrow0) << 2);
      const float* v1 = vt + (row0 + vrow1) * 32 + ((g ^ vrow1) << 2);
      // scores of 16 keys: hi hi, and the cross products in sums of their own (the
      // chain of dependent products is what a warp waits for here)
      float sc[2][4], sx[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) sc[i][c] = sx[i][c] = 0.f;
#pragma unroll
      for (int ks = 0; ks < NS; ++ks) {
        uint32_t qh[4], ql[4];
        ldsm_x4(qh, aqh + ks * 32);
        ldsm_x4(ql, aql + ks * 32);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float4 x = *reinterpret_cast<const float4*>((ks & 1 ? k1 : k0) + 256 * i);
          uint32_t kh[2], kl[2];
          split2(x.x, x.y, kh[0], kl[0]);
          split2(x.z, x.w, kh[1], kl[1]);
          mma16816(sc[i], qh, kh[0], kh[1]);
          mma16816(sx[i], qh, kl[0], kl[1]);
          mma16816(sx[i], ql, kh[0], kh[1]);
        }
        if (ks & 1) k0 += rows * 32, k1 += rows * 32;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) sc[i][c] += sx[i][c];
      // position - base of this thread's keys 8 i + 2 j + c; a ring slot holds the
      // last position before base that falls on it
      int rel[4];
      bool clear = true;  // every row of the tile sees every key
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = row0 + (i >> 1) * 8 + (i & 1 ? vrow1 : vrow0);
        const int back = last - (p * part + k);
        rel[i] = own ? k : -1 - (back < 0 ? back + W : back);
        if (k >= lim) rel[i] = 1 << 30;
        clear = clear && rel[i] < 0 && rel[i] >= T - W;
      }
      if (!__all_sync(0xffffffffu, clear)) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (rel[i] > tq[h] || rel[i] <= tq[h] - W) sc[i >> 1][2 * h + (i & 1)] = -INFINITY;
      }
      uint32_t ph[4], pl[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float mx = fmaxf(fmaxf(sc[0][2 * h], sc[0][2 * h + 1]),
                         fmaxf(sc[1][2 * h], sc[1][2 * h + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        mx = fmaxf(mx * scale, m[h]);
        if (tl != kw || p) {  // not the first keys: rescale
          const float f = tc::ex2(m[h] - mx);
          l[h] *= f;
#pragma unroll
          for (int i = 0; i < 4 * NG; ++i) {
            acc[i][2 * h] *= f;
            acc[i][2 * h + 1] *= f;
          }
        }
        m[h] = mx;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float x0 = tc::ex2(fmaf(sc[i][2 * h], scale, -mx));
          const float x1 = tc::ex2(fmaf(sc[i][2 * h + 1], scale, -mx));
          l[h] += x0 + x1;
          split2(x0, x1, ph[2 * i + h], pl[2 * i + h]);
        }
      }
      // values: rows of keys 2j, 2j + 1, 2j + 8, 2j + 9, columns 4 g .. 4 g + 3 of each 32
#pragma unroll
      for (int q = 0; q < NG; ++q) {
        float4 x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          x[u] = *reinterpret_cast<const float4*>((u & 1 ? v1 : v0) + 256 * (u >> 1));
        v0 += rows * 32, v1 += rows * 32;
        if (row0 + 16 > lim) {
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (row0 + (u & 1 ? vrow1 : vrow0) + (u >> 1) * 8 >= lim)
              x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t vh[2], vl[2];
#pragma unroll
          for (int u = 0; u < 2; ++u)
            split2(reinterpret_cast<const float*>(&x[2 * u])[i],
                   reinterpret_cast<const float*>(&x[2 * u + 1])[i], vh[u], vl[u]);
          mma16816(acc[4 * q + i], ph, vh[0], vh[1]);
          mma16816(acc[4 * q + i], ph, vl[0], vl[1]);
          mma16816(acc[4 * q + i], pl, vh[0], vh[1]);
        }
      }
    }
  }
  // the warps meet: a coefficient for each warp's row, from the common maximum and
  // sum and the sinks, then the outputs times it, written over the keys and added
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    if (j == 0) {
      sMax[warp * 16 + g + 8 * h] = m[h];
      sSum[warp * 16 + g + 8 * h] = l[h];
    }
  }
  live = __syncthreads_and(live);
  for (int e = tid >> 4; e < RQ; e += nt >> 4) {  // a row a half warp, a lane a warp of its tile
    const int w = (lane16 * QT + (e >> 4)), at = w * 16 + (e & 15);
    const bool in = lane16 < kws;
    const float mw = in ? sMax[at] : -1e30f;
    float top = fmaxf(mw, fmaxf(sink0, sink1));
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    const float f = tc::ex2(mw - top);
    float sum = (in ? f * sSum[at] : 0.f) + tc::ex2(sink0 - top) + tc::ex2(sink1 - top);
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    if (in) sCof[at] = f / sum;
  }
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float f = sCof[warp * 16 + g + 8 * h];
    float* row = sO + (warp * 16 + g + 8 * h) * LO + 8 * j;
#pragma unroll
    for (int q = 0; q < NG; ++q)
#pragma unroll
      for (int u = 0; u < 2; ++u)  // columns 8 j + 4 u + (0 .. 3)
        *reinterpret_cast<float4*>(row + 32 * q + 4 * u) =
            make_float4(f * acc[4 * q][2 * h + u], f * acc[4 * q + 1][2 * h + u],
                        f * acc[4 * q + 2][2 * h + u], f * acc[4 * q + 3][2 * h + u]);
  }
  __syncthreads();
  for (int e = tid; e < RQ * (DP / 4); e += nt) {
    const int r = e / (DP / 4), d = (e - r * (DP / 4)) * 4, row = r0 + r;
    if (row >= R || d >= D || !live) continue;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = 0; w < kws; ++w) {
      const float4 v = *reinterpret_cast<const float4*>(
          sO + ((w * QT + (r >> 4)) * 16 + (r & 15)) * LO + d);
      x.x += v.x;
      x.y += v.y;
      x.z += v.z;
      x.w += v.w;
    }
    const float any = x.x + x.y + x.z + x.w;
    if (any != any)
      x = alone(reinterpret_cast<const bf16*>(ws + wo.q + pass * kQBytes) + r * LQ, RQ * LQ,
                kring, vring, nr, last, W, reinterpret_cast<const float*>(ws + wo.k),
                reinterpret_cast<const float*>(ws + wo.v), TN, row % T, D, d, a.meta, a.n_meta);
    bf16* yr = a.y + ((size_t)(b * a.H + hk * rep) * T + row) * D + d;  // D is even
    *reinterpret_cast<uint32_t*>(yr) = pack_bf16(x.x, x.y);
    if (d + 2 < D) *reinterpret_cast<uint32_t*>(yr + 2) = pack_bf16(x.z, x.w);
  }
  if (tid == 0 && !live) tc::mbar_wait(bar, phase, 96);  // a late load is not left on its way
}

int ring_map(CUtensorMap* m, const float* p, const SwaBlockArgs& a, int heads) {
  auto fn = tc::encode_tiled_fn();
  if (!fn) {
    set_error("lz_swa_decode_block: cuTensorMapEncodeTiled is not available");
    return LZ_ERR_CUDA;
  }
  const cuuint64_t dims[3] = {(cuuint64_t)a.D, (cuuint64_t)a.W, (cuuint64_t)heads};
  const cuuint64_t strides[2] = {(cuuint64_t)a.D * 4, (cuuint64_t)a.W * a.D * 4};
  const cuuint32_t box[3] = {32, (cuuint32_t)a.part, 1}, es[3] = {1, 1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<float*>(p), dims,
                        strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("lz_swa_decode_block: the tensor map of a ring could not be encoded, driver code " +
              std::to_string((int)r));
    return LZ_ERR_CUDA;
  }
  return LZ_OK;
}

// As many warps as there are 16-key tiles (of a part of the ring and the block) for each
// row tile, in as few equal turns as fit.
int block_warps(int QT, int part, int T) {
  const int tiles = part / 16 + ((T + 15) >> 4), turns = ceil_div(tiles, kWarps / QT);
  return QT * std::max(ceil_div(tiles, turns), 4 / QT);
}

// Ring rows in shared memory at a time: 64 KB of keys and values at most, and less where a
// long block of wide heads (D > 128, T > 48) leaves no room for that.
int ring_part(int W, int DP, int QT, int T) {
  int part = std::min((W + 15) & ~15, 64 * 1024 / (DP * 8));
  while (part > 16 && swa_smem(DP, QT, part, T, block_warps(QT, part, T)).total > kSmem) part -= 16;
  return part;
}

// A failed call as this library's error (and no longer the runtime's: a later call would
// report it as its own).
int failed(cudaError_t e, const char* what) {
  set_error(std::string(what) + ": " + cudaGetErrorString(e));
  cudaGetLastError();
  return LZ_ERR_CUDA;
}
int launched(cudaError_t e, const char* what) {
  if (e != cudaSuccess) return failed(e, what);
  count_launches(1);
  return check_launch(what);
}

// What can be refused of the attention's launch: before the rotation writes the ring.
template <int DP, int QT>
int prepare_attend(SwaBlockArgs& a, CUtensorMap& tk, CUtensorMap& tv, int B) {
  static_assert(swa_smem(DP, QT, 16, kMaxBlock, kWarps).total <= kSmem, "every block fits");
  a.part = ring_part(a.W, DP, QT, a.T);
  a.tma = a.D % 4 == 0 && aligned16(a.kr) && aligned16(a.vr);
  if (a.tma) {
    int rc = ring_map(&tk, a.kr, a, B * a.Hkv);
    if (!rc) rc = ring_map(&tv, a.vr, a, B * a.Hkv);
    if (rc) return rc;
  }
  static bool done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 64 && !done[dev]) {
    const int most = swa_smem(DP, QT, 64 * 1024 / (DP * 8), kMaxBlock, kWarps).total;
    cudaError_t e = cudaFuncSetAttribute(swa_block_kernel<DP, QT>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         std::min(most, kSmem));
    if (e != cudaSuccess) return failed(e, "cudaFuncSetAttribute");
    done[dev] = true;
  }
  return LZ_OK;
}

template <int DP, int QT>
int launch_attend(const SwaBlockArgs& a, const CUtensorMap& tk, const CUtensorMap& tv, int B,
                  cudaStream_t st) {
  const int warps = block_warps(QT, a.part, a.T);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ceil_div(a.rep * a.T, 16 * QT), B, a.Hkv);
  cfg.blockDim = dim3(32 * warps);
  cfg.dynamicSmemBytes = swa_smem(DP, QT, a.part, a.T, warps).total;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return launched(cudaLaunchKernelEx(&cfg, swa_block_kernel<DP, QT>, tk, tv, a),
                  "swa_block_kernel");
}

template <typename XT, int DP, int QT>
int launch_swa_block(SwaBlockArgs& a, bool pairs, int B, cudaStream_t st) {
  CUtensorMap tk = {}, tv = {};
  int rc = a.T ? prepare_attend<DP, QT>(a, tk, tv, B) : LZ_OK;
  if (rc) return rc;
  const int rows = a.T + a.Tp, per = DP / 2 / (pairs ? 2 : 1);
  const dim3 grid(ceil_div(rows * per, 256), a.Hkv, B);
  if (pairs)
    swa_rotate_kernel<XT, DP, QT, 2><<<grid, 256, 0, st>>>(a);
  else
    swa_rotate_kernel<XT, DP, QT, 1><<<grid, 256, 0, st>>>(a);
  rc = launched(cudaSuccess, "swa_rotate_kernel");
  if (!rc && a.T) rc = launch_attend<DP, QT>(a, tk, tv, B, st);
  return rc;
}

int padded(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 128 ? 128 : 256; }
int row_tiles(int R) { return R <= 16 ? 1 : 2; }

template <typename XT>
int pick_swa_block(SwaBlockArgs& a, bool pairs, int B, cudaStream_t st) {
  const bool one = row_tiles(a.rep * a.T) == 1;
#define LZ_SB(DP_)                                              \
  return one ? launch_swa_block<XT, DP_, 1>(a, pairs, B, st)    \
             : launch_swa_block<XT, DP_, 2>(a, pairs, B, st)
  switch (padded(a.D)) {
    case 32:
      LZ_SB(32);
    case 64:
      LZ_SB(64);
    case 128:
      LZ_SB(128);
    default:
      LZ_SB(256);
  }
#undef LZ_SB
}

size_t swa_bytes(int B, int H, int Hkv, int T, int D) {
  if (!T) return 0;
  const int R = H / Hkv * T;
  return (size_t)B * Hkv * swa_work(padded(D), row_tiles(R), R, T).total;
}

}  // namespace
int swa_block_timeout_flag(unsigned int* out) { return tc::read_timeout_flag_here(out); }
int swa_block_timeout_clear() { return tc::clear_timeout_flag_here(); }
}  // namespace lz

extern "C" size_t lz_swa_decode_block_workspace_bytes(int B, int H, int Hkv, int T, int D) {
  if (B < 1 || H < 1 || Hkv < 1 || H % Hkv || T < 0 || T > lz::kMaxBlock || D < 2 || D > 256)
    return 0;
  return lz::swa_bytes(B, H, Hkv, T, D);
}

extern "C" int lz_swa_decode_block(const void* q, const void* k, const void* v, int x_dtype,
                                   const long long* strides, const void* cos, const void* sin,
                                   int cs_dtype, long long cs_sb, const void* k_prev,
                                   const void* v_prev, const long long* strides_prev,
                                   const void* cos_prev, const void* sin_prev, long long cs_prev_sb,
                                   const int* count, float* k_ring, float* v_ring, const int* pos,
                                   const float* meta, int n_meta, void* y, void* workspace,
                                   size_t workspace_bytes, int B, int H, int Hkv, int T,
                                   int T_prev, int window, int D, void* stream) {
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
  LZ_REQUIRE(B <= 65535 && Hkv <= 65535 && (long long)H / Hkv * T < (1ll << 20),
             LZ_ERR_UNSUPPORTED, "too many sequences or heads");
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
  LZ_REQUIRE(!T || (workspace && workspace_bytes >= swa_bytes(B, H, Hkv, T, D)), LZ_ERR_WORKSPACE,
             "workspace too small, see lz_swa_decode_block_workspace_bytes");
  LZ_REQUIRE(!T || aligned16(workspace), LZ_ERR_INVALID_ARGUMENT,
             "workspace must be 16-byte aligned");
  SwaBlockArgs a = {};
  a.ws = static_cast<unsigned char*>(workspace);
  if (T) {
    a.q = {q, strides[0], strides[1], strides[2]};
    a.k = {k, strides[4], strides[5], strides[6]};
    a.v = {v, strides[8], strides[9], strides[10]};
    LZ_REQUIRE(strides[3] == 1 && strides[7] == 1 && strides[11] == 1, LZ_ERR_INVALID_ARGUMENT,
               "the last dimension must be contiguous");
  }
  if (T_prev) {
    a.kp = {k_prev, strides_prev[0], strides_prev[1], strides_prev[2]};
    a.vp = {v_prev, strides_prev[4], strides_prev[5], strides_prev[6]};
    LZ_REQUIRE(strides_prev[3] == 1 && strides_prev[7] == 1, LZ_ERR_INVALID_ARGUMENT,
               "the last dimension must be contiguous");
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
  a.rep = H / Hkv;
  a.withhold = g_withhold_block.load(std::memory_order_relaxed);
  // two columns at a time: even strides and halves, bases on two elements
  const size_t xs = 2 * (x_dtype == LZ_DTYPE_BF16 ? 2 : 4), cs2 = 2 * (cb ? 2 : 4);
  const auto even = [](const Heads& h, size_t to) {
    return reinterpret_cast<uintptr_t>(h.p) % to == 0 && ((h.sb | h.sh | h.st) & 1) == 0;
  };
  const auto even_r = [&](const Rotary& r) {
    return (reinterpret_cast<uintptr_t>(r.cos) | reinterpret_cast<uintptr_t>(r.sin)) % cs2 == 0 &&
           (r.sb & 1) == 0;
  };
  const bool pairs =
      D % 4 == 0 &&
            ((reinterpret_cast<uintptr_t>(k_ring) | reinterpret_cast<uintptr_t>(v_ring)) & 7) == 0 &&
            even(a.q, xs) && even(a.k, xs) && even(a.v, xs) && even(a.kp, xs) &&
            even(a.vp, xs) && even_r(a.rot) && even_r(a.rot_p);
  auto st = static_cast<cudaStream_t>(stream);
  return x_dtype == LZ_DTYPE_F32 ? pick_swa_block<float>(a, pairs, B, st)
                                 : pick_swa_block<bf16>(a, pairs, B, st);
}
