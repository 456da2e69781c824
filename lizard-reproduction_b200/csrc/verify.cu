// Verification of drafted tokens against the target's probabilities.
//
// For one sequence with drafted tokens x_0 .. x_{n-1}, p_i = softmax(target
// logits i / T) and q_i = softmax(draft logits i / T): token i is accepted while
// u_i q_i(x_i) < p_i(x_i). After the first refusal, at a, the next token is drawn
// from max(p_a - q_a, 0), after n acceptances from p_n; a draw from weights r is
// argmax_j r_j / e_j with the given e_j ~ Exp(1) (an exponential race: the
// winner's law is r / sum r, so the residual needs no normalising sum, no prefix
// sum and no order of additions, and ties go to the lowest index). The emitted
// tokens then follow p exactly. T < 1e-5 is the greedy limit: a drafted token has
// to be the target's argmax, and the next token is the argmax.
//
// Bound: both logits are read once, B (2 K + 1) V elements, for the softmax
// statistics: memory. Kernel 1 takes every needed row in pieces (one block per
// piece, maximum and sum in one pass, 16-byte loads); kernel 2 joins the pieces of its
// sequence's rows in every block (a few hundred bytes), walks the acceptance
// test and races over its own piece of the one row that decides, and the
// sequence's last block to finish writes the result. Keys of the race are
// (score, ~index) in 64 bits under atomicMax, so no order of blocks can change
// the answer. Measured, 64 sequences of 7 drafts over 128256, bf16: 63 us, 45 of them
// the statistics (246 MB, 5.5 TB/s); kernel 2 reads 64 MB in the other 18, behind the
// join and before the last block's finish. (Prefetching its noise to L2 under kernel 1
// took 66 us, two steps of its loads in flight 65: registers for resident warps.)
#include <algorithm>

#include "common.cuh"
#include "tc.cuh"

namespace lz {
namespace {

constexpr int kT = 256;
constexpr int kU = 4;  // 16-byte vectors a thread keeps in flight
constexpr int kMaxDraft = 64;
constexpr float kGreedy = 1e-5f;  // temperatures below this (and NaN) are greedy
constexpr int kMaxPieces = 128;

struct Piece {
  float m, s;  // maximum and sum of exp((x - m) / T) of a piece of a row
  int idx;     // lowest index of the maximum (greedy rows)
  int pad;
};
struct SeqState {
  unsigned long long key;  // the race's best (score bits, ~index); 0 = none yet
  unsigned int done;       // blocks of kernel 2 that have finished
  unsigned int pad;
};

struct VerifyArgs {
  const void *target, *draft;
  long long t_sb, t_sr, d_sb, d_sr, n_sb;
  const void* tokens;
  const float *u, *noise, *temp;
  const int* lengths;
  void* out;
  int* accepted;
  Piece* pieces;
  SeqState* seq;
  float temp0;
  int tok64, B, K, V, np, np2;
};

template <typename T>
__device__ __forceinline__ float ld(const T* p) { return static_cast<float>(*p); }
template <>
__device__ __forceinline__ float ld<bf16>(const bf16* p) { return __bfloat162float(*p); }

__device__ __forceinline__ void launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
}
__device__ __forceinline__ void grid_dependency_wait() {
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
}

// A logit as the operator reads it: NaN is a masked token, +inf the largest number.
__device__ __forceinline__ float clean(float x) { return fminf(fmaxf(x, -INFINITY), 3.402823466e38f); }

// 16 bytes of logits as floats
__device__ __forceinline__ void unpack(const uint4& w, float (&x)[8]) {
  x[0] = bf16_lo(w.x), x[1] = bf16_hi(w.x), x[2] = bf16_lo(w.y), x[3] = bf16_hi(w.y);
  x[4] = bf16_lo(w.z), x[5] = bf16_hi(w.z), x[6] = bf16_lo(w.w), x[7] = bf16_hi(w.w);
}
__device__ __forceinline__ void unpack(const uint4& w, float (&x)[4]) {
  x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y);
  x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
}

// kU vectors a lane, 32 apart, in flight at once; past the end they hold -inf.
__device__ __forceinline__ void load(uint4 (&w)[kU], const uint4* p, int i, int end, float) {
#pragma unroll
  for (int u = 0; u < kU; ++u)
    w[u] = i + u * 32 < end ? __ldg(p + i + u * 32)
                            : make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u);
}
__device__ __forceinline__ void load(uint4 (&w)[kU], const uint4* p, int i, int end, bf16) {
#pragma unroll
  for (int u = 0; u < kU; ++u)
    w[u] = i + u * 32 < end ? __ldg(p + i + u * 32)
                            : make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
}
// The largest of a vector's logits (a NaN is passed over unless every one is).
__device__ __forceinline__ float top(const uint4& w, float) {
  return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)),
               fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
}
__device__ __forceinline__ float top(const uint4& w, bf16) {
  const auto* h = reinterpret_cast<const __nv_bfloat162*>(&w);
  const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float top(const uint4 (&w)[kU], float) {
  float m = top(w[0], 0.f);
#pragma unroll
  for (int u = 1; u < kU; ++u) m = fmaxf(m, top(w[u], 0.f));
  return m;
}
__device__ __forceinline__ float top(const uint4 (&w)[kU], bf16) {
  const auto* h = reinterpret_cast<const __nv_bfloat162*>(w);
  __nv_bfloat162 m = h[0];
#pragma unroll
  for (int i = 1; i < 4 * kU; ++i) m = __hmax2(m, h[i]);
  return fmaxf(__low2float(m), __high2float(m));
}
// Two fp32 operations an instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<const unsigned long long&>(a)),
        "l"(reinterpret_cast<const unsigned long long&>(b)),
        "l"(reinterpret_cast<const unsigned long long&>(c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;\n"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<const unsigned long long&>(a)),
        "l"(reinterpret_cast<const unsigned long long&>(b)));
  return d;
}

struct Stat {
  float m, s;
};
// Merge of two (maximum, sum) pairs; c = log2(e) / T.
__device__ __forceinline__ Stat join(Stat a, Stat b, float c) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return {m, 0.f};
  // a side with nothing left has m = -inf and s = 0 (and c is 0 at an infinite temperature)
  return {m, (a.s > 0.f ? a.s * exp2f((a.m - m) * c) : 0.f) +
                 (b.s > 0.f ? b.s * exp2f((b.m - m) * c) : 0.f)};
}

// The same over a warp: the maximum first, then one rescale and a plain sum.
__device__ __forceinline__ Stat warp_join(Stat a, float c) {
  float m = a.m, s = a.s;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  s = a.m > -INFINITY ? s * exp2f((a.m - m) * c) : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return {m, s};
}

__device__ __forceinline__ float temperature(const VerifyArgs& a, int b) {
  return a.temp ? a.temp[b] : a.temp0;
}
__device__ __forceinline__ int drafted(const VerifyArgs& a, int b) {
  return a.lengths ? min(max(a.lengths[b], 0), a.K) : a.K;
}
__device__ __forceinline__ long long token_at(const VerifyArgs& a, int b, int i) {
  const size_t at = (size_t)b * a.K + i;
  return a.tok64 ? static_cast<const long long*>(a.tokens)[at]
                 : (long long)static_cast<const int*>(a.tokens)[at];
}

// 16-byte vectors a piece of a row, in whole steps of a warp.
__device__ __forceinline__ int piece_vectors(int nv, int np) {
  const int per = (nv + np - 1) / np;
  return (per + kU * 32 - 1) / (kU * 32) * (kU * 32);
}

// A warp's piece of a row: vectors v0 .. v1 of 16 bytes, and for the row's first
// piece the elements before and after all vectors, a lane each.
template <typename T>
struct Span {
  const T* x;
  int head, v0, v1, edge, edge_at;
  __device__ __forceinline__ const uint4* vectors() const {
    return reinterpret_cast<const uint4*>(x + head);
  }
};

// The rare ways through a piece are functions of their own, so that their registers
// do not weigh on the usual one.
// Greedy: the largest logit and its lowest index.
template <typename T>
__device__ __noinline__ Piece greedy_piece(const Span<T> sp) {
  constexpr int VE = 16 / sizeof(T);
  const int lane = threadIdx.x & 31;
  const uint4* xv = sp.vectors();
  float m = -INFINITY;
  int at = -1;   // index of m for an element taken one by one,
  int vec = -1;  // or the first vector that holds m
  if (lane < sp.edge && ld(sp.x + sp.edge_at) > m) m = ld(sp.x + sp.edge_at), at = sp.edge_at;
  float vm = -INFINITY;
  for (int i = sp.v0 + lane; i < sp.v1; i += kU * 32) {
    uint4 w[kU];
    load(w, xv, i, sp.v1, T());
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const float t1 = top(w[u], T());
      if (t1 > vm) vm = t1, vec = i + u * 32;
    }
  }
  unsigned long long best = 0;  // (ordered bits of the logit, ~index)
  const auto offer = [&](float v, int i) {
    const unsigned int u = __float_as_uint(v + 0.f);  // -0 counts as 0
    const unsigned int o = u & 0x80000000u ? ~u : u | 0x80000000u;
    best = max(best, (unsigned long long)o << 32 | (unsigned int)~i);
  };
  if (at >= 0) offer(m, at);
  if (vec >= 0) {
    float f[VE];
    unpack(xv[vec], f);
#pragma unroll
    for (int e = VE - 1; e >= 0; --e)
      if (f[e] == vm) at = sp.head + vec * VE + e;
    offer(vm, at);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (!best) return Piece{-INFINITY, 0.f, -1, 0};
  const unsigned int o = (unsigned int)(best >> 32);
  return Piece{__uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o), 0.f,
               (int)~(unsigned int)best, 0};
}
// A piece with NaN or huge values: every logit cleaned.
template <typename T>
__device__ __noinline__ Stat cleaned_piece(const Span<T> sp, float c) {
  constexpr int VE = 16 / sizeof(T);
  const int lane = threadIdx.x & 31;
  const uint4* xv = sp.vectors();
  Stat st = {-INFINITY, 0.f};
  const auto add = [&](float v) {
    v = clean(v);
    if (v > st.m) {
      if (st.m > -INFINITY) st.s *= exp2f((st.m - v) * c);
      st.m = v;
    }
    if (v > -INFINITY) st.s += exp2f((v - st.m) * c);
  };
  if (lane < sp.edge) add(ld(sp.x + sp.edge_at));
  for (int i = sp.v0 + lane; i < sp.v1; i += 32) {
    float f[VE];
    unpack(xv[i], f);
#pragma unroll
    for (int e = 0; e < VE; ++e) add(f[e]);
  }
  return warp_join(st, c);
}

// Statistics of the pieces of the rows, a warp each: a warp's lanes read 16 bytes
// apiece, kU times in flight. (Loading the next vectors ahead of the sums costs
// more in resident warps than it hides: 47 us against 41 for 960 rows of 128256.)
template <typename T>
__global__ void __launch_bounds__(kT, 6) verify_stats_kernel(const VerifyArgs a) {
  constexpr int VE = 16 / sizeof(T);
  const int lane = threadIdx.x & 31, piece = blockIdx.x * (kT / 32) + (threadIdx.x >> 5);
  const int nrow = 2 * a.K + 1, b = blockIdx.y / nrow, r = blockIdx.y - b * nrow;
  launch_dependents();  // verify_draw_kernel reads its own inputs while this one runs
  if (blockIdx.x == 0 && r == 0 && threadIdx.x == 0) a.seq[b] = {0ull, 0u, 0u};
  if (piece >= a.np) return;
  const float t = temperature(a, b);
  const bool greedy = !(t >= kGreedy);
  const int n = drafted(a, b);
  if (r <= a.K ? r > n : (greedy || r - a.K - 1 >= n)) return;
  Span<T> sp;
  sp.x = r <= a.K ? static_cast<const T*>(a.target) + b * a.t_sb + r * a.t_sr
                  : static_cast<const T*>(a.draft) + b * a.d_sb + (r - a.K - 1) * a.d_sr;
  // head up to a 16-byte boundary, whole vectors, tail; head and tail go to piece 0
  sp.head = min(a.V, (int)(((16 - (reinterpret_cast<uintptr_t>(sp.x) & 15)) & 15) / sizeof(T)));
  const int nv = (a.V - sp.head) / VE, tail0 = sp.head + nv * VE;
  const int per = piece_vectors(nv, a.np);
  sp.v0 = min(nv, per * piece);
  sp.v1 = min(nv, sp.v0 + per);
  // up to 2 (VE - 1) elements taken one by one, a lane each
  sp.edge = piece == 0 ? sp.head + a.V - tail0 : 0;
  sp.edge_at = lane < sp.head ? lane : tail0 + lane - sp.head;
  Piece* out = a.pieces + (size_t)blockIdx.y * a.np + piece;
  if (greedy) {
    const Piece p = greedy_piece(sp);
    if (lane == 0) *out = p;
    return;
  }
  const uint4* xv = sp.vectors();
  const float c = kLog2e / t;
  Stat st = {-INFINITY, 0.f};
  float mc = 0.f;  // m c, rounded; its rounding error is taken out of the sum at the end
  float2 sum[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
  const auto rebase = [&](float m) {
    const float omc = mc;
    mc = m * c;
    if (st.m > -INFINITY) {
      const float f = tc::ex2(omc - mc);
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i].x *= f, sum[i].y *= f;
    }
    st.m = m;
  };
  if (lane < sp.edge) {
    const float v = ld(sp.x + sp.edge_at);
    if (v > st.m) rebase(v);
    if (st.m > -INFINITY) sum[0].x = tc::ex2(fmaf(v, c, -mc));
  }
  for (int i = sp.v0 + lane; i < sp.v1; i += kU * 32) {
    uint4 w[kU];
    if (i - lane + kU * 32 <= sp.v1) {
#pragma unroll
      for (int u = 0; u < kU; ++u) w[u] = __ldg(xv + i + u * 32);
    } else {
      load(w, xv, i, sp.v1, T());
    }
    const float vm = top(w, T());
    if (vm > st.m) rebase(vm);
    if (st.m == -INFINITY) continue;
    const float2 cc = make_float2(c, c), nm = make_float2(-mc, -mc);
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      float f[VE];
      unpack(w[u], f);
#pragma unroll
      for (int e = 0; e < VE; e += 2) {
        const float2 g = fma2(make_float2(f[e], f[e + 1]), cc, nm);
        sum[(e >> 1) & 3] = add2(sum[(e >> 1) & 3], make_float2(tc::ex2(g.x), tc::ex2(g.y)));
      }
    }
  }
  sum[0] = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
  st.s = sum[0].x + sum[0].y;
  // sum of 2^(x c - fl(m c)) -> sum of 2^((x - m) c)
  if (st.m > -INFINITY) st.s *= exp2f(-fmaf(st.m, c, -mc));
  st = warp_join(st, c);
  if (!(st.s < INFINITY && st.m < INFINITY)) st = cleaned_piece(sp, c);
  if (lane == 0) *out = {st.m, st.s, -1, 0};
}

// The weight of element j in the race: p - q where positive (p alone without q).
struct Row {
  float m, s;  // maximum and sum
};
__device__ __forceinline__ float prob(float x, Row r, float inv_t) {
  x = clean(x);
  return x > -INFINITY && r.s > 0.f ? expf((x - r.m) * inv_t) / r.s : 0.f;
}
__device__ __forceinline__ unsigned long long race_key(float w, float e, int j) {
  if (!(w > 0.f) || !(e > 0.f)) return 0;
  return (unsigned long long)__float_as_uint(w / e) << 32 | (unsigned int)~j;
}

__device__ __forceinline__ void load8(const bf16* p, float (&x)[8]) {
  unpack(__ldg(reinterpret_cast<const uint4*>(p)), x);
}
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 u = __ldg(reinterpret_cast<const float4*>(p));
  const float4 v = __ldg(reinterpret_cast<const float4*>(p) + 1);
  x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
  x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
}

template <typename T>
__global__ void __launch_bounds__(kT) verify_draw_kernel(const VerifyArgs a) {
  __shared__ Row sP[kMaxDraft + 1], sQ[kMaxDraft];
  __shared__ int sArg[kMaxDraft + 1], sOk[kMaxDraft + 1], sLast;
  __shared__ unsigned long long sKey;
  __shared__ float sBar[kT / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.y, K = a.K, V = a.V;
  const float t = temperature(a, b);
  const bool greedy = !(t >= kGreedy);
  const float inv_t = 1.f / t, c = kLog2e / t;
  const int n = drafted(a, b);
  const T* tg = static_cast<const T*>(a.target) + b * a.t_sb;
  const T* dr = static_cast<const T*>(a.draft) + b * a.d_sb;
  const Piece* pb = a.pieces + (size_t)b * (2 * K + 1) * a.np;

  // what does not come from the statistics: the drafted tokens and their logits
  long long tok = -1;
  float tx = 0.f, dx = 0.f, ui = 0.f;
  if (tid < n) {
    tok = token_at(a, b, tid);
    if (tok >= 0 && tok < V && !greedy) {
      tx = ld(tg + tid * a.t_sr + tok);
      dx = ld(dr + tid * a.d_sr + tok);
      ui = a.u[(size_t)b * K + tid];
    }
  }
  grid_dependency_wait();
  // join the pieces of the n + 1 target rows and the n draft rows, a warp per row
  for (int r = warp; r < 2 * n + 1; r += kT / 32) {
    const int row = r <= n ? r : K + 1 + (r - n - 1);
    if (greedy && r > n) continue;
    Stat st = {-INFINITY, 0.f};
    int idx = -1;
    for (int k = lane; k < a.np; k += 32) {
      const Piece p = pb[(size_t)row * a.np + k];
      if (greedy) {  // pieces 1.. follow each other; piece 0 also holds the row's tail
        if (p.idx >= 0 && (p.m > st.m || (p.m == st.m && p.idx < idx))) st.m = p.m, idx = p.idx;
      } else {
        st = join(st, {p.m, p.s}, c);
      }
    }
    if (greedy) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float m = __shfl_xor_sync(0xffffffffu, st.m, o);
        const int i2 = __shfl_xor_sync(0xffffffffu, idx, o);
        if (i2 >= 0 && (idx < 0 || m > st.m || (m == st.m && i2 < idx))) st.m = m, idx = i2;
      }
    } else {
      st = warp_join(st, c);
    }
    if (lane == 0) {
      if (r <= n) {
        sP[r] = {st.m, st.s};
        sArg[r] = idx;
      } else {
        sQ[r - n - 1] = {st.m, st.s};
      }
    }
  }
  if (tid == 0) sKey = 0;
  __syncthreads();
  if (tid < n) {  // n <= 64
    bool ok = tok >= 0 && tok < V;
    if (ok)
      ok = greedy ? tok == sArg[tid] : ui * prob(dx, sQ[tid], inv_t) < prob(tx, sP[tid], inv_t);
    sOk[tid] = ok;
  }
  __syncthreads();
  int acc = 0;
  while (acc < n && sOk[acc]) ++acc;

  const T* px = tg + acc * a.t_sr;
  const T* qx = acc < n ? dr + acc * a.d_sr : nullptr;
  const float* ex = a.noise + b * a.n_sb;
  const Row P = sP[acc], Q = acc < n ? sQ[acc] : Row{0.f, 0.f};
  const auto weight = [&](int j, bool residual) {
    const float p = prob(ld(px + j), P, inv_t);
    return residual && qx ? p - prob(ld(qx + j), Q, inv_t) : p;
  };
  const auto publish = [&](unsigned long long best) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0 && best) atomicMax(&sKey, best);
    __syncthreads();
  };
  if (!greedy && P.s > 0.f) {
    // First with the hardware's 2^x and 1/x: both of p and q are then within 2^-14
    // of their values wherever they do not underflow, so 5e-4 of either bounds every
    // score from both sides. Then only the tokens whose upper bound reaches the
    // block's best lower bound (a few of thousands) are evaluated with the accurate
    // exp and divisions. Noise that is not positive (or too small to invert) and
    // probabilities that are not finite go to the accurate form at once.
    const int per = (V / 8 + a.np2) / a.np2 * 8;  // whole eights, a.np2 times covers V
    const int j0 = min(V, per * (int)blockIdx.x), j1 = min(V, j0 + per);
    const bool vec = ((reinterpret_cast<uintptr_t>(px) | reinterpret_cast<uintptr_t>(qx) |
                       reinterpret_cast<uintptr_t>(ex)) & 15) == 0;
    const float poff = -log2f(P.s), qoff = Q.s > 0.f ? -log2f(Q.s) : -INFINITY;
    // a warp takes 256 tokens at a time, 8 a lane
    const auto token = [&](int w0, bool whole, int i) {
      return w0 + (whole ? lane * 8 + i : i * 32 + lane);
    };
    // Bounds of the scores of a lane's 8 tokens: the largest lower and upper one,
    // and the tokens that need the accurate form (upper bound above 0 and at least
    // `bar`, or not bounded).
    const auto bounds = [&](int w0, float bar, float& lo, float& hi) {
      const bool whole = vec && w0 + 256 <= j1;
      float x[8], y[8], e[8];
      if (whole) {
        load8(px + w0 + lane * 8, x);
        load8(ex + w0 + lane * 8, e);
        if (qx) load8(qx + w0 + lane * 8, y);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int j = token(w0, false, i);
          x[i] = j < j1 ? ld(px + j) : -INFINITY;
          y[i] = j < j1 && qx ? ld(qx + j) : 0.f;
          e[i] = j < j1 ? ex[j] : 1.f;
        }
      }
      unsigned int need = 0;
      lo = hi = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = tc::ex2(fmaf(x[i] - P.m, c, poff));
        const float q = qx ? tc::ex2(fmaf(y[i] - Q.m, c, qoff)) : 0.f;
        const float both = p + q, w = p - q;
        float r;
        asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(e[i]));
        if (!(both < INFINITY && e[i] >= 1e-30f)) {
          need |= 1u << i;
          continue;
        }
        const float top = fmaf(both, 5e-4f, w) * r;
        lo = fmaxf(lo, fmaf(both, -5e-4f, w) * r);
        hi = fmaxf(hi, top);
        if (top > 0.f && top >= bar) need |= 1u << i;
      }
      return need;
    };
    unsigned long long best = 0;
    const auto evaluate = [&](int w0, unsigned int need) {  // may name tokens past the end
      const bool whole = vec && w0 + 256 <= j1;
      for (; need; need &= need - 1) {
        const int j = token(w0, whole, __ffs(need) - 1);
        if (j < j1) best = max(best, race_key(weight(j, true), ex[j], j));
      }
    };
    // the largest upper bounds of a lane: of one step, and of all its other steps
    float low = 0.f, high = 0.f, rest = 0.f;
    int at = j0;
    for (int w0 = j0 + warp * 256; w0 < j1; w0 += kT * 8) {
      float lo, hi;
      const unsigned int need = bounds(w0, INFINITY, lo, hi);
      low = fmaxf(low, lo);
      rest = fmaxf(rest, fminf(high, hi));
      if (hi > high) high = hi, at = w0;
      if (need) evaluate(w0, need);
    }
    low = fmaxf(low, __uint_as_float((unsigned int)(best >> 32)));
    low = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(low)));
    if (lane == 0) sBar[warp] = low;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kT / 32; ++w) low = fmaxf(low, sBar[w]);
    if (high > 0.f && high >= low) {
      const bool all = rest > 0.f && rest >= low;
      for (int w0 = all ? j0 + warp * 256 : at; w0 < j1; w0 += kT * 8) {
        float lo, hi;
        evaluate(w0, bounds(w0, low, lo, hi));
        if (!all) break;
      }
    }
    publish(best);
  }
  if (tid == 0) {
    if (!greedy && sKey) atomicMax(&a.seq[b].key, sKey);
    __threadfence();
    sLast = atomicAdd(&a.seq[b].done, 1u) == (unsigned)a.np2 - 1;
  }
  __syncthreads();
  if (!sLast) return;
  __threadfence();
  if (tid == 0) sKey = greedy ? 0 : atomicMax(&a.seq[b].key, 0ull);
  __syncthreads();
  // Nothing found: only scores that underflow are left, or the residual is empty
  // (p and q agree over all of V) and the draw is from p.
  for (int residual = 1; residual >= 0; --residual) {
    if (greedy || sKey) break;
    unsigned long long best = 0;
    for (int j = tid; j < V; j += kT) best = max(best, race_key(weight(j, residual), ex[j], j));
    __syncthreads();
    publish(best);
  }
  const int next = greedy ? sArg[acc] : (sKey ? (int)~(unsigned int)sKey : -1);
  for (int i = tid; i <= K; i += kT) {
    const long long x = i < acc ? token_at(a, b, i) : (i == acc ? next : -1);
    const size_t at = (size_t)b * (K + 1) + i;
    if (a.tok64)
      static_cast<long long*>(a.out)[at] = x;
    else
      static_cast<int*>(a.out)[at] = (int)x;
  }
  if (tid == 0) a.accepted[b] = acc;
}

// Pieces of a row: enough of them for `per_sm` on each of the machine's 148 SMs,
// none of fewer than `least` elements.
int pieces_of(int rows, int V, int per_sm, int least) {
  const int want = 148 * per_sm / std::max(rows, 1);
  return std::max(1, std::min({want, ceil_div(V, least), kMaxPieces}));
}

size_t verify_bytes(int B, int K, int V) {
  const int rows = B * (2 * K + 1);
  return (size_t)rows * pieces_of(rows, V, 210, 2048) * sizeof(Piece) + (size_t)B * sizeof(SeqState);
}

template <typename T>
int launch_verify(VerifyArgs& a, cudaStream_t st) {
  verify_stats_kernel<T>
      <<<dim3(ceil_div(a.np, kT / 32), a.B * (2 * a.K + 1)), kT, 0, st>>>(a);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.np2, a.B);
  cfg.blockDim = dim3(kT);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, verify_draw_kernel<T>, a);
  if (e != cudaSuccess) {
    set_error(std::string("verify_draw_kernel: ") + cudaGetErrorString(e));
    return LZ_ERR_CUDA;
  }
  count_launches(2);
  return check_launch("verify_drafts");
}

}  // namespace
}  // namespace lz

extern "C" size_t lz_verify_drafts_workspace_bytes(int B, int K, int V) {
  if (B < 1 || K < 0 || K > lz::kMaxDraft || V < 1 || B > 65535 / (2 * K + 1)) return 0;
  return lz::verify_bytes(B, K, V);
}

extern "C" int lz_verify_drafts(const void* target, long long target_sb, long long target_sr,
                                const void* draft, long long draft_sb, long long draft_sr,
                                int x_dtype, const void* tokens, int tokens_64,
                                const float* uniforms, const float* noise, long long noise_sb,
                                const float* temperature, float temperature_all,
                                const int* lengths, void* out_tokens, int* accepted,
                                void* workspace, size_t workspace_bytes, int B, int K, int V,
                                void* stream) {
  using namespace lz;
  clear_error();
  LZ_REQUIRE(B >= 1 && K >= 0 && V >= 1, LZ_ERR_INVALID_ARGUMENT, "sizes must be positive");
  LZ_REQUIRE(K <= kMaxDraft, LZ_ERR_UNSUPPORTED, "at most 64 drafted tokens");
  LZ_REQUIRE(V <= 1 << 30, LZ_ERR_UNSUPPORTED, "the vocabulary is too large");
  LZ_REQUIRE(B <= 65535 / (2 * K + 1), LZ_ERR_UNSUPPORTED, "too many sequences");
  LZ_REQUIRE(x_dtype == LZ_DTYPE_F32 || x_dtype == LZ_DTYPE_BF16, LZ_ERR_INVALID_ARGUMENT,
             "logits must be LZ_DTYPE_F32 or LZ_DTYPE_BF16");
  LZ_REQUIRE(target && noise && out_tokens && accepted, LZ_ERR_INVALID_ARGUMENT, "null pointer");
  LZ_REQUIRE(K == 0 || (draft && tokens && uniforms), LZ_ERR_INVALID_ARGUMENT,
             "null pointer in the draft");
  const size_t need = verify_bytes(B, K, V);
  LZ_REQUIRE(workspace && workspace_bytes >= need, LZ_ERR_WORKSPACE,
             "workspace too small, see lz_verify_drafts_workspace_bytes");
  LZ_REQUIRE(aligned16(workspace), LZ_ERR_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
  const int rows = B * (2 * K + 1);
  VerifyArgs a = {};
  a.target = target;
  a.draft = draft;
  a.t_sb = target_sb;
  a.t_sr = target_sr;
  a.d_sb = draft_sb;
  a.d_sr = draft_sr;
  a.n_sb = noise_sb;
  a.tokens = tokens;
  a.tok64 = tokens_64 ? 1 : 0;
  a.u = uniforms;
  a.noise = noise;
  a.temp = temperature;
  a.temp0 = temperature_all;
  a.lengths = lengths;
  a.out = out_tokens;
  a.accepted = accepted;
  a.B = B;
  a.K = K;
  a.V = V;
  a.np = pieces_of(rows, V, 210, 2048);
  a.np2 = pieces_of(B, V, 4, 1024);
  a.seq = static_cast<SeqState*>(workspace);
  a.pieces = reinterpret_cast<Piece*>(a.seq + B);
  auto st = static_cast<cudaStream_t>(stream);
  return x_dtype == LZ_DTYPE_F32 ? launch_verify<float>(a, st) : launch_verify<bf16>(a, st);
}
