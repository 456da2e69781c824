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
// the answer.
#include <algorithm>

#include "common.cuh"
#include "tc.cuh"

namespace lz {
namespace {

constexpr int kT = 256;
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

struct Stat {
  float m, s;
};
// Merge of two (maximum, sum) pairs; c = log2(e) / T.
__device__ __forceinline__ Stat join(Stat a, Stat b, float c) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return {m, 0.f};
  // a side with nothing left has m = -inf and s = 0
  return {m, a.s * exp2f((a.m - m) * c) + b.s * exp2f((b.m - m) * c)};
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

// Statistics of one piece of one row.
template <typename T>
__global__ void __launch_bounds__(kT) verify_stats_kernel(const VerifyArgs a) {
  constexpr int VE = 16 / sizeof(T);
  __shared__ Stat sS[kT / 32];
  __shared__ unsigned long long sKey;
  const int tid = threadIdx.x, piece = blockIdx.x;
  const int nrow = 2 * a.K + 1, b = blockIdx.y / nrow, r = blockIdx.y - b * nrow;
  if (piece == 0 && r == 0 && tid == 0) a.seq[b] = {0ull, 0u, 0u};
  const float t = temperature(a, b);
  const bool greedy = !(t >= kGreedy);
  const int n = drafted(a, b);
  if (r <= a.K ? r > n : (greedy || r - a.K - 1 >= n)) return;
  const T* x = r <= a.K ? static_cast<const T*>(a.target) + b * a.t_sb + r * a.t_sr
                        : static_cast<const T*>(a.draft) + b * a.d_sb + (r - a.K - 1) * a.d_sr;
  // head up to a 16-byte boundary, whole vectors, tail; head and tail go to piece 0
  const int head = min(a.V, (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
  const int nv = (a.V - head) / VE, tail0 = head + nv * VE;
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  const int v0 = (int)((long long)nv * piece / a.np), v1 = (int)((long long)nv * (piece + 1) / a.np);
  const int edge = piece == 0 ? head + a.V - tail0 : 0;  // elements taken one by one
  const auto edge_at = [&](int i) { return i < head ? i : tail0 + i - head; };

  if (greedy) {
    unsigned long long best = 0;  // (ordered bits of the logit, ~index)
    const auto offer = [&](float v, int i) {
      v = clean(v);
      if (v == -INFINITY) return;
      const unsigned int u = __float_as_uint(v + 0.f);  // -0 counts as 0
      const unsigned int o = u & 0x80000000u ? ~u : u | 0x80000000u;
      const unsigned long long key = (unsigned long long)o << 32 | (unsigned int)~i;
      if (key > best) best = key;
    };
    for (int i = tid; i < edge; i += kT) offer(ld(x + edge_at(i)), edge_at(i));
    for (int i = v0 + tid; i < v1; i += kT) {
      float f[VE];
      unpack(xv[i], f);
#pragma unroll
      for (int e = 0; e < VE; ++e) offer(f[e], head + i * VE + e);
    }
    if (tid == 0) sKey = 0;
    __syncthreads();
    if (best) atomicMax(&sKey, best);
    __syncthreads();
    if (tid == 0) {
      const unsigned int o = (unsigned int)(sKey >> 32);
      const float m = sKey ? __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o) : -INFINITY;
      a.pieces[(size_t)blockIdx.y * a.np + piece] = {m, 0.f, sKey ? (int)~(unsigned int)sKey : -1, 0};
    }
    return;
  }

  const float c = kLog2e / t;
  // two tries: the second, of a piece that holds NaN or huge values, cleans every logit
  for (int slow = 0; slow < 2; ++slow) {
    Stat st = {-INFINITY, 0.f};
    float mc = 0.f;  // m c, rounded; its rounding error is taken out of the sum at the end
    const auto rebase = [&](float m) {
      const float old = st.m, omc = mc;
      st.m = m;
      mc = m * c;
      if (old > -INFINITY) st.s *= tc::ex2(slow ? (old - m) * c : omc - mc);
    };
    const auto add = [&](float v) {
      if (slow) {
        v = clean(v);
        if (v > st.m) rebase(v);
        if (v > -INFINITY) st.s += exp2f((v - st.m) * c);
      } else {
        if (v > st.m) rebase(v);
        if (st.m > -INFINITY) st.s += tc::ex2(fmaf(v, c, -mc));
      }
    };
    for (int i = tid; i < edge; i += kT) add(ld(x + edge_at(i)));
    for (int i = v0 + tid; i < v1; i += kT) {
      float f[VE];
      unpack(xv[i], f);
#pragma unroll
      for (int e = 0; e < VE; ++e) add(f[e]);
    }
    // sum of 2^(x c - fl(m c)) -> sum of 2^((x - m) c)
    if (!slow && st.m > -INFINITY) st.s *= exp2f(-fmaf(st.m, c, -mc));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      st = join(st, {__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o)},
                c);
    if ((tid & 31) == 0) sS[tid >> 5] = st;
    __syncthreads();
    st = sS[0];
#pragma unroll
    for (int w = 1; w < kT / 32; ++w) st = join(st, sS[w], c);
    __syncthreads();
    // the same for every thread: a finite sum of a finite maximum (or nothing left) stands
    if (slow || (st.s < INFINITY && st.m < INFINITY)) {
      if (tid == 0) a.pieces[(size_t)blockIdx.y * a.np + piece] = {st.m, st.s, -1, 0};
      return;
    }
  }
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

template <typename T>
__global__ void __launch_bounds__(kT) verify_draw_kernel(const VerifyArgs a) {
  __shared__ Row sP[kMaxDraft + 1], sQ[kMaxDraft];
  __shared__ int sArg[kMaxDraft + 1], sOk[kMaxDraft + 1], sLast;
  __shared__ unsigned long long sKey;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.y, K = a.K, V = a.V;
  const float t = temperature(a, b);
  const bool greedy = !(t >= kGreedy);
  const float inv_t = 1.f / t, c = kLog2e / t;
  const int n = drafted(a, b);
  const T* tg = static_cast<const T*>(a.target) + b * a.t_sb;
  const T* dr = static_cast<const T*>(a.draft) + b * a.d_sb;
  const Piece* pb = a.pieces + (size_t)b * (2 * K + 1) * a.np;

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
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float m = __shfl_xor_sync(0xffffffffu, st.m, o);
      const float s = __shfl_xor_sync(0xffffffffu, st.s, o);
      const int i2 = __shfl_xor_sync(0xffffffffu, idx, o);
      if (greedy) {
        if (i2 >= 0 && (idx < 0 || m > st.m || (m == st.m && i2 < idx))) st.m = m, idx = i2;
      } else {
        st = join(st, {m, s}, c);
      }
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
  for (int i = tid; i < n; i += kT) {
    const long long x = token_at(a, b, i);
    bool ok = x >= 0 && x < V;
    if (ok) {
      if (greedy)
        ok = x == sArg[i];
      else
        ok = a.u[(size_t)b * K + i] * prob(ld(dr + i * a.d_sr + x), sQ[i], inv_t) <
             prob(ld(tg + i * a.t_sr + x), sP[i], inv_t);
    }
    sOk[i] = ok;
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
  if (!greedy) {
    unsigned long long best = 0;
    const int j0 = (int)((long long)V * blockIdx.x / a.np2);
    const int j1 = (int)((long long)V * (blockIdx.x + 1) / a.np2);
    for (int j = j0 + tid; j < j1; j += kT) best = max(best, race_key(weight(j, true), ex[j], j));
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
  if (!greedy && !sKey && qx) {
    // p and q agree to the last bit over all of V: the residual is empty, draw from p
    unsigned long long best = 0;
    for (int j = tid; j < V; j += kT) best = max(best, race_key(weight(j, false), ex[j], j));
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

// Pieces of a row: enough blocks for the machine's 148 SMs several times over,
// none of fewer than 4096 elements.
int pieces_of(int rows, int V, int least) {
  const int want = ceil_div(148 * 6, std::max(rows, 1));
  return std::max(1, std::min({want, ceil_div(V, least), kMaxPieces}));
}

size_t verify_bytes(int B, int K, int V) {
  const int rows = B * (2 * K + 1);
  return (size_t)rows * pieces_of(rows, V, 4096) * sizeof(Piece) + (size_t)B * sizeof(SeqState);
}

template <typename T>
int launch_verify(VerifyArgs& a, cudaStream_t st) {
  verify_stats_kernel<T><<<dim3(a.np, a.B * (2 * a.K + 1)), kT, 0, st>>>(a);
  verify_draw_kernel<T><<<dim3(a.np2, a.B), kT, 0, st>>>(a);
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
  a.np = pieces_of(rows, V, 4096);
  a.np2 = pieces_of(B, V, 1024);
  a.seq = static_cast<SeqState*>(workspace);
  a.pieces = reinterpret_cast<Piece*>(a.seq + B);
  auto st = static_cast<cudaStream_t>(stream);
  return x_dtype == LZ_DTYPE_F32 ? launch_verify<float>(a, st) : launch_verify<bf16>(a, st);
}
