// Scoring of given tokens from rows of logits for gfx950: log-probability, rank, entropy and the most likely
// alternatives in one pass over each row.
//
// With m = max x, l = sum e^(x - m) and t = sum (x - m) e^(x - m) over a row:
//   log-probability of v = (x_v - m) - ln l,   entropy = ln l - t / l,
//   rank of v = #{j : x_j > x_v, or x_j = x_v and j < v}.
// Every lane keeps its own (m, l, t), rescaled where its largest value grows:
//   l' = l e^(m - m'),   t' = (t + l (m - m')) e^(m - m'),
// and lanes, waves and slices meet by the same rule with sums in a fixed order, so a call's bits repeat.  m starts at
// the lowest finite value and x - m is kept above -1000 (e^-1000 is 0 in fp32): masked entries (-inf, or the type's
// lowest value beside larger ones) add 0 to l and t, and a row of nothing but lowest values is uniform.
//
// A row is cut into slices (one workgroup each) until the launch fills the chip; the slices' results meet in a second,
// small launch.  Alternatives: each wave keeps its `top` best (value, index) in order, one a lane, and looks at a lane's
// values one by one only where the lane's largest (which the softmax has formed anyway) passes the wave's last.
#include "common.hpp"

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxTop = 64, kMaxTokens = 64, kMaxSlices = 64;
constexpr float kLowest = -3.402823466e38f, kFloor = -1000.0f, kLog2e = 1.44269504088896341f;
constexpr int kNone = 0x7fffffff;  // the index of an alternative that is not there

struct ScoreArgs {
  const void *x;
  long long stride;       // elements from one row to the next
  const int32_t *tokens;  // [B, nt]
  float *logprob, *entropy, *top_lp;
  int32_t *rank, *top_ids;
  float *part;  // [B, ns, words]: m, l, t, -, nt counts, top (value, index)
  int B, V, nt, top, ns, slice, words;
};

template <typename T>
struct Elems;  // 16 bytes of a row's values
template <>
struct Elems<uint16_t> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float one(const uint16_t *p) { return bf2f(*p); }
  static __device__ __forceinline__ void widen(const uint4 &q, float *v) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; i++) v[2 * i] = bf2f(w[i] & 0xffffu), v[2 * i + 1] = bf2f_hi(w[i]);
  }
};
template <>
struct Elems<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float one(const float *p) { return *p; }
  static __device__ __forceinline__ void widen(const uint4 &q, float *v) {
    v[0] = __uint_as_float(q.x), v[1] = __uint_as_float(q.y), v[2] = __uint_as_float(q.z), v[3] = __uint_as_float(q.w);
  }
};

struct Stat {
  float m, l, t;
};

// e^d for a d that is at most 0 (or NaN, which stays).
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

__device__ __forceinline__ Stat join(const Stat &a, const Stat &b) {
  const float m = fmaxf(a.m, b.m);
  const float da = fmaxf(a.m - m, kFloor), db = fmaxf(b.m - m, kFloor);
  const float ea = exp_of(da), eb = exp_of(db);
  return {m, fmaf(a.l, ea, b.l * eb), fmaf(fmaf(a.l, da, a.t), ea, fmaf(b.l, db, b.t) * eb)};
}

__device__ __forceinline__ Stat wave_join(Stat s) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) s = join(s, {shfl_xor_f(s.m, o), shfl_xor_f(s.l, o), shfl_xor_f(s.t, o)});
  return s;
}

// Whether (v, i) stands before (w, j): larger value, then lower index.  A NaN stands before nothing.
__device__ __forceinline__ bool before(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

__device__ __forceinline__ float lane_f(float v, int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l)); }

// A wave's best alternatives, lane i the i-th (lanes from `top` on hold what fell off).
struct Best {
  float v;
  int i;
  float last_v;  // of lane top - 1 (uniform)
  int last_i;
  __device__ __forceinline__ void clear() { v = last_v = -__builtin_inff(), i = last_i = kNone; }
  __device__ __forceinline__ void insert(float nv, int ni, int top) {  // (uniform)
    const int p = __builtin_popcountll(__ballot(before(v, i, nv, ni)));
    const int l = lane_id();
    const float pv = __shfl_up(v, 1, 64);
    const int pi = __shfl_up(i, 1, 64);
    v = l < p ? v : l == p ? nv : pv;
    i = l < p ? i : l == p ? ni : pi;
    last_v = lane_f(v, top - 1);
    last_i = __builtin_amdgcn_readlane(i, top - 1);
  }
};

// The `top` best of n sorted lists (n <= 64), lane j walking list j: at(j, k) is its k-th entry.  Called by a whole
// wave; put(k, v, i) by every lane with the k-th best.
template <typename At, typename Put>
__device__ __forceinline__ void merge_lists(int n, int top, At &&at, Put &&put) {
  const int l = lane_id();
  int k = 0;
  float v = -__builtin_inff();
  int i = kNone;
  if (l < n) at(l, 0, v, i);
  for (int r = 0; r < top; r++) {
    float bv = v;
    int bi = i;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const float ov = shfl_xor_f(bv, o);
      const int oi = __shfl_xor(bi, o, 64);
      if (before(ov, oi, bv, bi)) bv = ov, bi = oi;
    }
    put(r, bv, bi);
    if (bi != kNone && i == bi) {  // (indices differ between the lists)
      k++;
      v = -__builtin_inff(), i = kNone;
      if (k < top) at(l, k, v, i);
    }
  }
}

// The outputs of row b from its state, its tokens' counts and its alternatives.
__device__ __forceinline__ float logprob_of(float x, const Stat &s, double ln_l) {
  if (s.l != s.l) return __builtin_nanf("");       // a NaN or +inf in the row
  if (!(x > -__builtin_inff())) return x;          // (-inf, also in a row of nothing else; or a NaN)
  return (float)((double)x - (double)s.m - ln_l);
}

template <typename T>
__device__ __forceinline__ void write_row(const ScoreArgs &a, int b, const Stat &s, int tid, int threads, const int *counts) {
  const T *row = (const T *)a.x + (long long)b * a.stride;
  const double ln_l = log((double)s.l);
  if (tid == 0) a.entropy[b] = s.l != s.l ? __builtin_nanf("") : s.l > 0.0f ? (float)fmax(ln_l - (double)s.t / (double)s.l, 0.0) : 0.0f;
  for (int q = tid; q < a.nt; q += threads) {
    const int tok = a.tokens[(long long)b * a.nt + q];
    const bool in = tok >= 0 && tok < a.V;
    const float x = in ? Elems<T>::one(row + tok) : 0.0f;
    a.logprob[(long long)b * a.nt + q] = in ? logprob_of(x, s, ln_l) : 0.0f;
    a.rank[(long long)b * a.nt + q] = in && x == x ? counts[q] : -1;
  }
}

// U: 16-byte words a thread takes of a step.
template <typename T, int U>
__global__ __launch_bounds__(kThreads) void score_rows_kernel(const ScoreArgs a) {
  constexpr int N = Elems<T>::N, kStep = kThreads * U;  // values of a word, words of a step
  __shared__ Stat s_stat[kWaves];
  __shared__ float s_x[kMaxTokens];
  __shared__ int s_tok[kMaxTokens], s_cnt[kMaxTokens];
  __shared__ float s_v[kWaves][kMaxTop];
  __shared__ int s_i[kWaves][kMaxTop];
  const int b = blockIdx.x / a.ns, sl = blockIdx.x % a.ns;
  const int tid = threadIdx.x, wave = tid >> 6;
  const T *row = (const T *)a.x + (long long)b * a.stride;
  // words of 16 bytes at aligned addresses: the row begins `off` values into the first
  const int off = (int)(((uintptr_t)row & 15) / sizeof(T));
  const int words = (a.V + off + N - 1) / N;
  const int w0 = sl * a.slice, w1 = min(words, w0 + a.slice);
  for (int q = tid; q < a.nt; q += kThreads) {
    const int tok = a.tokens[(long long)b * a.nt + q];
    const bool in = tok >= 0 && tok < a.V;
    s_tok[q] = in ? tok : -1;
    s_x[q] = in ? Elems<T>::one(row + tok) : __builtin_nanf("");
    s_cnt[q] = 0;
  }
  __syncthreads();
  const float xt = a.nt ? s_x[0] : __builtin_nanf("");
  const int tok = a.nt ? s_tok[0] : -1;
  Stat st{kLowest, 0.0f, 0.0f};
  Best best;
  best.clear();
  int count = 0;  // the wave's values before the first token's (uniform)

  auto step = [&](int base) {
    float x[U][N];
    bool whole = true;
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int w = base + u * kThreads + tid, i0 = w * N - off;
      if (w < w1 && i0 >= 0 && i0 + N <= a.V) {
        Elems<T>::widen(*(const uint4 *)(row + i0), x[u]);
      } else {  // past the slice, or a word that the row's ends cut
        whole = false;
#pragma unroll
        for (int j = 0; j < N; j++)
          x[u][j] = w < w1 && i0 + j >= 0 && i0 + j < a.V ? Elems<T>::one(row + i0 + j) : -__builtin_inff();
      }
    }
    float top = -__builtin_inff();
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int j = 0; j < N; j++) top = fmaxf(top, x[u][j]);
    if (top > st.m) {
      const float d = fmaxf(st.m - top, kFloor), e = exp_of(d);
      st.t = fmaf(st.l, d, st.t) * e;
      st.l *= e;
      st.m = top;
    }
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int j = 0; j < N; j++) {
        // (not fmaxf: a NaN has to stay one)
        const float r = x[u][j] - st.m, d = r < kFloor ? kFloor : r, e = exp_of(d);
        st.l += e;
        st.t = fmaf(e, d, st.t);
      }
    const bool all = __all(whole);
    // ranks: a step behind or before the token compares one way
    const int i_lo = base * N - off, i_hi = (base + kStep) * N - off;
    if (a.nt == 1 && all && (i_hi <= tok || i_lo > tok)) {
      if (i_lo > tok) {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int j = 0; j < N; j++) count += __builtin_popcountll(__ballot(x[u][j] > xt));
      } else {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int j = 0; j < N; j++) count += __builtin_popcountll(__ballot(x[u][j] >= xt));
      }
    } else {
      for (int q = 0; q < a.nt; q++) {
        const float xq = s_x[q];
        const int tq = s_tok[q];
        int c = 0;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int j = 0; j < N; j++) {
            const int w = base + u * kThreads + tid, i = w * N - off + j;
            const bool in = w < w1 && i >= 0 && i < a.V;
            c += __builtin_popcountll(__ballot(in && before(x[u][j], i, xq, tq)));
          }
        if (a.nt == 1) count += c;
        else if (lane_id() == 0 && c) atomicAdd(&s_cnt[q], c);
      }
    }
    if (a.top && __any(top > best.last_v || best.last_i == kNone)) {
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int j = 0; j < N; j++) {
          const int w = base + u * kThreads + tid, i = w * N - off + j;
          const bool in = w < w1 && i >= 0 && i < a.V;
          const float v = x[u][j];
          uint64_t mask = __ballot(in && before(v, i, best.last_v, best.last_i));
          while (mask) {
            const int l = __builtin_ctzll(mask);
            best.insert(lane_f(v, l), __builtin_amdgcn_readlane(i, l), a.top);
            mask &= mask - 1;
            mask &= __ballot(before(v, i, best.last_v, best.last_i));
          }
        }
    }
  };
  for (int base = w0; base < w1; base += kStep) step(base);

  st = wave_join(st);
  if (lane_id() == 0) {
    s_stat[wave] = st;
    if (a.nt == 1 && count) atomicAdd(&s_cnt[0], count);
  }
  if (lane_id() < a.top) s_v[wave][lane_id()] = best.v, s_i[wave][lane_id()] = best.i;
  __syncthreads();
  st = s_stat[0];
#pragma unroll
  for (int w = 1; w < kWaves; w++) st = join(st, s_stat[w]);
  const double ln_l = log((double)st.l);
  if (a.ns == 1) {
    write_row<T>(a, b, st, tid, kThreads, s_cnt);
  } else {
    float *p = a.part + (long long)blockIdx.x * a.words;
    if (tid == 0) p[0] = st.m, p[1] = st.l, p[2] = st.t;
    for (int q = tid; q < a.nt; q += kThreads) ((int *)p)[4 + q] = s_cnt[q];
  }
  if (a.top && wave == 0) {
    merge_lists(
        kWaves, a.top, [&](int w, int k, float &v, int &i) { v = s_v[w][k], i = s_i[w][k]; },
        [&](int r, float v, int i) {
          if (lane_id() != 0) return;
          if (a.ns == 1) {
            a.top_ids[(long long)b * a.top + r] = i == kNone ? -1 : i;
            a.top_lp[(long long)b * a.top + r] = i == kNone ? __builtin_nanf("") : logprob_of(v, st, ln_l);
          } else {
            float *p = a.part + (long long)blockIdx.x * a.words + 4 + a.nt + 2 * r;
            p[0] = v;
            ((int *)p)[1] = i;
          }
        });
  }
}

// The slices of a row put together by one wave.
template <typename T>
__global__ __launch_bounds__(64) void score_merge_kernel(const ScoreArgs a) {
  __shared__ int s_cnt[kMaxTokens];
  extern __shared__ float s_list[];  // [ns][top] values, then indices
  const int b = blockIdx.x, l = lane_id();
  const float *part = a.part + (long long)b * a.ns * a.words;
  Stat st{kLowest, 0.0f, 0.0f};
  if (l < a.ns) st = {part[l * a.words], part[l * a.words + 1], part[l * a.words + 2]};
  int *s_idx = (int *)s_list + a.ns * a.top;
  for (int e = l; e < a.ns * a.top; e += 64) {
    const int s = e / a.top, k = e % a.top;
    const float *p = part + s * a.words + 4 + a.nt + 2 * k;
    s_list[e] = p[0];
    s_idx[e] = ((const int *)p)[1];
  }
  for (int q = 0; q < a.nt; q++) {
    int c = l < a.ns ? ((const int *)part)[l * a.words + 4 + q] : 0;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) c += __shfl_xor(c, o, 64);
    if (l == 0) s_cnt[q] = c;
  }
  st = wave_join(st);
  __syncthreads();
  write_row<T>(a, b, st, l, 64, s_cnt);
  if (!a.top) return;
  const double ln_l = log((double)st.l);
  merge_lists(
      a.ns, a.top, [&](int s, int k, float &v, int &i) { v = s_list[s * a.top + k], i = s_idx[s * a.top + k]; },
      [&](int r, float v, int i) {
        if (l != 0) return;
        a.top_ids[(long long)b * a.top + r] = i == kNone ? -1 : i;
        a.top_lp[(long long)b * a.top + r] = i == kNone ? __builtin_nanf("") : logprob_of(v, st, ln_l);
      });
}

// Slices of a row: enough workgroups to fill the chip eight times over, none of fewer than 2,048 values.
int slices_of(long long B, int V) {
  const long long want = 2048 / (B > 0 ? B : 1), most = ((long long)V + 2047) / 2048;
  const long long n = want < most ? want : most;
  return n < 1 ? 1 : n > kMaxSlices ? kMaxSlices : (int)n;
}

int part_words(int nt, int top) { return 4 + nt + 2 * top; }

template <typename T>
int launch(ScoreArgs a, hipStream_t st) {
  constexpr int N = Elems<T>::N;
  const long long words = ((long long)a.V + 2 * N - 2) / N;  // (of a row that begins anywhere)
  const long long blocks = (long long)a.B * a.ns;
  a.slice = (int)((words + a.ns - 1) / a.ns);
  if (a.slice <= 2 * kThreads)
    score_rows_kernel<T, 1><<<(unsigned)blocks, kThreads, 0, st>>>(a);
  else
    score_rows_kernel<T, 4><<<(unsigned)blocks, kThreads, 0, st>>>(a);
  int rc = jit::check_launch("jit_token_logprobs");
  if (rc != JIT_OK || a.ns == 1) return rc;
  score_merge_kernel<T><<<a.B, 64, (size_t)a.ns * a.top * 8, st>>>(a);
  return jit::check_launch("jit_token_logprobs (merge)");
}

}  // namespace

extern "C" long long jit_token_logprobs_workspace_bytes(int B, int V, int n_tokens, int top) {
  if (B < 0 || V <= 0 || n_tokens < 0 || top < 0) return -1;
  const int ns = slices_of(B, V);
  return ns == 1 ? 0 : (long long)B * ns * part_words(n_tokens, top) * 4;
}

extern "C" int jit_token_logprobs(const void *logits, int fp32, int B, int V, long long row_stride, const int32_t *tokens,
                                  int n_tokens, int top, float *logprob, int32_t *rank, float *entropy,
                                  int32_t *top_ids, float *top_logprobs, void *workspace, long long workspace_bytes,
                                  void *stream) {
  if (B < 0 || V <= 0 || n_tokens < 0 || top < 0 || row_stride < V)
    return jit::fail(JIT_EINVAL, "token_logprobs: bad dims B=%d V=%d row_stride=%lld n_tokens=%d top=%d", B, V, row_stride,
                     n_tokens, top);
  if (top > V) return jit::fail(JIT_EINVAL, "token_logprobs: top=%d of %d values", top, V);
  if (top > kMaxTop || n_tokens > kMaxTokens)
    return jit::fail(JIT_EUNSUPPORTED, "token_logprobs covers up to %d alternatives and %d tokens a row, got %d and %d",
                     kMaxTop, kMaxTokens, top, n_tokens);
  if (V > (1 << 30)) return jit::fail(JIT_EUNSUPPORTED, "token_logprobs covers rows of up to 2^30 values, got %d", V);
  const int ns = slices_of(B, V);
  if ((long long)B * ns > 0x7fffffffLL)
    return jit::fail(JIT_EUNSUPPORTED, "token_logprobs covers up to 2^31 - 1 workgroups, got %d rows", B);
  if (B == 0) return JIT_OK;
  if (!logits || !entropy || (n_tokens && (!tokens || !logprob || !rank)) || (top && (!top_ids || !top_logprobs)))
    return jit::fail(JIT_EINVAL, "token_logprobs: null pointer");
  if ((uintptr_t)logits & (fp32 ? 3 : 1)) return jit::fail(JIT_EINVAL, "token_logprobs: the logits are not aligned");
  const long long need = jit_token_logprobs_workspace_bytes(B, V, n_tokens, top);
  if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
    return jit::fail(JIT_EINVAL, "token_logprobs: a workspace of %lld bytes, 16-byte aligned, is needed", need);
  ScoreArgs a{logits, row_stride, tokens, logprob, entropy, top_logprobs, rank, top_ids, (float *)workspace,
              B, V, n_tokens, top, ns, 0, part_words(n_tokens, top)};
  return fp32 ? launch<float>(a, (hipStream_t)stream) : launch<uint16_t>(a, (hipStream_t)stream);
}
