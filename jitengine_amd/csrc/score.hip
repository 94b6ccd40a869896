// Scoring of given tokens from rows of logits for gfx950: log-probability, rank, entropy and the most likely
// alternatives in one pass over each row.
//
// With m about max x over a row and, in base 2, y = (x - m) log2 e, l = sum 2^y, t = sum y 2^y:
//   log-probability of v = (y_v - log2 l) ln 2,   entropy = (log2 l - t / l) ln 2,
//   rank of v = #{j : x_j > x_v, or x_j = x_v and j < v}.
// Every lane keeps its own (m, l, t), rescaled where its values grow well past m; lanes, waves and slices meet by the same
// rule in a fixed order, so a call's bits repeat.  y is one fused multiply-add x log2 e - (m log2 e), whose second term's
// rounding is the same for every y and cancels; where that rounding would itself be many powers of two (m far from 0, as in
// a row of nothing but mask values of -1e9 or -1e30), y is (x - m) log2 e.
// Masked entries (-inf, or the type's lowest value beside larger ones) add 0; a row of nothing but lowest values is uniform.
//
// A row is cut into slices, one workgroup each, until the launch fills the chip; a second, small launch puts a row's
// slices together.  Alternatives: a wave keeps the values that pass a threshold in LDS (the threshold is the `top`-th
// largest of its lanes' largest, found bit by bit with ballots, later of what it has kept), and what is kept at the end is
// put in order by counting, for each, those that stand before it.  Lists kept in order by insertion cost 4 times as much
// (32 rows, 20 alternatives: 67 + 19 us).
//
// What bounds it: many rows, the vector ALU (a value takes 5 1/2 instructions of 4 cycles and an exponential of 16, one
// instruction more for the rank: 2,048 rows of 151,936 bf16 values, 622 MB, in 131 to 138 us, 4.5 to 4.7 TB/s; a large copy
// reaches 4.8); few rows, latency: 1 row of 151,936 in 6.6 + 5.4 us of two launches, 32 rows of 248,320 under a mask in 17.5
// + 5.8.  fp32 rows: 2,048 in 239 us, 5.2 TB/s; 1 in 13.7 (bf16 11.3, both calls in a graph).  Several tokens a row cost a
// ballot and a count for each value of a lane and token: 2,048 rows take 124 us with 1 token and no alternatives, 141 with 2,
// 340 with 8, 2,250 with 64; 1 row 7.0, 8.0, 11.0 and 41.
#include "common.hpp"

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxTop = 64, kMaxTokens = 64, kMaxSlices = 64;
constexpr int kRoom = 128;  // values a wave keeps: at least kMaxTop + 64
constexpr float kLowest = -3.402823466e38f, kFloor = -2000.0f, kLog2e = 1.44269504088896341f;
constexpr float kNear = 1048576.0f;  // |m log2 e| up to which it is rounded: by at most 2^-4 there
constexpr double kLn2 = 0.693147180559945309;

struct ScoreArgs {
  const void *x;
  long long stride;       // elements from one row to the next
  const int32_t *tokens;  // [B, nt]
  float *logprob, *entropy, *top_lp;
  int32_t *rank, *top_ids;
  float *part;  // [B, ns, words]: m, l, t, -, nt counts, then top keys
  int B, V, nt, top, ns, slice, words;
};

template <typename T>
struct Elems;  // 16 bytes of a row's values
template <>
struct Elems<uint16_t> {
  static constexpr int N = 8;
  static constexpr uint32_t kLowestWord = 0xff80ff80u;  // -inf
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
  static constexpr uint32_t kLowestWord = 0xff800000u;
  static __device__ __forceinline__ float one(const float *p) { return *p; }
  static __device__ __forceinline__ void widen(const uint4 &q, float *v) {
    v[0] = __uint_as_float(q.x), v[1] = __uint_as_float(q.y), v[2] = __uint_as_float(q.z), v[3] = __uint_as_float(q.w);
  }
};

// One of four.
__device__ __forceinline__ uint32_t pick(uint4 q, int i) {
  const uint32_t lo = i & 1 ? q.y : q.x, hi = i & 1 ? q.w : q.z;
  return i & 2 ? hi : lo;
}

// Value j of a lane's words.
template <typename T>
__device__ __forceinline__ float value_at(uint4 q0, uint4 q1, int j) {
  constexpr int P = 4 / sizeof(T);
  const uint32_t a = pick(q0, j / P), b = pick(q1, j / P), w = j / P & 4 ? b : a;
  if constexpr (sizeof(T) == 2)
    return __uint_as_float(j & 1 ? w & 0xffff0000u : w << 16);
  else
    return __uint_as_float(w);
}

// The largest value below x > -inf (so that v >= x is v > prev(x)).
__device__ __forceinline__ float prev(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return __uint_as_float(u == 0 ? 0x80000001u : u & 0x80000000u ? u + 1 : u - 1);
}

// ------------------------------------------------------------------ a row's softmax
struct Stat {
  float m, l, t;
};

// Whether y is formed with m log2 e rounded, or with the difference to m.
__device__ __forceinline__ bool is_near(float m) { return fabsf(m * kLog2e) < kNear; }

// y from one reference to a larger one: between the two terms that were subtracted, rounded or not, so that it adds no error
// (floor at -2000, where 2^y is 0; a NaN stays one).
__device__ __forceinline__ float between(float a, float b) {
#pragma clang fp contract(off)
  const float ra = a * kLog2e, rb = b * kLog2e;
  float r = ra - rb;
  if (__builtin_expect(!(fmaxf(fabsf(ra), fabsf(rb)) < kNear), 0))
    r = is_near(b) ? fmaf(a, kLog2e, -rb) : is_near(a) ? -fmaf(b, kLog2e, -ra) : (a - b) * kLog2e;
  return r < kFloor ? kFloor : r;
}

__device__ __forceinline__ Stat rebase(const Stat &s, float m) {
  const float d = s.m == m ? 0.0f : between(s.m, m), e = __builtin_amdgcn_exp2f(d);
  return {m, s.l * e, fmaf(s.l, d, s.t) * e};
}

__device__ __forceinline__ Stat join(const Stat &a, const Stat &b) {
  const float m = fmaxf(a.m, b.m);
  const Stat p = rebase(a, m), q = rebase(b, m);
  return {m, p.l + q.l, p.t + q.t};
}

__device__ __forceinline__ Stat wave_join(Stat s) {
  const Stat r = rebase(s, wave_butterfly<true>(s.m));
  return {r.m, wave_butterfly<false>(r.l), wave_butterfly<false>(r.t)};
}

// The log-probability of a logit x in a row of state s, log_l = log2 l.  (l is rounded, so that of a token with nearly all
// of the probability can come out above 0 by some 2^-24: it is 0 then.)
__device__ __forceinline__ float logprob_of(float x, const Stat &s, double log_l) {
  if (s.l != s.l) return __builtin_nanf("");  // a NaN or +inf in the row
  if (!(x > -__builtin_inff())) return x;     // (-inf, also in a row of nothing else; or a NaN)
  const bool near = is_near(s.m);
  const float by = near ? kLog2e : 1.0f, mb = near ? s.m * kLog2e : s.m;
  return (float)fmin(((double)x * (double)by - (double)mb) * (near ? kLn2 : 1.0) - log_l * kLn2, 0.0);
}

// ------------------------------------------------------------------ order
// A value and its index as one number, larger for what stands before: the larger value, then the lower index.  0 is none.
__device__ __forceinline__ uint64_t key_of(float v, int i) {
  const uint32_t u = __float_as_uint(v + 0.0f);  // (-0 ties +0)
  return (uint64_t)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t u = (uint32_t)(k >> 32);
  return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ int key_index(uint64_t k) { return (int)~(uint32_t)k; }

// The n-th largest of the lanes' values (-inf where fewer are numbers): bit by bit from the top over order-preserving keys;
// a bf16 is decided by its 16 bits.
template <int BITS>
__device__ __forceinline__ float nth_of_lanes(float v, int n) {
  const uint32_t u = __float_as_uint(v + 0.0f), k = v == v ? (u & 0x80000000u ? ~u : u | 0x80000000u) : 0u;
  uint32_t least = 0;
  for (int bit = 31; bit >= 32 - BITS; bit--) {
    const uint32_t at = least | 1u << bit;
    if (__builtin_popcountll(__ballot(k >= at)) >= n) least = at;
  }
  const float r = __uint_as_float((least & 0x80000000u ? least ^ 0x80000000u : ~least) & ~(uint32_t)0 << (32 - BITS));
  return r == r && least ? r : -__builtin_inff();
}

// What a wave keeps of its values: keys in LDS (kRoom, and space for the first kMaxTop of them in order).  `top` of the
// values met are not below `bar`; what ties it may stand before them in the step that set it, and stands behind them later.
struct Kept {
  uint64_t *at;
  int count;  // (uniform)
  float bar, least;  // a value passes that is larger than `least`: bar, or the value before it
  __device__ __forceinline__ void raise(float v) { bar = fmaxf(bar, v), least = prev(bar); }
  // Takes the values that pass of every lane's words x (as bits q), of indices i + j + u step.
  template <typename T, int U, int N>
  __device__ __forceinline__ void put(const float (&x)[U][N], const uint4 (&q)[U], int i, int step, int top) {
    uint32_t bits = 0;  // the first value's on top
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int j = 0; j < N; j++) bits = bits + bits + (x[u][j] > least);
    uint64_t mask;
    while ((mask = __ballot(bits != 0))) {
      if (count + __builtin_popcountll(mask) > kRoom) squeeze(top);
      const int at_bit = 31 - __builtin_clz(bits | 1), j = U * N - 1 - at_bit;
      if (bits) {
        const int lower = __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
        at[count + lower] = key_of(value_at<T>(q[0], q[U - 1], j), i + (j / N) * step + j % N);
        bits ^= 1u << at_bit;
      }
      count += __builtin_popcountll(mask);
    }
  }
  // Leaves the `top` first, in order.
  __device__ __forceinline__ void squeeze(int top) {
    uint64_t *to = at + kRoom;
    for (int e = lane_id(); e < (count + 63) / 64 * 64; e += 64) {
      const uint64_t k = e < count ? at[e] : 0;
      int r = 0;
#pragma unroll 4
      for (int j = 0; j < count; j++) r += at[j] > k;
      if (k && r < top) to[r] = k;
    }
    count = min(count, top);
    if (lane_id() < count) at[lane_id()] = to[lane_id()];
    if (count == top) raise(key_value(to[top - 1]));
  }
};

// The first `top` of n keys in LDS, put(r, key) by the thread that has the r-th; every thread of the workgroup calls it.
template <typename Put>
__device__ __forceinline__ void rank_keys(const uint64_t *keys, int n, int top, Put &&put) {
  for (int e = threadIdx.x; e < n; e += kThreads) {
    const uint64_t k = keys[e];
    int r = 0;
#pragma unroll 4
    for (int j = 0; j < n; j++) r += keys[j] > k;
    if (k && r < top) put(r, k);
  }
}

// Outputs of row b that need its whole state; counts of the values before each token.
template <typename T, typename Count>
__device__ __forceinline__ void write_row(const ScoreArgs &a, int b, const Stat &s, double log_l, int tid, int threads,
                                          Count &&count_of) {
  const T *row = (const T *)a.x + (long long)b * a.stride;
  if (tid == 0) {
    const float h = s.l > 0.0f ? (float)(fmax(log_l - (double)s.t / (double)s.l, 0.0) * kLn2) : 0.0f;
    a.entropy[b] = s.l != s.l ? __builtin_nanf("") : h;
  }
  for (int q = tid; q < a.nt; q += threads) {
    const int tok = a.tokens[(long long)b * a.nt + q];
    const bool in = tok >= 0 && tok < a.V;
    const float x = in ? Elems<T>::one(row + tok) : 0.0f;
    a.logprob[(long long)b * a.nt + q] = in ? logprob_of(x, s, log_l) : 0.0f;
    a.rank[(long long)b * a.nt + q] = in && x == x ? count_of(q) : -1;
  }
}

__device__ __forceinline__ void write_alternative(const ScoreArgs &a, int b, const Stat &s, double log_l, int r, uint64_t k) {
  a.top_ids[(long long)b * a.top + r] = key_index(k);
  a.top_lp[(long long)b * a.top + r] = logprob_of(key_value(k), s, log_l);
}

// Fewer than `top` logits of row b are numbers above -inf: its -inf entries follow in order of index (log-probability
// -inf, or NaN in a NaN row), -1 and NaN past the last number.  One wave.
template <typename T>
__device__ __forceinline__ void write_rest(const ScoreArgs &a, int b, const Stat &s, int have) {
  const T *row = (const T *)a.x + (long long)b * a.stride;
  const int l = lane_id();
  for (int i0 = 0; i0 < a.V && have < a.top; i0 += 64) {
    const bool is = i0 + l < a.V && Elems<T>::one(row + i0 + l) == -__builtin_inff();
    const uint64_t mask = __ballot(is);
    const int r = have + __builtin_popcountll(mask & (((uint64_t)1 << l) - 1));
    if (is && r < a.top) {
      a.top_ids[(long long)b * a.top + r] = i0 + l;
      a.top_lp[(long long)b * a.top + r] = s.l != s.l ? __builtin_nanf("") : -__builtin_inff();
    }
    have += __builtin_popcountll(mask);
  }
  for (int r = have + l; r < a.top; r += 64) {
    a.top_ids[(long long)b * a.top + r] = -1;
    a.top_lp[(long long)b * a.top + r] = __builtin_nanf("");
  }
}

// ------------------------------------------------------------------ a slice of a row
constexpr int U = 2;  // 16-byte words a thread takes of a step (5 alternatives, calls in a graph, with 2, 1 and 4 words: 1 row
                      // of 151,936 11.7, 12.9, 12.4 us; 300 rows 41, 45, 46; 2,048 rows 149, 152, 161; 64 x 32,000 13, 12, 17)
template <typename T>
__global__ __launch_bounds__(kThreads) void score_rows_kernel(const ScoreArgs a) {
  constexpr int N = Elems<T>::N, kStep = kThreads * U, kBits = sizeof(T) * 8;  // values of a word, words of a step
  constexpr float kInf = __builtin_inff();
  __shared__ Stat s_stat[kWaves];
  __shared__ float s_x[kMaxTokens], s_bar[kWaves];
  __shared__ int s_tok[kMaxTokens], s_cnt[kWaves][kMaxTokens], s_n;
  __shared__ uint64_t s_keep[kWaves * (kRoom + kMaxTop)];
  const int b = blockIdx.x / a.ns, sl = blockIdx.x % a.ns;
  const int tid = threadIdx.x, wave = tid >> 6;
  const T *row = (const T *)a.x + (long long)b * a.stride;
  // words of 16 bytes at aligned addresses: the row begins `off` values into the first
  const int off = (int)(((uintptr_t)row & 15) / sizeof(T));
  const int words = (a.V + off + N - 1) / N;
  const int w0 = sl * a.slice, w1 = min(words, w0 + a.slice);
  uint4 raw[U];
  auto load = [&](int base) {
    if (base + kStep <= w1 && base * N >= off && (base + kStep) * N - off <= a.V) {
#pragma unroll
      for (int u = 0; u < U; u++) raw[u] = *(const uint4 *)(row + ((base + u * kThreads + tid) * N - off));
      return;
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int w = base + u * kThreads + tid, i0 = w * N - off;
      constexpr uint32_t kLow = Elems<T>::kLowestWord;
      raw[u] = {kLow, kLow, kLow, kLow};
      if (w >= w1) continue;
      if (i0 >= 0 && i0 + N <= a.V) {
        raw[u] = *(const uint4 *)(row + i0);
      } else {  // a word that the row's ends cut
        uint64_t h[2] = {kLow | (uint64_t)kLow << 32, kLow | (uint64_t)kLow << 32};
#pragma unroll 1
        for (int j = 0; j < N; j++) {
          if (i0 + j < 0 || i0 + j >= a.V) continue;
          const int at = j * kBits & 63;
          const uint64_t ones = (((uint64_t)1 << kBits) - 1) << at;
          uint64_t v;
          if constexpr (sizeof(T) == 2)
            v = row[i0 + j];
          else
            v = __float_as_uint(row[i0 + j]);
          if (j * 2 < N)
            h[0] = (h[0] & ~ones) | v << at;
          else
            h[1] = (h[1] & ~ones) | v << at;
        }
        raw[u] = {(uint32_t)h[0], (uint32_t)(h[0] >> 32), (uint32_t)h[1], (uint32_t)(h[1] >> 32)};
      }
    }
  };
  load(w0);
  float xt = __builtin_nanf("");
  int tok = -1, count = 0;  // the wave's values before the only token's (uniform)
  if (a.nt == 1) {
    tok = a.tokens[b];
    if (tok >= 0 && tok < a.V) {
      // (and what equals it in its own word)
      const int wt = (tok + off) / N, i = wt * N - off + tid;
      xt = Elems<T>::one(row + tok);
      if (wt >= w0 && wt < w1 && wave == 0) count = __builtin_popcountll(__ballot(i >= 0 && i < tok && Elems<T>::one(row + i) == xt));
    } else {
      tok = -1;
    }
  } else if (a.nt) {
    for (int q = tid; q < a.nt; q += kThreads) {
      const int t = a.tokens[(long long)b * a.nt + q];
      const bool in = t >= 0 && t < a.V;
      s_tok[q] = in ? t : -1;
      s_x[q] = in ? Elems<T>::one(row + t) : __builtin_nanf("");
#pragma unroll
      for (int w = 0; w < kWaves; w++) s_cnt[w][q] = 0;
    }
    __syncthreads();
  }
  Stat st{kLowest, 0.0f, 0.0f};
  Kept kept{s_keep + wave * (kRoom + kMaxTop), 0, -kInf, -kInf};

  for (int base = w0; base < w1; base += kStep) {
    float x[U][N];
    uint4 cur[U];
#pragma unroll
    for (int u = 0; u < U; u++) cur[u] = raw[u], Elems<T>::widen(raw[u], x[u]);
    if (base + kStep < w1) load(base + kStep);
    float top = -kInf;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int j = 0; j < N; j++) top = fmaxf(top, x[u][j]);
    // (a reference that lags by up to 8 costs nothing: 2^y stays below 2^12; following every larger value took 40
    // instructions a step)
    if (top > st.m + 8.0f) st = rebase(st, top);
    // a lane that has met nothing but masked values takes the wave's largest; where that one is far from 0 too, all lanes
    // have it, and form y alike
    if (!__all(is_near(st.m))) {
      st = rebase(st, wave_butterfly<true>(st.m));
    }
    const float ref = st.m * kLog2e;
    const bool far = !__all(is_near(st.m));
    float l = st.l, t = st.t;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int j = 0; j < N; j++) {
        const float y = fmaf(x[u][j], kLog2e, -ref), e = __builtin_amdgcn_exp2f(y);
        l += e;
        t = fmaf(e, y, t);
      }
    // once more where a masked value (0 times -inf) or a NaN is among them, or y is the other one (one instruction a value
    // less for rows without)
    if (far || __any(t != t)) {
      l = st.l, t = st.t;
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int j = 0; j < N; j++) {
          const float r = far ? (x[u][j] - st.m) * kLog2e : fmaf(x[u][j], kLog2e, -ref), y = r < kFloor ? kFloor : r;
          const float e = __builtin_amdgcn_exp2f(y);
          l += e;
          t = fmaf(e, y, t);
        }
    }
    st.l = l, st.t = t;
    // ranks: a value equal to a token's counts where it is in a word before the token's (the token's own word below;
    // -inf, what fills words up, never passes)
    for (int q = 0; q < a.nt; q++) {
      const float xq = a.nt == 1 ? xt : s_x[q];
      const int wq = ((a.nt == 1 ? tok : s_tok[q]) + off) / N;
      const float pq = xq > -kInf ? prev(xq) : xq;
      int c = 0;
#pragma unroll
      for (int u = 0; u < U; u++) {
        const float least = base + u * kThreads + tid < wq ? pq : xq;
#pragma unroll
        for (int j = 0; j < N; j++) c += __builtin_popcountll(__ballot(x[u][j] > least));
      }
      if (a.nt == 1)
        count += c;
      else if (lane_id() == 0)
        s_cnt[wave][q] += c;
    }
    if (a.top && __any(top > kept.least)) {
      if (__builtin_popcountll(__ballot(top > kept.least)) >= a.top) kept.raise(nth_of_lanes<kBits>(top, a.top));
      kept.put<T>(x, cur, (base + tid) * N - off, kThreads * N, a.top);
      if (kept.count > 2 * a.top) kept.squeeze(a.top);  // (raises the bar, so that few steps come here)
      kept.least = kept.bar;
    }
  }

  // what equals one of several tokens in its own word before it; of a -inf token, all that is -inf before it
  if (a.nt > 1 || xt == -kInf) {
    for (int q = wave; q < a.nt; q += kWaves) {
      const float xq = a.nt == 1 ? xt : s_x[q];
      const int tq = a.nt == 1 ? tok : s_tok[q], wq = (tq + off) / N;
      const int from = xq == -kInf ? w0 : max(w0, wq), to = min(w1, a.nt == 1 ? wq : wq + 1);
      const int i1 = min(tq, to * N - off);
      int c = 0;
      for (int i0 = max(0, from * N - off); i0 < i1; i0 += 64) {
        const int i = i0 + lane_id();
        c += __builtin_popcountll(__ballot(i < i1 && Elems<T>::one(row + i) == xq));
      }
      if (a.nt == 1)
        count += c;
      else if (lane_id() == 0)
        s_cnt[wave][q] += c;
    }
  }
  st = wave_join(st);
  if (kept.count > kMaxTop) kept.squeeze(a.top);
  if (lane_id() == 0) {
    s_stat[wave] = st;
    s_bar[wave] = kept.bar;
    if (a.nt == 1) s_cnt[wave][0] = count;
  }
  if (tid == 0) s_n = 0;
  __syncthreads();
  st = s_stat[0];
#pragma unroll
  for (int w = 1; w < kWaves; w++) st = join(st, s_stat[w]);
  float *part = a.part + (long long)blockIdx.x * a.words;
  auto count_of = [&](int q) {
    int c = 0;
#pragma unroll
    for (int w = 0; w < kWaves; w++) c += s_cnt[w][q];
    return c;
  };
  double log_l = 0.0;
  if (a.ns == 1) {
    log_l = log2((double)st.l);
    write_row<T>(a, b, st, log_l, tid, kThreads, count_of);
  } else {
    if (tid == 0) part[0] = st.m, part[1] = st.l, part[2] = st.t;
    for (int q = tid; q < a.nt; q += kThreads) ((int *)part)[4 + q] = count_of(q);
  }
  if (!a.top) return;
  // what the waves have kept, but for what is below the largest bar
  __shared__ uint64_t s_all[kWaves * kMaxTop];
  float bar = s_bar[0];
#pragma unroll
  for (int w = 1; w < kWaves; w++) bar = fmaxf(bar, s_bar[w]);
  if (lane_id() < kept.count) {
    const uint64_t k = kept.at[lane_id()];
    if (key_value(k) >= bar) s_all[atomicAdd(&s_n, 1)] = k;  // (in any order: they are ranked)
  }
  __syncthreads();
  const int n = s_n;
  uint64_t *to = (uint64_t *)(part + 4 + a.nt + (a.nt & 1));
  rank_keys(s_all, n, a.top, [&](int r, uint64_t k) {
    if (a.ns == 1)
      write_alternative(a, b, st, log_l, r, k);
    else
      to[r] = k;
  });
  if (a.ns == 1) {
    if (n < a.top && wave == 0) write_rest<T>(a, b, st, n);
  } else {
    for (int r = n + tid; r < a.top; r += kThreads) to[r] = 0;
  }
}

// ------------------------------------------------------------------ the slices of a row put together
template <typename T>
__global__ __launch_bounds__(kThreads) void score_merge_kernel(const ScoreArgs a) {
  __shared__ Stat s_stat;
  __shared__ int s_cnt[kMaxTokens], s_n;
  __shared__ uint64_t s_least;
  extern __shared__ uint64_t s_keys[];  // [ns top] the slices' keys, then those that pass
  const int b = blockIdx.x, tid = threadIdx.x, l = lane_id(), wave = tid >> 6, all = a.ns * a.top;
  const float *part = a.part + (long long)b * a.ns * a.words;
  const int keys_at = 4 + a.nt + (a.nt & 1);
  if (tid == 0) s_n = 0, s_least = 0;
  for (int e = tid; e < all; e += kThreads)
    s_keys[e] = *(const uint64_t *)(part + (long long)(e / a.top) * a.words + keys_at + 2 * (e % a.top));
  if (wave == 0) {
    Stat st{kLowest, 0.0f, 0.0f};
    const float *p = part + (long long)l * a.words;
    if (l < a.ns) st = {p[0], p[1], p[2]};
    st = wave_join(st);
    if (l == 0) s_stat = st;
  }
  for (int q = wave; q < a.nt; q += kWaves) {
    int c = 0;
    if (l < a.ns) c = ((const int *)part)[(long long)l * a.words + 4 + q];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) c += __shfl_xor(c, o, 64);
    if (l == 0) s_cnt[q] = c;
  }
  __syncthreads();
  const Stat st = s_stat;
  const double log_l = log2((double)st.l);
  write_row<T>(a, b, st, log_l, tid, kThreads, [&](int q) { return s_cnt[q]; });
  if (!a.top) return;
  // `top` keys are at least this: the top-th of the slices' first, or the least of their d-th where d each make `top`
  const int d = (a.top + a.ns - 1) / a.ns;
  if (d == 1) {
    if (tid < a.ns) {
      const uint64_t k = s_keys[tid * a.top];
      int r = 0;
#pragma unroll 4
      for (int j = 0; j < a.ns; j++) r += s_keys[j * a.top] > k;
      if (r == a.top - 1 && k) s_least = k;
    }
  } else if (wave == 0) {
    uint64_t k = l < a.ns ? s_keys[l * a.top + d - 1] : ~0ull;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint64_t y = (uint64_t)__shfl_xor((long long)k, o, 64);
      k = y < k ? y : k;
    }
    if (l == 0) s_least = k;
  }
  __syncthreads();
  const uint64_t least = s_least ? s_least : 1;
  uint64_t *pass = s_keys + all;
  for (int e = tid; e < all; e += kThreads) {
    const uint64_t k = s_keys[e];
    if (k >= least) pass[atomicAdd(&s_n, 1)] = k;  // (in any order: they are ranked)
  }
  __syncthreads();
  const int n = s_n;
  rank_keys(pass, n, a.top, [&](int r, uint64_t k) { write_alternative(a, b, st, log_l, r, k); });
  if (n < a.top && wave == 0) write_rest<T>(a, b, st, n);
}

// Slices of a row: 1,024 workgroups or so (32 rows of 248,320 bf16: 23 us; 26 with 2,048, 30 with 512), none of fewer
// than 2,048 values.  (Of many alternatives, as many as the second launch's LDS holds keys of.)
int slices_of(long long B, int V, int top) {
  const long long want = 1024 / (B > 0 ? B : 1), most = ((long long)V + 2047) / 2048;
  const long long n = want < most ? want : most, cap = top > kMaxTop / 2 ? kMaxSlices / 2 : kMaxSlices;
  return n < 1 ? 1 : n > cap ? (int)cap : (int)n;
}

int part_words(int nt, int top) { return (4 + nt + (nt & 1) + 2 * top + 3) / 4 * 4; }

template <typename T>
int launch(ScoreArgs a, hipStream_t st) {
  constexpr int N = Elems<T>::N;
  const long long words = ((long long)a.V + 2 * N - 2) / N;  // (of a row that begins anywhere)
  const unsigned blocks = (unsigned)((long long)a.B * a.ns);
  a.slice = (int)((words + a.ns - 1) / a.ns);
  score_rows_kernel<T><<<blocks, kThreads, 0, st>>>(a);
  int rc = jit::check_launch("jit_token_logprobs");
  if (rc != JIT_OK || a.ns == 1) return rc;
  score_merge_kernel<T><<<a.B, kThreads, (size_t)a.ns * a.top * 16, st>>>(a);
  return jit::check_launch("jit_token_logprobs (merge)");
}

}  // namespace

extern "C" long long jit_token_logprobs_workspace_bytes(int B, int V, int n_tokens, int top) {
  if (B < 0 || V <= 0 || n_tokens < 0 || top < 0) return -1;
  const int ns = slices_of(B, V, top);
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
  const int ns = slices_of(B, V, top);
  if ((long long)B * ns * kThreads > 0xffffffffLL)  // (a launch has fewer than 2^32 threads)
    return jit::fail(JIT_EUNSUPPORTED, "token_logprobs covers up to 2^24 - 1 rows, got %d", B);
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
