// Scoring of given tokens straight from hidden rows and the packed 4-bit head: logits = x . W^T tile by tile on the
// matrix cores, each tile folded into its tokens' running softmax state, so no logit but the given token's reaches
// memory.
//
// With w = s q + b over groups of 64, a logit is sum_g s_g sum_k x_k (q_k + 16) + (b_g - 16 s_g) sum_k x_k: the products
// x (q + 16) are exact in the matrix cores' fp32 sums, and scales and biases enter in fp32; nothing is rounded to fewer
// bits.  (q + 16 is a bf16 by one shift and one AND-OR: 16 is the least power of two whose bf16 steps hold 4 bits below it,
// and the nearer the offset, the less the two sums cancel.)
#include "qtile.hpp"

namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr float kLowest = -3.402823466e38f, kFloor = -1000.0f, kLog2e = 1.44269504088896341f;

struct HeadArgs {
  const uint16_t *x;
  const uint8_t *w;
  const int32_t *tokens;
  float *part;     // [token tiles][parts][3][16 TT]
  float *picked;   // [T] the given tokens' logits
  float *logprob, *entropy, *lse;
  int T, K, V, parts;
};

struct Stat {
  float m, l, t;
};

__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

__device__ __forceinline__ Stat join(const Stat &a, const Stat &b) {
  const float m = fmaxf(a.m, b.m);
  const float da = fmaxf(a.m - m, kFloor), db = fmaxf(b.m - m, kFloor);
  const float ea = exp_of(da), eb = exp_of(db);
  return {m, fmaf(a.l, ea, b.l * eb), fmaf(fmaf(a.l, da, a.t), ea, fmaf(b.l, db, b.t) * eb)};
}

// The 8 values of a packed word as bf16 q + 16.
__device__ __forceinline__ Frag8 unpack16(uint32_t w, uint32_t m, uint32_t c) {
  Frag8 f;
  f.u[0] = ((w << 3) & m) | c;
  f.u[1] = ((w >> 1) & m) | c;
  f.u[2] = ((w >> 5) & m) | c;
  f.u[3] = ((w >> 9) & m) | c;
  return f;
}

// A wave walks 16-row blocks of the head against 16 TT tokens.
template <int TT>
__global__ __launch_bounds__(kThreads) void head_score_kernel(const HeadArgs a) {
  __shared__ float s_part[kWaves][3][16 * TT];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id(), lr = l & 15, lg = l >> 4;
  const int t0 = 16 * TT * blockIdx.y, GP = a.K >> 7, blocks = a.V >> 4;
  const long long blk_bytes = (long long)GP * qtile::kTileBytes;
  uint32_t um = 0x00780078u, uc = 0x41804180u;
  asm volatile("" : "+v"(um), "+v"(uc));
  Frag8 ones;
#pragma unroll
  for (int i = 0; i < 4; i++) ones.u[i] = 0x3F803F80u;
  const uint16_t *xr[TT];
  int tok[TT];
  Stat st[TT];
#pragma unroll
  for (int t = 0; t < TT; t++) {
    const int r = t0 + 16 * t + lr;
    xr[t] = a.x + (long long)min(r, a.T - 1) * a.K + 16 * lg;
    tok[t] = r < a.T ? a.tokens[r] : -1;
    st[t] = {kLowest, 0.0f, 0.0f};
  }
  for (int b = blockIdx.x * kWaves + wave; b < blocks; b += gridDim.x * kWaves) {
    const uint8_t *blk = a.w + b * blk_bytes;
    f32x4 acc[TT];
#pragma unroll
    for (int t = 0; t < TT; t++) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int p = 0; p < GP; p++) {
      const uint4 q = *(const uint4 *)(blk + p * qtile::kNibbleBytes + 16 * l);
      // (scale pair, bias pair) of rows 4 lg .. + 3
      const uint4 *sp = (const uint4 *)(blk + (long long)GP * qtile::kNibbleBytes + p * qtile::kScaleBytes + 32 * lg);
      const uint4 s01 = sp[0], s23 = sp[1];
      const uint32_t sw[4] = {s01.x, s01.z, s23.x, s23.z}, bw[4] = {s01.y, s01.w, s23.y, s23.w};
#pragma unroll
      for (int g = 0; g < 2; g++) {
        const Frag8 w0 = unpack16(g ? q.z : q.x, um, uc), w1 = unpack16(g ? q.w : q.y, um, uc);
        float s[4], o[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          s[i] = g ? bf2f_hi(sw[i]) : bf2f(sw[i] & 0xffffu);
          o[i] = fmaf(-16.0f, s[i], g ? bf2f_hi(bw[i]) : bf2f(bw[i] & 0xffffu));
        }
#pragma unroll
        for (int t = 0; t < TT; t++) {
          Frag8 x0, x1;
          x0.q = *(const uint4 *)(xr[t] + 128 * p + 64 * g);
          x1.q = *(const uint4 *)(xr[t] + 128 * p + 64 * g + 8);
          f32x4 c = mfma16x16x32(w0, x0, f32x4{0.f, 0.f, 0.f, 0.f}), n = mfma16x16x32(ones, x0, f32x4{0.f, 0.f, 0.f, 0.f});
          c = mfma16x16x32(w1, x1, c);
          n = mfma16x16x32(ones, x1, n);
#pragma unroll
          for (int i = 0; i < 4; i++) acc[t][i] = fmaf(o[i], n[i], fmaf(s[i], c[i], acc[t][i]));
        }
      }
    }
    // acc[t][i]: row 16 b + 4 lg + i, token t0 + 16 t + lr
#pragma unroll
    for (int t = 0; t < TT; t++) {
      const int d = tok[t] - 16 * b - 4 * lg;
      if (d >= 0 && d < 4) a.picked[t0 + 16 * t + lr] = d == 0 ? acc[t][0] : d == 1 ? acc[t][1] : d == 2 ? acc[t][2] : acc[t][3];
      const float top = fmaxf(fmaxf(acc[t][0], acc[t][1]), fmaxf(acc[t][2], acc[t][3]));
      if (top > st[t].m) {
        const float dm = fmaxf(st[t].m - top, kFloor), e = exp_of(dm);
        st[t].t = fmaf(st[t].l, dm, st[t].t) * e;
        st[t].l *= e;
        st[t].m = top;
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float r = acc[t][i] - st[t].m, dv = r < kFloor ? kFloor : r, e = exp_of(dv);
        st[t].l += e;
        st[t].t = fmaf(e, dv, st[t].t);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < TT; t++) {
#pragma unroll
    for (int o = 16; o < 64; o <<= 1)
      st[t] = join(st[t], {shfl_xor_f(st[t].m, o), shfl_xor_f(st[t].l, o), shfl_xor_f(st[t].t, o)});
    if (lg == 0) {
      s_part[wave][0][16 * t + lr] = st[t].m;
      s_part[wave][1][16 * t + lr] = st[t].l;
      s_part[wave][2][16 * t + lr] = st[t].t;
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < 16 * TT; c += kThreads) {
    Stat s{s_part[0][0][c], s_part[0][1][c], s_part[0][2][c]};
#pragma unroll
    for (int w = 1; w < kWaves; w++) s = join(s, {s_part[w][0][c], s_part[w][1][c], s_part[w][2][c]});
    float *p = a.part + ((long long)blockIdx.y * a.parts + blockIdx.x) * 3 * 16 * TT + c;
    p[0] = s.m, p[16 * TT] = s.l, p[32 * TT] = s.t;
  }
}

// One wave a token: the parts put together in a fixed order.
__global__ __launch_bounds__(64) void head_merge_kernel(const HeadArgs a, int tile) {
  const int tok = blockIdx.x, l = lane_id();
  const float *p = a.part + (long long)(tok / tile) * a.parts * 3 * tile + tok % tile;
  Stat s{kLowest, 0.0f, 0.0f};
  for (int i = l; i < a.parts; i += 64) {
    const float *q = p + (long long)i * 3 * tile;
    s = join(s, {q[0], q[tile], q[2 * tile]});
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) s = join(s, {shfl_xor_f(s.m, o), shfl_xor_f(s.l, o), shfl_xor_f(s.t, o)});
  if (l) return;
  const double ln_l = log((double)s.l), lse = (double)s.m + ln_l;
  const bool nan = s.l != s.l;
  const int v = a.tokens[tok];
  const bool in = v >= 0 && v < a.V;
  a.lse[tok] = nan ? __builtin_nanf("") : (float)lse;
  a.entropy[tok] = nan ? __builtin_nanf("") : (float)fmax(ln_l - (double)s.t / (double)s.l, 0.0);
  a.logprob[tok] = !in ? 0.0f : nan ? __builtin_nanf("") : (float)((double)a.picked[tok] - (double)s.m - ln_l);
}

constexpr int kMaxParts = 512;

int tile_of(int T) { return T <= 16 ? 16 : T <= 32 ? 32 : T <= 64 ? 64 : 128; }

}  // namespace

extern "C" long long jit_head_logprobs_workspace_bytes(int T, int K, int V) {
  if (T < 0 || K <= 0 || V <= 0) return -1;
  const long long tile = tile_of(T), tiles = (T + tile - 1) / tile;
  return 4 * (tiles * kMaxParts * 3 * tile + T);
}

extern "C" int jit_head_logprobs(const uint16_t *x, int T, int K, const void *w, int V, const int32_t *tokens,
                                 float *logprob, float *entropy, float *lse, void *workspace, long long workspace_bytes,
                                 void *stream) {
  if (T < 0 || K <= 0 || V <= 0) return jit::fail(JIT_EINVAL, "head_logprobs: bad dims T=%d K=%d V=%d", T, K, V);
  if (K % 128 != 0 || V % 16 != 0)
    return jit::fail(JIT_EUNSUPPORTED, "head_logprobs covers K %% 128 == 0 and V %% 16 == 0, got K=%d V=%d", K, V);
  if (T > (1 << 20)) return jit::fail(JIT_EUNSUPPORTED, "head_logprobs covers up to 2^20 rows, got %d", T);
  if (T == 0) return JIT_OK;
  if (!x || !w || !tokens || !logprob || !entropy || !lse) return jit::fail(JIT_EINVAL, "head_logprobs: null pointer");
  if (((uintptr_t)x | (uintptr_t)w) & 15) return jit::fail(JIT_EINVAL, "head_logprobs: x and the head must be 16-byte aligned");
  const long long need = jit_head_logprobs_workspace_bytes(T, K, V);
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))
    return jit::fail(JIT_EINVAL, "head_logprobs: a workspace of %lld bytes, 16-byte aligned, is needed", need);
  const int tile = tile_of(T), tiles = (T + tile - 1) / tile;
  const int fill = (V / 16 + kWaves - 1) / kWaves, parts = fill < kMaxParts ? fill : kMaxParts;
  float *part = (float *)workspace;
  const HeadArgs a{x, (const uint8_t *)w, tokens, part, part + (long long)tiles * kMaxParts * 3 * tile,
                   logprob, entropy, lse, T, K, V, parts};
  const hipStream_t st = (hipStream_t)stream;
  const dim3 grid(parts, tiles);
  switch (tile) {
    case 16: head_score_kernel<1><<<grid, kThreads, 0, st>>>(a); break;
    case 32: head_score_kernel<2><<<grid, kThreads, 0, st>>>(a); break;
    case 64: head_score_kernel<4><<<grid, kThreads, 0, st>>>(a); break;
    default: head_score_kernel<8><<<grid, kThreads, 0, st>>>(a); break;
  }
  const int rc = jit::check_launch("jit_head_logprobs");
  if (rc != JIT_OK) return rc;
  head_merge_kernel<<<T, 64, 0, st>>>(a, tile);
  return jit::check_launch("jit_head_logprobs (merge)");
}
