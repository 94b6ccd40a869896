// What the kernels that score straight from hidden rows share: their arguments, a token's running softmax, the weights'
// unpacking, and loads straight into LDS.
#pragma once

#include <type_traits>

#include "qtile.hpp"

namespace head {

constexpr int kThreads = 512, kWaves = 8;
constexpr float kLowest = -3.402823466e38f, kFloor = -1000.0f, kLog2e = 1.44269504088896341f;
constexpr float kFar = 0x1p28f;  // |m| up to which a row is a distribution: m is rounded by at most 8 there
// Where references begin: a tile of logits that all lie below it (in a row whose others do not) adds 0, instead of
// exponentials of its reference's own rounding.  So do the rows that are not there, whose logit is kDead.
constexpr float kStart = -kFar;
constexpr float kDead = -0x1p127f;  // (its product with log2 e is finite)

struct HeadArgs {
  const uint16_t *x;
  const uint8_t *w;
  const int32_t *tokens;
  const uint16_t *xs;  // [3][T16][G32] the groups' sums of x
  float *part;     // [parts][segs][3][32 TT]: a run's states of each tile it meets
  float *picked;   // [T] the given tokens' logits
  float *logprob, *entropy, *lse;
  int T, K, V, parts, segs, tiles, T16, G32;
  int unit;  // 16-row blocks that stay together where a tile of many rows is cut into runs
};

// A token's softmax in base 2 against a reference m near its largest logit: with y = x log2 e - m, l = sum 2^y and
// t = sum y 2^y.  (m is what every y was formed with, so its own rounding cancels.)
struct Stat {
  float m, l, t;
};

__device__ __forceinline__ Stat rebase(const Stat &s, float m) {
  const float d = fmaxf(s.m - m, kFloor), e = __builtin_amdgcn_exp2f(d);
  return {m, s.l * e, fmaf(s.l, d, s.t) * e};
}

__device__ __forceinline__ Stat join(const Stat &a, const Stat &b) {
  const float m = fmaxf(a.m, b.m);
  const Stat p = rebase(a, m), q = rebase(b, m);
  return {m, p.l + q.l, p.t + q.t};
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

// s_waitcnt vmcnt(N) alone; the fence keeps the reads of what has landed behind it.
template <int N>
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4 << 14) | (7 << 4) | (15 << 8));
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void bare_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// 1 KB straight into LDS (16 bytes a lane; M0 wants a wait state before the load that takes it), and 256 bytes
__device__ __forceinline__ void load_lds(const void *base, uint32_t off, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(dst) : "memory", "m0");
}

__device__ __forceinline__ void load_lds4(const void *base, uint32_t off, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "s"(dst) : "memory", "m0");
}

// score_head_mid.hip: the tokens of its one tile for T rows (0: not taken), its runs, its launch.
int mid_tile(long long T, int K);
int mid_parts(int V);
int launch_mid(const HeadArgs &a, hipStream_t st);

}  // namespace head
