// Scoring of given tokens straight from hidden rows and the packed 4-bit head: logits = x . W^T tile by tile on the
// matrix cores, each tile folded into its tokens' running softmax state, so no logit but the given token's reaches
// memory.
//
// With w = s q + b over groups of 64, a logit is sum_g s_g sum_k x_k (q_k + 16) + (b_g - 16 s_g) sum_k x_k: the products
// x (q + 16) are exact in the matrix cores' fp32 sums, and scales and biases enter in fp32; nothing is rounded to fewer
// bits.  (q + 16 is a bf16 by one shift and one AND-OR: 16 is the least power of two whose bf16 steps hold 4 bits below it,
// and the nearer the offset, the less the two sums cancel.)
#include <type_traits>

#include "score_head.hpp"

namespace {

using namespace head;

// Lane exchanges within each half of a wave: lane l ^ 16, mirrored in 16, in 8, then lanes l ^ 2 and l ^ 1.
template <int STEP>
__device__ __forceinline__ float half_swap(float v) {
  if constexpr (STEP == 0) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(lane_id() & 16 ? r[0] : r[1]);
  } else {
    constexpr int ctrl = STEP == 1 ? 0x140 : STEP == 2 ? 0x141 : STEP == 3 ? 0x4E : 0xB1;
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xF, 0xF, true));
  }
}
__device__ __forceinline__ float half_max(float v) {
  v = max_xor16(v);
  v = fmaxf(v, half_swap<1>(v));
  v = fmaxf(v, half_swap<2>(v));
  v = fmaxf(v, half_swap<3>(v));
  return fmaxf(v, half_swap<4>(v));
}
// Sums over the 32 lanes of a half of N values each, N / 32 of them left in each lane: in every step a lane gives half
// of its values to its partner and takes the partner's other half.  Lane l ends with values N (l % 32) / 32 .. + N / 32 - 1
// (its bits from the top choose the halves).
template <int N, int STEP = 0>
__device__ __forceinline__ void half_scatter_sum(float *v) {
  if constexpr (STEP < 5) {
    constexpr int H = N / 2;
    const bool up = lane_id() >> (4 - STEP) & 1;
#pragma unroll
    for (int j = 0; j < H; j++) {
      if constexpr (STEP == 0) {
        // (the swap of rows puts the lower rows' first values and the upper rows' second ones side by side)
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[j]), __float_as_uint(v[j + H]), false, false);
        v[j] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
      } else {
        const float keep = up ? v[j + H] : v[j], give = up ? v[j] : v[j + H];
        v[j] = keep + half_swap<STEP>(give);
      }
    }
    half_scatter_sum<H, STEP + 1>(v);
  }
}

// ------------------------------------------------------------------ sums of x over the groups
// xs[3][T16][GP32] bf16: each group's sum over a token's 64 values as three bf16 pieces (24 bits, exact), for the bias
// term's products; groups past K / 64 and tokens past T are 0.  One wave a token and 32 groups.
__global__ __launch_bounds__(64) void head_xsum_kernel(const uint16_t *__restrict__ x, int T, int K, int T16, int G32,
                                                       uint16_t *__restrict__ xs) {
  const int tok = blockIdx.x, l = lane_id(), g = 32 * blockIdx.y + (l >> 1);
  float s = 0.0f;
  if (tok < T && 64 * g < K) {
    const uint4 *p = (const uint4 *)(x + (long long)tok * K + 64 * g + 32 * (l & 1));
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint4 q = p[i];
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; j++) s += bf2f(w[j] & 0xffffu) + bf2f_hi(w[j]);
    }
  }
  s += shfl_xor_f(s, 1);
  if (l & 1) return;
  const long long plane = (long long)T16 * G32, at = (long long)tok * G32 + g;
#pragma unroll
  for (int i = 0; i < 3; i++) {
    const float h = bf2f(f2bf(s));
    xs[i * plane + at] = (uint16_t)(__float_as_uint(h) >> 16);
    s -= h;
  }
}

// ------------------------------------------------------------------ many rows
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kRB = 2;               // 32-row blocks of a wave
constexpr int kMaxTT = 4;            // token tiles of 32
constexpr int kUnit = 2 * kWaves * kRB;  // 16-row blocks that the waves take at a time
constexpr int kWStage = 2 * kRB * qtile::kTileBytes;  // a wave's weights of a step: its 16-row blocks' nibbles, then scales
constexpr int kWLoads = 3 * kRB;     // loads of them

// LDS of a workgroup: two steps' activations, two steps' weights, the groups' sums, the given tokens, the waves' states.
template <int TT>
struct Lds {
  static constexpr int NT = 32 * TT, kStage = NT * 256, kW = 2 * kStage, kSums = kW + 2 * kWaves * kWStage;
  static constexpr bool kHasSums = TT <= 3;  // (four tiles have no room for them)
  static constexpr int kToks = kSums + (kHasSums ? 3 * NT * 64 : 0), kState = kToks + 4 * NT;
  static constexpr int kBytes = kState + kWaves * 12 * NT;
  static_assert(kBytes <= 160 * 1024, "gfx950 gives a workgroup at most 160 KB of LDS");
};

// A workgroup of 8 waves, one a CU, walks 64 kWaves rows of the head at a time (a wave 32 RB of them) against 32 TT tokens.
// Products are 32 x 32 x 16: tokens on the rows, head rows on the columns, so a lane's scale is its own row's.  The work
// is the line of (token tile, unit of 32 or 16 blocks) pairs, tiles first to last, cut into equal runs, one a workgroup (the 8
// waves do a unit at a time, so that no run has a part of one but at a tile's end).  What bounds
// it: the issue slots that products (11 of their 32 cycles), scaling and unpacking share, at a clock that power holds near
// 1.7 GHz: 2,048 rows of 248,320 x 2,048 take 2.04 to 2.22 ms, 1 PFLOP/s (a bare bf16 product of the library 1.68 ms).  Of a
// tile's cycles 65% are its steps with what they wait for, 15% their barriers, 10% the biases and 10% the softmax.  Registers
// spill: 139 of three token tiles, mostly around biases and softmax, and 65 of four, where an offset of load_x and one of the
// rows' LDS addresses come back from memory behind a step's barrier, with a wait for every load before them: what the step
// has just asked for ahead (x(p + 1), w(p + 2)) then has to land at its beginning.
template <int TT>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void head_tile_kernel(const HeadArgs a) {
  using L = Lds<TT>;
  constexpr int NT = L::NT, kStage = L::kStage;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id(), lr = l & 15, row = l & 31, h = l >> 5;
  // (an XCD has consecutive runs: their few tiles' rows of x stay in its L2)
  const int n = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  const int GP = a.K >> 7, blocks = a.V >> 4;
  const uint32_t blk_bytes = (uint32_t)GP * qtile::kTileBytes;
  uint32_t um = 0x00780078u, uc = 0x41804180u;
  asm volatile("" : "+v"(um), "+s"(uc));  // (in registers: v_and_or_b32 takes no literals, and one scalar)
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds);
  const bool short_k = L::kHasSums && a.G32 == 32;
  uint8_t *xsum = lds + L::kSums;  // [3][NT][32] bf16 (K <= 2048)
  int *toks = (int *)(lds + L::kToks);
  float *st = (float *)(lds + L::kState) + wave * 3 * NT;  // the wave's m, l, t [NT]
  const long long plane = (long long)a.T16 * a.G32;
  uint32_t xat[4];  // the lane's piece of product j of group 0 in a stage's first token tile (group 1: the slot's bit 3)
#pragma unroll
  for (int j = 0; j < 4; j++) xat[j] = row * 256 + 16 * ((4 * h + j) ^ lr);
  const int srow = 4 * (wave & 3) + (l >> 4), spiece = (l & 15) ^ srow;
  const uint32_t xoff = (uint32_t)srow * (uint32_t)a.K * 2u + 16 * spiece;
  const uint32_t wlds = lds0 + L::kW + wave * kWStage;  // + kWaves kWStage for odd steps
  // the lane's words of a step: rows 32 r + row; word pair c (products 2 c, 2 c + 1) of group g at + 256 c + 8 g
  const uint8_t *wmine = lds + L::kW + wave * kWStage + (l >> 4 & 1) * qtile::kNibbleBytes + 16 * (32 * h + lr);
  const uint8_t *smine = lds + L::kW + wave * kWStage + 2 * kRB * qtile::kNibbleBytes + row * 8;

  const int units = (blocks + a.unit - 1) / a.unit;  // of a tile
  const long long line = (long long)a.tiles * units;
  long long at0 = line * n / a.parts;
  const long long at1 = line * (n + 1) / a.parts;
  if (n >= a.parts) return;
  for (int seg = 0; at0 < at1; seg++) {
    const int tile = (int)(at0 / units), u0 = (int)(at0 % units), u1 = (int)min((long long)units, u0 + (at1 - at0));
    const int r0 = u0 * a.unit, r1 = min(blocks, u1 * a.unit);
    at0 += u1 - u0;
    const int t0 = NT * tile;
    if (seg) __syncthreads();  // (the last tile's states are read)
    for (int c = l; c < NT; c += 64) st[c] = kStart, st[NT + c] = st[2 * NT + c] = 0.0f;
    for (int c = threadIdx.x; c < NT; c += kThreads) toks[c] = t0 + c < a.T ? a.tokens[t0 + c] : -1;
    if (short_k)
      for (int c = threadIdx.x; c < 3 * NT * 4; c += kThreads)
        ((uint4 *)xsum)[c] = ((const uint4 *)(a.xs + c / (4 * NT) * plane + (long long)t0 * 32))[c % (4 * NT)];

    // activations: a wave's load i brings rows 16 k + 4 (wave % 4) .. + 3 of the tile, k = 2 i + wave / 4; row r's piece c
    // sits in slot c ^ r % 16.  (Rows past T read the last row again: the 16 rows that T cuts have offsets of their own,
    // later ones are those again.)
    const int cut = (a.T - 1 - t0) >> 4;
    const uint32_t xoff_cut = (uint32_t)min(srow, a.T - 1 - t0 - 16 * cut) * (uint32_t)a.K * 2u + 16 * spiece;
    auto load_x = [&](int p, int stage) {
#pragma unroll
      for (int i = 0; i < TT; i++) {
        const int k = 2 * i + (wave >> 2);
        load_lds(a.x + (long long)(t0 + 16 * min(k, cut)) * a.K + 128 * p, k < cut ? xoff : xoff_cut,
                 __builtin_amdgcn_readfirstlane(lds0 + stage * kStage + k * 4096 + (wave & 3) * 1024));
      }
    };
    __syncthreads();
    int stage = 0;
    load_x(0, 0);
  // `tiles` tiles of RB 32-row blocks a wave, from 16-row block b0 on
  auto walk = [&](auto rb_c, int b0, int tiles) {
    constexpr int RB = decltype(rb_c)::value;
    if (tiles <= 0) return;
    int first = b0 + 2 * RB * wave;
    // weights of step p into their stage: (blocks past the head read its last one, for nothing)
    const uint32_t scales = GP * qtile::kNibbleBytes;
    auto load_w = [&](int p) {
      const uint32_t to = wlds + (p & 1) * (kWaves * kWStage);
      p = min(p, GP - 1);  // (past the last: loaded and unused, so that every step waits for the same counts)
#pragma unroll
      for (int b = 0; b < 2 * RB; b++)
        load_lds(a.w + (long long)min(first + b, blocks - 1) * blk_bytes + p * qtile::kNibbleBytes, 16 * l,
                 __builtin_amdgcn_readfirstlane(to + b * qtile::kNibbleBytes));
#pragma unroll
      for (int r = 0; r < RB; r++) {  // (the scale tiles of two blocks, 32 words each)
        const int b = min(first + 2 * r, blocks - 1);
        load_lds4(a.w + (long long)b * blk_bytes + scales + p * qtile::kScaleBytes,
                  (l >> 5 && b + 1 < blocks ? blk_bytes : 0u) + 4 * (l & 31),
                  __builtin_amdgcn_readfirstlane(to + 2 * kRB * qtile::kNibbleBytes + r * 256));
      }
    };
    load_w(0);
    load_w(1);
    for (; tiles > 0; tiles--) {
    f32x16 acc[RB][TT];
#pragma unroll
    for (int r = 0; r < RB; r++)
#pragma unroll
      for (int t = 0; t < TT; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[r][t][i] = 0.0f;
    // A step is a chain of four products for each group, token tile and row block.  Chain n's products stand beside chain
    // n - 1's sums and, when a row block's last chain of a group has gone, the unpacking of its weights for the next.
    // Loads go out as x(p + 1) at the top of step p and w(p + 2) when step p has unpacked its group 1.
    Frag8 wf[RB][4];
    float s[RB];
    uint2 wq[2];
    uint32_t ws;
    f32x16 c[2];
    auto ask = [&](int p, int g, int r) {  // the words and scales of row block r's group g
      const int o = (p & 1) * (kWaves * kWStage) + 2 * r * qtile::kNibbleBytes + 8 * g;
      wq[0] = *(const uint2 *)(wmine + o);
      wq[1] = *(const uint2 *)(wmine + o + 256);
      ws = *(const uint32_t *)(smine + (p & 1) * (kWaves * kWStage) + r * 256);
    };
    auto unpack = [&](int r, int j) { wf[r][j] = unpack16(j & 1 ? wq[j >> 1].y : wq[j >> 1].x, um, uc); };
    auto scale = [&](int g, int r) { s[r] = g ? bf2f_hi(ws) : bf2f(ws & 0xffffu); };
    wait_loads<kWLoads * RB / kRB>();  // w(0)
#pragma unroll
    for (int r = 0; r < (RB > 1 ? RB - 1 : 1); r++) {
      ask(0, 0, r);
#pragma unroll
      for (int j = 0; j < 4; j++) unpack(r, j);
      scale(0, r);
    }
    if (RB > 1) s[RB - 1] = 0.0f;
    constexpr int kChains = 2 * TT * RB;
#pragma unroll
    for (int i = 0; i < 16; i++) c[(kChains - 1) & 1][i] = 0.0f;  // (the first step's first sums add nothing)
    auto sums = [&](int n, int i0, int i1) {  // of chain n
      const int r = n % RB, t = n / RB % TT;
#pragma unroll
      for (int i = i0; i < i1; i++) acc[r][t][i] = fmaf(s[r], c[n & 1][i], acc[r][t][i]);
    };
    for (int p = 0; p < GP; p++) {
      wait_loads<kWLoads * RB / kRB>();  // x(p); w(p + 1) may be on its way
      bare_barrier();
      load_x(p + 1 < GP ? p + 1 : 0, stage ^ 1);
      const uint8_t *xs = lds + stage * kStage;
      // unit u's pieces lie in slots 4 u .. + 3 of six: the next unit's first two come during its last chain, the other
      // two when that chain has passed theirs
      Frag8 x[6];
      auto read_x = [&](int u, int j) {
        x[(4 * u + j) % 6].q = *(const uint4 *)(xs + (u / TT ? xat[j] ^ 128u : xat[j]) + u % TT * 8192);
      };
#pragma unroll
      for (int j = 0; j < 4; j++) read_x(0, j);
#pragma unroll
      for (int n = 0; n < kChains; n++) {
        const int u = n / RB, r = n % RB, g = u / TT, t = u % TT;
        const bool ahead = r == RB - 1 && u + 1 < 2 * TT;
        // row block q's last chain of group up / TT was the one before this (RB > 1): its next weights are unpacked here
        const int q = (n + RB - 1) % RB, up = n ? (n - 1) / RB : -1;
        const bool turn = RB > 1 && (!n || up % TT == TT - 1);  // (the last one's of a step: in the next step's first)
        const int tp = n ? up / TT : 0, tg = n ? 1 - up / TT : 0;
        if (ahead) read_x(u + 1, 0), read_x(u + 1, 1);
        if (turn) {
          if (tp && q == 0) wait_loads<TT + kWLoads>();  // w(p + 1)
          ask(p + tp, tg, q);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
          f32x16 z;
#pragma unroll
          for (int i = 0; i < 16; i++) z[i] = 0.0f;
          c[n & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[(4 * u + j) % 6].v, wf[r][j].v, j ? c[n & 1] : z, 0, 0, 0);
          if (ahead && j >= 1 && j < 3) read_x(u + 1, j + 1);
          if constexpr (RB > 1)
            if (j) sums(n ? n - 1 : kChains - 1, j == 1 ? 0 : j == 2 ? 6 : 11, j == 1 ? 6 : j == 2 ? 11 : 16);
          if (turn && j) {
            unpack(q, j - 1);
            if (j == 3) unpack(q, 3);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if (turn) scale(tg, q);
        if (RB > 1 && n == TT * RB) load_w(p + 2);  // (group 1 of the last row block is out)
        if (RB == 1) {
          sums(n, 0, 16);
          if (t == TT - 1) {
            if (g) wait_loads<TT + kWLoads / 2>();
            ask(p + g, 1 - g, 0);
#pragma unroll
            for (int j = 0; j < 4; j++) unpack(0, j);
            scale(1 - g, 0);
            if (!g) load_w(p + 2);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      stage ^= 1;
    }
    if constexpr (RB > 1) sums(kChains - 1, 0, 16);
    // biases: sum_g (b - 16 s)_g X_g over 16 groups at a time, X in its three pieces, the smallest first.  The next tile's
    // first weights are asked for behind the scales and biases.
    const int at = first;
    for (int g0 = 0; g0 < a.G32; g0 += 32) {
      Frag8 fs[2][RB], fb[2][RB];
#pragma unroll
      for (int r = 0; r < RB; r++) {
        const int b = min(at + 2 * r, blocks - 1);
        const uint8_t *sp = a.w + (long long)b * blk_bytes + scales;
        const uint32_t so = (l & 16 && b + 1 < blocks ? blk_bytes : 0u) + 8 * lr;
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const int p = g0 / 2 + 8 * k + 4 * h + j;
            const uint2 v = *(const uint2 *)(sp + (so + min(p, GP - 1) * qtile::kScaleBytes));
            fs[k][r].u[j] = p < GP ? v.x : 0u;
            fb[k][r].u[j] = p < GP ? v.y : 0u;
          }
      }
      if (g0 + 32 >= a.G32) {
        asm volatile("" ::: "memory");
        first += 2 * kWaves * RB;
        load_w(0);
        load_w(1);
      }
#pragma unroll
      for (int t = 0; t < TT; t++) {
        Frag8 x[2][3];
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
          for (int i = 0; i < 3; i++)
            x[k][i].q = short_k ? *(const uint4 *)(xsum + ((i * NT + 32 * t + row) * 64 + 32 * k + 16 * h))
                                : *(const uint4 *)(a.xs + i * plane + (long long)(t0 + 32 * t + row) * a.G32 + g0 + 16 * k + 8 * h);
#pragma unroll
        for (int r = 0; r < RB; r++) {
          f32x16 d;
#pragma unroll
          for (int i = 0; i < 16; i++) d[i] = 0.0f;
#pragma unroll
          for (int k = 0; k < 2; k++)
#pragma unroll
            for (int i = 2; i >= 0; i--) {
              d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[k][i].v, fs[k][r].v, d, 0, 0, 0);
              acc[r][t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[k][i].v, fb[k][r].v, acc[r][t], 0, 0, 0);
            }
#pragma unroll
          for (int i = 0; i < 16; i++) acc[r][t][i] = fmaf(-16.0f, d[i], acc[r][t][i]);
        }
      }
    }
    // acc[r][t][i]: head row 16 at + 32 r + row, token t0 + 32 t + 8 (i / 4) + 4 h + i % 4
    const int live = 16 * (r1 - at);  // rows that are there
    if (live <= 0) continue;
    if (live < 32 * RB) {
#pragma unroll
      for (int r = 0; r < RB; r++)
        if (32 * r + row >= live) {
#pragma unroll
          for (int t = 0; t < TT; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[r][t][i] = kDead;
        }
    }
    // given tokens of these rows, and how far the largest logits lie above their references
    float over = kLowest;
    const uint32_t mine = min(live, 32 * RB);
#pragma unroll
    for (int t = 0; t < TT; t++)
#pragma unroll
      for (int i4 = 0; i4 < 4; i4++) {
        const int4 tk = *(const int4 *)(toks + 32 * t + 8 * i4 + 4 * h);
        const int v[4] = {tk.x - 16 * at, tk.y - 16 * at, tk.z - 16 * at, tk.w - 16 * at};
        if (__any((uint32_t)v[0] < mine || (uint32_t)v[1] < mine || (uint32_t)v[2] < mine || (uint32_t)v[3] < mine)) {
#pragma unroll
          for (int r = 0; r < RB; r++)
#pragma unroll
            for (int i = 0; i < 4; i++)
              if (v[i] == 32 * r + row && (uint32_t)v[i] < mine) a.picked[t0 + 32 * t + 8 * i4 + 4 * h + i] = acc[r][t][4 * i4 + i];
        }
        const f32x4 m = *(const f32x4 *)(st + 32 * t + 8 * i4 + 4 * h);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float x = acc[0][t][4 * i4 + i];
#pragma unroll
          for (int r = 1; r < RB; r++) x = fmaxf(x, acc[r][t][4 * i4 + i]);
          over = fmaxf(over, fmaf(x, kLog2e, -m[i]));
        }
      }
    // References rise where some 2^y would grow past 2^64 (the first tile's do); everything else is summed as it is.
    if (__any(over > 64.0f)) {
#pragma unroll
      for (int t = 0; t < TT; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
          float x = acc[0][t][i];
#pragma unroll
          for (int r = 1; r < RB; r++) x = fmaxf(x, acc[r][t][i]);
          x = half_max(x) * kLog2e;
          float *p = st + 32 * t + 8 * (i / 4) + 4 * h + i % 4;
          const Stat s0{p[0], p[NT], p[2 * NT]}, n0 = rebase(s0, fmaxf(s0.m, x));
          if (row == 0) p[0] = n0.m, p[NT] = n0.l, p[2 * NT] = n0.t;
        }
      asm volatile("" ::: "memory");  // (a wave's LDS accesses complete in order)
    }
    // sums over the rows, 32 tokens at a time: each lane ends with one of its half's 16 tokens or none
#pragma unroll
    for (int t = 0; t < TT; t++) {
      float v[32];  // l of the half's 16 tokens, then t
#pragma unroll
      for (int i4 = 0; i4 < 4; i4++) {
        const f32x4 m = *(const f32x4 *)(st + 32 * t + 8 * i4 + 4 * h);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float p = 0.0f, q = 0.0f;
#pragma unroll
          for (int r = 0; r < RB; r++) {
            const float y = fmaf(acc[r][t][4 * i4 + i], kLog2e, -m[i]), e = __builtin_amdgcn_exp2f(y);
            p += e;
            q = fmaf(e, y, q);
          }
          v[4 * i4 + i] = p, v[16 + 4 * i4 + i] = q;
        }
      }
      half_scatter_sum<32>(v);
      // lane `row` has value `row`: l of token index row % 16, or its t
      st[NT + (row >= 16 ? NT : 0) + 32 * t + 8 * (lr >> 2) + 4 * h + (lr & 3)] += v[0];
    }
    asm volatile("" ::: "memory");
    }
  };
  constexpr int span = kUnit;
  const int n_full = (r1 - r0) / span, rest = (r1 - r0) % span;
  walk(std::integral_constant<int, kRB>{}, r0, n_full + (rest > span / 2 ? 1 : 0));
  if (rest > 0 && rest <= span / 2) walk(std::integral_constant<int, 1>{}, r0 + span * n_full, 1);
    wait_loads<0>();  // (the last stages that were asked for)
    __syncthreads();
    const float *all = (const float *)(lds + L::kState);
    for (int c = threadIdx.x; c < NT; c += kThreads) {
      Stat s{all[c], all[NT + c], all[2 * NT + c]};
#pragma unroll
      for (int i = 1; i < kWaves; i++) {
        const float *p = all + 3 * NT * i + c;
        s = join(s, {p[0], p[NT], p[2 * NT]});
      }
      float *p = a.part + ((long long)n * a.segs + seg) * 3 * NT + c;
      p[0] = s.m, p[NT] = s.l, p[2 * NT] = s.t;
    }
  }
}

// ------------------------------------------------------------------ few rows
// Up to 16 rows, held in LDS: 8 waves a workgroup, one workgroup a CU, each wave streaming 16-row blocks of the head of
// its own with RING KB of weights in flight (16 x 16 x 32 products, tokens on the rows).  Bound by the head's bytes: 1 row
// of 151,936 x 2,048 (175 MB) takes 38 to 40 us, 4.4 to 4.6 TB/s (a call 40 us, of head_tile_kernel 59).
constexpr int kFewBytes = 128 * 1024;  // LDS for the rows
constexpr int kFewChunks = 2;          // 32-group chunks of a row at most (K <= 4096)

template <int RING>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void head_few_kernel(const HeadArgs a) {
  constexpr int NT = 16;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ float s_state[kWaves][3][NT];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id(), lr = l & 15, lg = l >> 4;
  const int n = blockIdx.x, GP = a.K >> 7, blocks = a.V >> 4, row_bytes = 2 * a.K;
  const int r0 = (int)((long long)blocks * n / a.parts), r1 = (int)((long long)blocks * (n + 1) / a.parts);
  const long long blk_bytes = (long long)GP * qtile::kTileBytes;
  uint32_t um = 0x00780078u, uc = 0x41804180u;
  asm volatile("" : "+v"(um), "+s"(uc));

  uint4 ring[RING];
  uint2 sb[kFewChunks][4], sn[kFewChunks][4];  // scale and bias pairs of pair 16 c + 4 lg + j, this block's and the next's
  const int chunks = a.G32 / 32;
  auto blk = [&](int b) { return a.w + min(b, blocks - 1) * blk_bytes; };  // (past the run: loaded and unused)
  auto load_pair = [&](int b, int p) { return ld_stream16(blk(b) + p * qtile::kNibbleBytes + 16 * l); };
  auto load_scales = [&](int b, uint2 (&to)[kFewChunks][4]) {
    const uint8_t *sp = blk(b) + (long long)GP * qtile::kNibbleBytes + 8 * lr;
#pragma unroll
    for (int c = 0; c < kFewChunks; c++)
      if (c < chunks) {
#pragma unroll
        for (int j = 0; j < 4; j++) to[c][j] = *(const uint2 *)(sp + min(16 * c + 4 * lg + j, GP - 1) * qtile::kScaleBytes);
      }
  };
  // The rows (zeros past T, piece c of a pair in slot c ^ row) are asked for ahead of the weights: loads come back in
  // order, and nothing starts without them.
  const int per_row = row_bytes / 16, pieces = NT * per_row;
  auto row_piece = [&](int c) {
    const int row = c / per_row, piece = c % per_row;
    return c < pieces && row < a.T ? *(const uint4 *)(a.x + (long long)row * a.K + 8 * piece) : make_uint4(0u, 0u, 0u, 0u);
  };
  auto put_piece = [&](int c, const uint4 &q) {
    const int row = c / per_row, piece = c % per_row;
    if (c < pieces) *(uint4 *)(lds + row * row_bytes + 16 * ((piece & ~15) | ((piece ^ row) & 15))) = q;
  };
  uint4 xq[8];
#pragma unroll
  for (int i = 0; i < 8; i++) xq[i] = row_piece(threadIdx.x + i * kThreads);
  asm volatile("" ::: "memory");
  int b = r0 + wave;
#pragma unroll
  for (int j = 0; j < RING; j++) ring[j] = load_pair(b, min(j, GP - 1));
  load_scales(b, sb);
  asm volatile("" ::: "memory");
#pragma unroll
  for (int i = 0; i < 8; i++) put_piece(threadIdx.x + i * kThreads, xq[i]);
  for (int c = threadIdx.x + 8 * kThreads; c < pieces; c += kThreads) put_piece(c, row_piece(c));
  // then each group's sum in three bf16 pieces [3][NT][G32]
  __syncthreads();
  uint16_t *xs = (uint16_t *)(lds + NT * row_bytes);
  for (int c = threadIdx.x; c < NT * a.G32; c += kThreads) {
    const int row = c / a.G32, g = c % a.G32;
    float s = 0.0f;
    if (64 * g < a.K)
      for (int i = 0; i < 8; i++) {
        const uint4 q = *(const uint4 *)(lds + row * row_bytes + 256 * (g >> 1) + 16 * ((8 * (g & 1) + i) ^ (row & 15)));
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; j++) s += bf2f(w[j] & 0xffffu) + bf2f_hi(w[j]);
      }
#pragma unroll
    for (int i = 0; i < 3; i++) {
      const float v = bf2f(f2bf(s));
      xs[i * NT * a.G32 + c] = (uint16_t)(__float_as_uint(v) >> 16);
      s -= v;
    }
  }
  __syncthreads();

  int tok[4];
  Stat st[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    tok[i] = 4 * lg + i < a.T ? a.tokens[4 * lg + i] : -1;
    st[i] = {kStart, 0.0f, 0.0f};
  }
  const uint8_t *xrow = lds + lr * row_bytes;
  for (; b < r1; b += kWaves) {
    load_scales(b + kWaves, sn);
    asm volatile("" ::: "memory");
    f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int p0 = 0; p0 < GP; p0 += RING) {
#pragma unroll
      for (int j = 0; j < RING; j++) {
        // (every load goes out, pairs past the last for nothing, so that the waits know how many are in flight)
        const int p = p0 + j;
        const uint4 q = ring[j];
        const bool more = p + RING < GP;
        ring[j] = load_pair(more ? b : b + kWaves, more ? p + RING : min(j, GP - 1));
        asm volatile("" ::: "memory");
        if (p < GP) {
          const uint32_t su = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * ((p & 12) * 4 + lr), (int)(p < 16 ? sb[0][j & 3].x : sb[1][j & 3].x));
#pragma unroll
          for (int g = 0; g < 2; g++) {
            const Frag8 w0 = unpack16(g ? q.z : q.x, um, uc), w1 = unpack16(g ? q.w : q.y, um, uc);
            const float s = g ? bf2f_hi(su) : bf2f(su & 0xffffu);
            Frag8 x0, x1;
            x0.q = *(const uint4 *)(xrow + 256 * p + 16 * ((8 * g + 2 * lg) ^ lr));
            x1.q = *(const uint4 *)(xrow + 256 * p + 16 * ((8 * g + 2 * lg + 1) ^ lr));
            f32x4 c = mfma16x16x32(x0, w0, f32x4{0.f, 0.f, 0.f, 0.f});
            c = mfma16x16x32(x1, w1, c);
#pragma unroll
            for (int i = 0; i < 4; i++) acc[i] = fmaf(s, c[i], acc[i]);
          }
        }
      }
    }
    // biases, as in head_tile_kernel
#pragma unroll
    for (int c = 0; c < kFewChunks; c++)
      if (c < chunks) {
        Frag8 fs, fb;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const bool in = 16 * c + 4 * lg + j < GP;
          fs.u[j] = in ? sb[c][j].x : 0u;
          fb.u[j] = in ? sb[c][j].y : 0u;
        }
        f32x4 d = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 2; i >= 0; i--) {
          Frag8 x;
          x.q = *(const uint4 *)(xs + (i * NT + lr) * a.G32 + 32 * c + 8 * lg);
          d = mfma16x16x32(x, fs, d);
          acc = mfma16x16x32(x, fb, acc);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] = fmaf(-16.0f, d[i], acc[i]);
      }
#pragma unroll
    for (int c = 0; c < kFewChunks; c++)
#pragma unroll
      for (int j = 0; j < 4; j++) sb[c][j] = sn[c][j];
    // acc[i]: head row 16 b + lr, token 4 lg + i; every lane keeps its own rows' state
    bool over = false;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (tok[i] == 16 * b + lr) a.picked[4 * lg + i] = acc[i];
      over |= fmaf(acc[i], kLog2e, -st[i].m) > 64.0f;
    }
    if (__any(over)) {
#pragma unroll
      for (int i = 0; i < 4; i++) st[i] = rebase(st[i], fmaxf(st[i].m, acc[i] * kLog2e));
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float y = fmaf(acc[i], kLog2e, -st[i].m), e = __builtin_amdgcn_exp2f(y);
      st[i].l += e;
      st[i].t = fmaf(e, y, st[i].t);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    Stat s = st[i];
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) s = join(s, {shfl_xor_f(s.m, o), shfl_xor_f(s.l, o), shfl_xor_f(s.t, o)});
    if (lr == 0) s_state[wave][0][4 * lg + i] = s.m, s_state[wave][1][4 * lg + i] = s.l, s_state[wave][2][4 * lg + i] = s.t;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < NT; c += kThreads) {
    Stat s{s_state[0][0][c], s_state[0][1][c], s_state[0][2][c]};
#pragma unroll
    for (int w = 1; w < kWaves; w++) s = join(s, {s_state[w][0][c], s_state[w][1][c], s_state[w][2][c]});
    float *p = a.part + (long long)n * a.segs * 3 * NT + c;
    p[0] = s.m, p[NT] = s.l, p[2 * NT] = s.t;
  }
}

// One wave a token: the runs that met its tile, put together in a fixed order.
__global__ __launch_bounds__(64) void head_merge_kernel(const HeadArgs a, int NT) {
  const int tok = blockIdx.x, l = lane_id(), tile = tok / NT;
  const long long units = ((a.V >> 4) + a.unit - 1) / a.unit, line = units * a.tiles, lo = tile * units, hi = lo + units;
  Stat s{kStart, 0.0f, 0.0f};
  if (a.tiles == 1) {  // (every run)
    const float *q = a.part + tok;
    const long long step = (long long)a.segs * 3 * NT;
#pragma unroll 4
    for (int n = l; n < a.parts; n += 64) s = join(s, {q[n * step], q[n * step + NT], q[n * step + 2 * NT]});
  } else {
    int n0 = (int)(lo * a.parts / line);  // the first run that ends past lo
    while (line * (n0 + 1) / a.parts <= lo) n0++;
    while (n0 > 0 && line * n0 / a.parts > lo) n0--;
    for (int n = n0 + l; n < a.parts; n += 64) {
      const long long from = line * n / a.parts, to = line * (n + 1) / a.parts;
      if (from >= hi) break;
      if (to <= from) continue;
      const float *q = a.part + ((long long)n * a.segs + tile - (int)(from / units)) * 3 * NT + tok % NT;
      s = join(s, {q[0], q[NT], q[2 * NT]});
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) s = join(s, {shfl_xor_f(s.m, o), shfl_xor_f(s.l, o), shfl_xor_f(s.t, o)});
  if (l) return;
  constexpr double kLn2 = 0.693147180559945309, kLog2 = (double)kLog2e;  // (log2 e as the states were formed with it)
  const double log_l = log2((double)s.l);
  // NaN (or +inf) among the logits leaves l NaN, -inf leaves t NaN; past kFar a reference's rounding is many powers of two
  const bool nan = !(s.l > 0x1p-20f && s.t == s.t && fabsf(s.m) <= kFar);
  const int v = a.tokens[tok];
  const bool in = v >= 0 && v < a.V;
  a.lse[tok] = nan ? __builtin_nanf("") : (float)(((double)s.m + log_l) * kLn2);
  a.entropy[tok] = nan ? __builtin_nanf("") : (float)(fmax(log_l - (double)s.t / (double)s.l, 0.0) * kLn2);
  // (not above 0, where the rounding of l would put a token that has nearly everything)
  a.logprob[tok] = !in ? 0.0f : nan ? __builtin_nanf("") : (float)fmin(((double)a.picked[tok] * kLog2 - (double)s.m - log_l) * kLn2, 0.0);
}

// Token tiles of a launch: 32 TT tokens each, TT as even as they come, so many that the last workgroup ends first.
// (Always the largest tiles, runs of any number of blocks: 500 rows x 2,000 x 512 58 us, x 20,000 x 1,024 66, x 40,000 x
// 2,048 135, 200 rows x 40,000 x 2,048 95, 129 x 151,936 x 2,048 176; so 17, 49, 128, 74, 167.)
// What 16 blocks of a tile of 1 .. 4 cost, relative to each other, as first measured.  Now 16 blocks of a workgroup take 13.5,
// 20.6, 28.2 and 38.9 us (384 rows x 262,144 x 2,048 in tiles of each kind: 647, 494, 452, 467 us), as 43 : 66 : 90 : 124.
constexpr int kHalfCost[kMaxTT] = {43, 63, 95, 103};
struct Shape {
  bool few, mid;  // up to 16 rows that fit LDS; one tile of up to 96
  int tt, tile, tiles, parts, segs, T16, G32, unit = kUnit;
  long long part_at, picked_at, bytes;
};
Shape shape_of(long long T, int K, int V) {
  Shape s;
  const int blocks = V / 16;
  s.G32 = (K / 64 + 31) / 32 * 32;
  s.mid = mid_tile(T, K) > 0;
  s.few = T <= 16 && 32LL * K <= kFewBytes;
  if (s.few) {
    s.tt = 0;
    s.tile = 16;
    s.tiles = s.segs = 1;
    s.parts = (blocks + kWaves - 1) / kWaves < 256 ? (blocks + kWaves - 1) / kWaves : 256;
    s.T16 = 0;  // (their sums stay in LDS)
  } else if (s.mid) {
    s.tt = 0;
    s.tile = mid_tile(T, K);
    s.tiles = s.segs = 1;
    s.parts = mid_parts(V);
    s.T16 = 0;
  } else {
    const long long n32 = (T + 31) / 32, halves = (blocks + kUnit / 2 - 1) / (kUnit / 2);
    long long best = 0;
    for (int most = kMaxTT; most > 0; most--) {
      const long long tiles = (n32 + most - 1) / most;
      const int tt = tiles ? (int)((n32 + tiles - 1) / tiles) : 1;
      const long long cost = (tiles * halves + 255) / 256 * kHalfCost[tt - 1];
      if (most < kMaxTT && cost >= best) continue;
      best = cost;
      s.tiles = (int)tiles;
      s.tt = tt;
    }
    s.tile = 32 * s.tt;
    const long long whole = s.tiles * (long long)((blocks + kUnit - 1) / kUnit);
    s.unit = s.tiles * halves > 256 && whole <= 256 ? kUnit : kUnit / 2;  // (whole walks where each has a workgroup)
    const long long line = s.tiles * (long long)((blocks + s.unit - 1) / s.unit);
    s.parts = line < 256 ? (int)(line < 1 ? 1 : line) : 256;
    s.segs = s.tiles / s.parts + 2;
    s.T16 = s.tiles * s.tile;
  }
  s.part_at = ((long long)3 * s.T16 * s.G32 * 2 + 15) / 16 * 16;
  s.picked_at = s.part_at + 4LL * 3 * s.parts * s.segs * s.tile;
  s.bytes = s.picked_at + 4 * T;
  return s;
}

template <int RING>
int launch_few(const HeadArgs &a, hipStream_t st) {
  static const bool wide = [] {  // (more than the static limit)
    (void)hipFuncSetAttribute((const void *)&head_few_kernel<RING>, hipFuncAttributeMaxDynamicSharedMemorySize,
                              kFewBytes + 3 * 16 * 32 * kFewChunks * 2);
    return true;
  }();
  (void)wide;
  head_few_kernel<RING><<<a.parts, kThreads, (size_t)16 * (2 * a.K + 6 * a.G32), st>>>(a);
  return jit::check_launch("jit_head_logprobs");
}

template <int TT>
int launch_tile(const HeadArgs &a, hipStream_t st) {
  constexpr int lds = Lds<TT>::kBytes;
  static const bool wide = [] {  // (more than the static limit)
    (void)hipFuncSetAttribute((const void *)&head_tile_kernel<TT>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    return true;
  }();
  (void)wide;
  head_tile_kernel<TT><<<(a.parts + 7) / 8 * 8, kThreads, lds, st>>>(a);
  return jit::check_launch("jit_head_logprobs");
}

}  // namespace

extern "C" long long jit_head_logprobs_workspace_bytes(int T, int K, int V) {
  if (T < 0 || K <= 0 || V <= 0) return -1;
  return shape_of(T, K, V).bytes;
}

extern "C" int jit_head_logprobs(const uint16_t *x, int T, int K, const void *w, int V, const int32_t *tokens,
                                 float *logprob, float *entropy, float *lse, void *workspace, long long workspace_bytes,
                                 void *stream) {
  if (T < 0 || K <= 0 || V <= 0) return jit::fail(JIT_EINVAL, "head_logprobs: bad dims T=%d K=%d V=%d", T, K, V);
  if (K % 128 != 0 || V % 16 != 0)
    return jit::fail(JIT_EUNSUPPORTED, "head_logprobs covers K %% 128 == 0 and V %% 16 == 0, got K=%d V=%d", K, V);
  // (a 16-row block's bytes, K / 128 tiles of 1,152, are offsets of 32 bits)
  if (T > (1 << 20) || K > (1 << 24) || (long long)T * K > 0x7fffffffLL)
    return jit::fail(JIT_EUNSUPPORTED, "head_logprobs covers up to 2^20 rows of up to 2^24 and 2^31 - 1 values of x, got %d x %d", T, K);
  if (T == 0) return JIT_OK;
  if (!x || !w || !tokens || !logprob || !entropy || !lse) return jit::fail(JIT_EINVAL, "head_logprobs: null pointer");
  if (((uintptr_t)x | (uintptr_t)w) & 15) return jit::fail(JIT_EINVAL, "head_logprobs: x and the head must be 16-byte aligned");
  const Shape s = shape_of(T, K, V);
  if (!workspace || workspace_bytes < s.bytes || ((uintptr_t)workspace & 15))
    return jit::fail(JIT_EINVAL, "head_logprobs: a workspace of %lld bytes, 16-byte aligned, is needed", s.bytes);
  uint8_t *ws = (uint8_t *)workspace;
  HeadArgs a{x, (const uint8_t *)w, tokens, (uint16_t *)ws, (float *)(ws + s.part_at), (float *)(ws + s.picked_at),
             logprob, entropy, lse, T, K, V, s.parts, s.segs, s.tiles, s.T16, s.G32, s.unit};
  const hipStream_t st = (hipStream_t)stream;
  int rc;
  if (s.few) {
    // (1 row of 151,936 x 2,048 takes 43 us in a graph with 16 in flight and 49 with 8, x 1,024 33 and 29, x 4,096 80 and 82)
    rc = K % 2048 == 0 ? launch_few<16>(a, st) : launch_few<8>(a, st);
  } else if (s.mid) {
    rc = launch_mid(a, st);
  } else {
    head_xsum_kernel<<<dim3(s.T16, s.G32 / 32), 64, 0, st>>>(x, T, K, s.T16, s.G32, (uint16_t *)ws);
    if ((rc = jit::check_launch("jit_head_logprobs (sums)")) != JIT_OK) return rc;
    switch (s.tt) {
      case 1: rc = launch_tile<1>(a, st); break;
      case 2: rc = launch_tile<2>(a, st); break;
      case 3: rc = launch_tile<3>(a, st); break;
      default: rc = launch_tile<4>(a, st); break;
    }
  }
  if (rc != JIT_OK) return rc;
  head_merge_kernel<<<T, 64, 0, st>>>(a, s.tile);
  return jit::check_launch("jit_head_logprobs (merge)");
}
