// Scoring from hidden rows (score_head.hip) for one tile of 17 to 96 rows: every weight byte comes once, by the wave that
// needs it, and the rows of x go through LDS two pairs at a time.
//
// A workgroup of 8 waves, one a CU, has a run of 16-row blocks of the head and takes 8 NB of them a pass.  A wave's NB
// blocks keep their sums over all of K in registers (16 x 16 x 32 products, tokens on the rows, head rows on the columns:
// a lane's scale is its own row's), so biases, softmax and the meeting of lanes and waves come once a pass.  What bounds
// it: the head's bytes below some 50 rows, past that the issue of products and the sums behind them (a 16 x 16 x 32
// product holds the issue port for some 11 of its 16 cycles).  77 rows x 151,936 x 2,048 take 83 to 90 us (head_tile_kernel:
// 127), 17 rows x 4,096 86 us (122), 96 rows x 4,096 190 us (222), 32 rows x 2,048 49 us.  From 33 rows on 5 blocks a wave
// spill registers (7, 47, 93, 138 of them for 48, 64, 80, 96 rows), of 96 rows weights that were asked for ahead too.
#include "score_head.hpp"

namespace {

using namespace head;

constexpr int kPairs = 2;  // of a step
constexpr int kMaxK = 4096;

template <int STEP>
__device__ __forceinline__ float row_swap(float v) {  // mirrored in 16, in 8, then lanes l ^ 2 and l ^ 1
  constexpr int ctrl = STEP == 0 ? 0x140 : STEP == 1 ? 0x141 : STEP == 2 ? 0x4E : 0xB1;
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xF, 0xF, true));
}
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, row_swap<0>(v));
  v = fmaxf(v, row_swap<1>(v));
  v = fmaxf(v, row_swap<2>(v));
  return fmaxf(v, row_swap<3>(v));
}
// Sums over a row's 16 lanes of N values each: in every step a lane gives half of its values to its partner and takes the
// partner's other half; lane l ends with values N (l % 16) / 16 .. + N / 16 - 1.
template <int N, int STEP = 0>
__device__ __forceinline__ void row_scatter_sum(float *v) {
  if constexpr (STEP < 4) {
    constexpr int H = N / 2;
    const bool up = lane_id() >> (3 - STEP) & 1;
#pragma unroll
    for (int j = 0; j < H; j++) {
      const float keep = up ? v[j + H] : v[j], give = up ? v[j] : v[j + H];
      v[j] = keep + row_swap<STEP>(give);
    }
    row_scatter_sum<H, STEP + 1>(v);
  }
}

template <int T16, int NB>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void head_mid_kernel(const HeadArgs a) {
  constexpr int NT = 16 * T16, kPair = NT * 256, kStage = kPairs * kPair;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];  // two steps' rows, the groups' sums, the given tokens
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id(), lr = l & 15, lg = l >> 4;
  const int n = blockIdx.x, GP = a.K >> 7, steps = (GP + kPairs - 1) / kPairs, blocks = a.V >> 4;
  const int r0 = (int)((long long)blocks * n / a.parts), r1 = (int)((long long)blocks * (n + 1) / a.parts);
  const long long blk_bytes = (long long)GP * qtile::kTileBytes;
  uint32_t um = 0x00780078u, uc = 0x41804180u;
  asm volatile("" : "+v"(um), "+s"(uc));
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds);
  uint16_t *xs = (uint16_t *)(lds + 2 * kStage);  // [3][NT][G32]
  int *toks = (int *)(xs + 3 * NT * a.G32);       // [NT]

  // a wave's load j brings 4 rows of 256 bytes: number q = wave + 8 j is pair q / (4 T16), token tile q / 4 % T16, rows
  // 4 (q % 4) ..; row r's piece c sits in slot c ^ r % 16.  (Rows past T read the last row again, see head_tile_kernel.)
  const int srow = 4 * (wave & 3) + (l >> 4), spiece = (l & 15) ^ srow, cut = (a.T - 1) >> 4;
  const uint32_t xoff = (uint32_t)srow * (uint32_t)a.K * 2u + 16 * spiece;
  const uint32_t xoff_cut = (uint32_t)min(srow, a.T - 1 - 16 * cut) * (uint32_t)a.K * 2u + 16 * spiece;
  auto load_x = [&](int step, int stage) {
#pragma unroll
    for (int j = 0; j < T16; j++) {
      const int q = wave + 8 * j, pp = q / (4 * T16), t = q / 4 % T16;
      load_lds(a.x + (long long)(16 * min(t, cut)) * a.K + 128 * min(kPairs * step + pp, GP - 1), t < cut ? xoff : xoff_cut,
               __builtin_amdgcn_readfirstlane(lds0 + stage * kStage + q * 1024));
    }
  };
  uint4 wq[NB][kPairs];
  uint32_t ws[NB];  // the scales of row lr, pair lg % 2
  const int span = kWaves * NB, passes = (r1 - r0 + span - 1) / span;
  auto block = [&](int pass, int i) { return r0 + pass * span + i * kWaves + wave; };
  auto load_w = [&](int pass, int step, int i) {  // (past the run: the start of its last block again, for nothing)
    const int b = block(pass, i);
    const uint8_t *wp = a.w + min(b, r1 - 1) * blk_bytes;
    step = b < r1 ? step : 0;
#pragma unroll
    for (int pp = 0; pp < kPairs; pp++)
      wq[i][pp] = ld_stream16(wp + min(kPairs * step + pp, GP - 1) * qtile::kNibbleBytes + (uint32_t)(16 * l));
    ws[i] = *(const uint32_t *)(wp + (uint32_t)(GP * qtile::kNibbleBytes + min(kPairs * step + (lg & 1), GP - 1) * qtile::kScaleBytes + 8 * lr));
    asm volatile("" ::: "memory");  // (asked for here, a step ahead of its use)
  };

  load_x(0, 0);
#pragma unroll
  for (int i = 0; i < NB; i++) load_w(0, 0, i);
  for (int c = threadIdx.x; c < 3 * NT * a.G32 / 2; c += kThreads) ((uint32_t *)xs)[c] = 0u;
  for (int c = threadIdx.x; c < NT; c += kThreads) toks[c] = c < a.T ? a.tokens[c] : -1;
  __syncthreads();

  Stat total{kStart, 0.0f, 0.0f};  // thread c: token c
  int stage = 0;
  for (int pass = 0; pass < passes; pass++) {
    f32x4 acc[NB][T16];
#pragma unroll
    for (int i = 0; i < NB; i++)
#pragma unroll
      for (int t = 0; t < T16; t++) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int step = 0; step < steps; step++) {
      wait_loads<3 * NB>();  // x(step); this step's weights may be on their way
      bare_barrier();
      load_x(step + 1 < steps ? step + 1 : 0, stage ^ 1);
      const uint8_t *xst = lds + stage * kStage;
      auto rows = [&](auto i0_c, auto nb_c) {  // blocks i0 .. i0 + nb - 1 against the step's rows
        constexpr int I0 = decltype(i0_c)::value, N = decltype(nb_c)::value;
#pragma unroll
        for (int pp = 0; pp < kPairs; pp++) {
          if (kPairs * step + pp >= GP) break;  // (uniform)
          uint32_t su[N];
#pragma unroll
          for (int i = 0; i < N; i++) su[i] = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * (16 * pp + lr), (int)ws[I0 + i]);
#pragma unroll
          for (int g = 0; g < 2; g++) {
            const uint8_t *xp = xst + pp * kPair + lr * 256;
            const int pa = 8 * g + 2 * lg, o0 = 16 * (pa ^ lr), o1 = 16 * ((pa + 1) ^ lr);
            Frag8 wf[N][2], x[2][2];
            float s[N];
            x[0][0].q = *(const uint4 *)(xp + o0);
            x[0][1].q = *(const uint4 *)(xp + o1);
#pragma unroll
            for (int i = 0; i < N; i++) {
              const uint4 &q = wq[I0 + i][pp];
              wf[i][0] = unpack16(g ? q.z : q.x, um, uc);
              wf[i][1] = unpack16(g ? q.w : q.y, um, uc);
              s[i] = g ? bf2f_hi(su[i]) : bf2f(su[i] & 0xffffu);
            }
            f32x4 c[2][N];
#pragma unroll
            for (int t = 0; t <= T16; t++) {  // tile t's products beside tile t - 1's sums
              if (t + 1 < T16) {
                x[(t + 1) & 1][0].q = *(const uint4 *)(xp + (t + 1) * 4096 + o0);
                x[(t + 1) & 1][1].q = *(const uint4 *)(xp + (t + 1) * 4096 + o1);
              }
              if (t < T16) {
#pragma unroll
                for (int i = 0; i < N; i++) c[t & 1][i] = mfma16x16x32(x[t & 1][0], wf[i][0], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int i = 0; i < N; i++) c[t & 1][i] = mfma16x16x32(x[t & 1][1], wf[i][1], c[t & 1][i]);
              }
              if (t > 0) {
#pragma unroll
                for (int i = 0; i < N; i++)
#pragma unroll
                  for (int k = 0; k < 4; k++) acc[I0 + i][t - 1][k] = fmaf(s[i], c[(t - 1) & 1][i][k], acc[I0 + i][t - 1][k]);
              }
            }
          }
        }
        const bool more = step + 1 < steps;
#pragma unroll
        for (int i = 0; i < N; i++) load_w(more ? pass : pass + 1, more ? step + 1 : 0, I0 + i);
      };
      rows(std::integral_constant<int, 0>{}, std::integral_constant<int, 2>{});
      if constexpr (NB >= 4) rows(std::integral_constant<int, 2>{}, std::integral_constant<int, 2>{});
      if constexpr (NB % 2) rows(std::integral_constant<int, NB - 1>{}, std::integral_constant<int, 1>{});
      // the groups' sums of x in three bf16 pieces, a thread a token and group
      if (pass == 0 && threadIdx.x < 2 * kPairs * NT) {
        const int row = threadIdx.x / (2 * kPairs), gi = threadIdx.x % (2 * kPairs), grp = 2 * kPairs * step + gi;
        if (grp < 2 * GP) {
          float s = 0.0f;
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const uint4 q = *(const uint4 *)(xst + (gi >> 1) * kPair + row * 256 + 16 * ((8 * (gi & 1) + i) ^ (row & 15)));
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int j = 0; j < 4; j++) s += bf2f(w[j] & 0xffffu) + bf2f_hi(w[j]);
          }
#pragma unroll
          for (int i = 0; i < 3; i++) {
            const float v = bf2f(f2bf(s));
            xs[(i * NT + row) * a.G32 + grp] = (uint16_t)(__float_as_uint(v) >> 16);
            s -= v;
          }
        }
      }
      stage ^= 1;
    }
    // biases: sum_g (b - 16 s)_g X_g over 32 groups at a time, X in its three pieces, the smallest first
    for (int c0 = 0; c0 < a.G32 / 2; c0 += 16) {
    uint2 sb[NB][4];  // of pairs c0 + 4 lg .. + 3, all asked for at once
#pragma unroll
    for (int i = 0; i < NB; i++) {
      const uint8_t *sp = a.w + min(block(pass, i), r1 - 1) * blk_bytes + (long long)GP * qtile::kNibbleBytes;
#pragma unroll
      for (int j = 0; j < 4; j++) sb[i][j] = *(const uint2 *)(sp + (uint32_t)(min(c0 + 4 * lg + j, GP - 1) * qtile::kScaleBytes + 8 * lr));
    }
    if (!c0) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      bare_barrier();  // the sums are there, and the last step's rows have been read
    }
#pragma unroll
    for (int i = 0; i < NB; i++) {
      Frag8 fs, fb;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const bool in = c0 + 4 * lg + j < GP;
        fs.u[j] = in ? sb[i][j].x : 0u;
        fb.u[j] = in ? sb[i][j].y : 0u;
      }
#pragma unroll
      for (int t = 0; t < T16; t++) {
        f32x4 d = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 2; k >= 0; k--) {
          Frag8 x;
          x.q = *(const uint4 *)(xs + (k * NT + 16 * t + lr) * a.G32 + 2 * c0 + 8 * lg);
          d = mfma16x16x32(x, fs, d);
          acc[i][t] = mfma16x16x32(x, fb, acc[i][t]);
        }
#pragma unroll
        for (int k = 0; k < 4; k++) acc[i][t][k] = fmaf(-16.0f, d[k], acc[i][t][k]);
      }
    }
    }
#pragma unroll
    for (int i = 0; i < NB; i++)
      if (block(pass, i) >= r1) {
#pragma unroll
        for (int t = 0; t < T16; t++) acc[i][t] = f32x4{kDead, kDead, kDead, kDead};
      }
    // acc[i][t][k]: head row 16 block(pass, i) + lr, token 16 t + 4 lg + k.  The waves' states of the pass meet in the stage
    // that the last step has left.
    float *scratch = (float *)(lds + (stage ^ 1) * kStage);  // [kWaves][3][NT]
    constexpr int NV = 4 * T16, NP = (NV + 15) / 16 * 16, kOwn = NP / 16;
    float ls[NP], ts[NP];
#pragma unroll
    for (int t = 0; t < T16; t++) {
      const int4 tk = *(const int4 *)(toks + 16 * t + 4 * lg);
      const int v[4] = {tk.x, tk.y, tk.z, tk.w};
#pragma unroll
      for (int k = 0; k < 4; k++) {
        float x = acc[0][t][k];
#pragma unroll
        for (int i = 0; i < NB; i++) {
          if (v[k] == 16 * block(pass, i) + lr && block(pass, i) < r1) a.picked[16 * t + 4 * lg + k] = acc[i][t][k];
          x = fmaxf(x, acc[i][t][k]);
        }
        const float m = fmaxf(row_max(x) * kLog2e, kStart);
        float p = 0.0f, q = 0.0f;
#pragma unroll
        for (int i = 0; i < NB; i++) {
          const float y = fmaf(acc[i][t][k], kLog2e, -m), e = __builtin_amdgcn_exp2f(y);
          p += e;
          q = fmaf(e, y, q);
        }
        ls[4 * t + k] = p, ts[4 * t + k] = q;
        if (lr == (4 * t + k) / kOwn) scratch[wave * 3 * NT + 16 * t + 4 * lg + k] = m;
      }
    }
#pragma unroll
    for (int j = NV; j < NP; j++) ls[j] = ts[j] = 0.0f;
    row_scatter_sum<NP>(ls);
    row_scatter_sum<NP>(ts);
#pragma unroll
    for (int k = 0; k < kOwn; k++) {
      const int j = kOwn * lr + k;
      if (j < NV) {
        float *p = scratch + wave * 3 * NT + 16 * (j >> 2) + 4 * lg + (j & 3);
        p[NT] = ls[k], p[2 * NT] = ts[k];
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    bare_barrier();
    if (threadIdx.x < NT) {
#pragma unroll
      for (int w = 0; w < kWaves; w++) {
        const float *p = scratch + w * 3 * NT + threadIdx.x;
        const Stat s{p[0], p[NT], p[2 * NT]};
        total = join(total, s);
      }
    }
    // (the next step's barrier stands between these reads and the loads into that stage)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  wait_loads<0>();
  if (threadIdx.x < NT) {
    float *p = a.part + (long long)n * 3 * NT + threadIdx.x;
    p[0] = total.m, p[NT] = total.l, p[2 * NT] = total.t;
  }
}

template <int T16, int NB>
int launch(const HeadArgs &a, hipStream_t st) {
  constexpr int most = 16 * T16 * (4 * 256 + 6 * (kMaxK / 64) + 4);
  static_assert(most <= 160 * 1024, "gfx950 gives a workgroup at most 160 KB of LDS");
  static const bool wide = [] {  // (more than the static limit)
    (void)hipFuncSetAttribute((const void *)&head_mid_kernel<T16, NB>, hipFuncAttributeMaxDynamicSharedMemorySize, most);
    return true;
  }();
  (void)wide;
  head_mid_kernel<T16, NB><<<a.parts, kThreads, 16 * T16 * (4 * 256 + 6 * a.G32 + 4), st>>>(a);
  return jit::check_launch("jit_head_logprobs");
}

// The blocks of a wave and pass: as few passes as MOST blocks allow, then as few blocks as those passes need.  (Up to 5, 3 or
// 2 blocks a pass: 32 rows x 151,936 x 2,048 47, 56, 66 us; 64 rows 76 to 80, 94, 99; 96 rows 109 to 114, 116, 122 -- though
// 5 blocks of 64 rows and more spill registers.)
template <int T16, int MOST>
int launch_even(const HeadArgs &a, hipStream_t st) {
  const int most = (a.V / 16 + a.parts - 1) / a.parts, a_wave = (most + kWaves - 1) / kWaves;
  const int passes = (a_wave + MOST - 1) / MOST, nb = (a_wave + passes - 1) / passes;
  if constexpr (MOST >= 5)
    if (nb > 4) return launch<T16, 5>(a, st);
  if constexpr (MOST >= 4)
    if (nb > 3) return launch<T16, 4>(a, st);
  if (nb > 2) return launch<T16, 3>(a, st);
  return launch<T16, 2>(a, st);
}

}  // namespace

namespace head {

int mid_tile(long long T, int K) {
  if (T <= 16 || T > 96 || K > kMaxK) return 0;
  return (int)(T + 15) / 16 * 16;
}

int mid_parts(int V) { return V / 16 < 4 * 256 ? (V / 16 + 3) / 4 : 256; }

int launch_mid(const HeadArgs &a, hipStream_t st) {
  switch (mid_tile(a.T, a.K)) {
    case 32: return launch_even<2, 5>(a, st);
    case 48: return launch_even<3, 5>(a, st);
    case 64: return launch_even<4, 5>(a, st);
    case 80: return launch_even<5, 5>(a, st);
    default: return launch_even<6, 5>(a, st);
  }
}

}  // namespace head
