// Attention over the 8-bit KV cache for gfx950: single tokens (split over the keys) and causal prompt chunks.
// Records and number format: kv8.hpp.
//
// Scores are formed from the codes, K_codes . Q^T in bf16 matrix instructions (codes and q are exact there), and
// take their key's scale afterwards; V's codes meet the probabilities in fp16 instructions (codes are exact, a
// probability keeps 11 bits, 8 times what bf16 would, at half the instructions of a bf16 high and low part).
#include "kv8.hpp"

namespace {

using namespace kv8;

constexpr float kLowest = -1e30f;  // the running maximum before any key: finite, so that rows without a key stay 0
// Probabilities are formed 2^15 times too large: fp16 then keeps 11 bits of those down to 2^-29 of a row's largest,
// and the factor cancels in the division by their sum.
constexpr float kPShift = 15.0f;

// ---------------------------------------------------------------- single tokens
// A sequence is cut into chunks by its own length alone, a chunk into 4 runs of a wave each.
constexpr int kSplits = 4;
constexpr int kChunk = 512, kLongChunks = 128, kChunkMax = 64 * kPage * kSplits;

__host__ __device__ __forceinline__ int chunk_tokens(int len) {
  if (len <= kChunk * kLongChunks) return kChunk;
  constexpr int kStep = 32 * kSplits;
  const long long c = (((long long)len + kLongChunks - 1) / kLongChunks + kStep - 1) / kStep * kStep;
  return c < kChunkMax ? (int)c : kChunkMax;
}
__host__ __device__ __forceinline__ int chunks_of(int len) {
  const int ck = chunk_tokens(len);
  return (int)(((long long)len + ck - 1) / ck);
}
// the most chunks of any length up to max_len
int max_chunks(int max_len) {
  if (max_len <= kChunk * kLongChunks) return chunks_of(max_len);
  const int n = (int)(((long long)max_len + kChunkMax - 1) / kChunkMax);
  return n > kLongChunks ? n : kLongChunks;
}

struct DecodeArgs {
  const uint16_t *q;
  const uint8_t *pool;
  const int32_t *page_table, *lens;
  float *part_o;   // [B][ncap][H][128]
  float *part_ml;  // [B][ncap][H][2]
  uint16_t *out;
  int num_pages, max_pages, B, H, Hkv, G, max_len, ncap;
  float qk_scale;  // scale * log2(e)
};

__device__ __forceinline__ int seq_len(const DecodeArgs &a, int b) {
  const long long most = (long long)a.max_pages * kPage;
  int L = max(a.lens[b], 0);
  L = min(L, a.max_len);
  return L > most ? (int)most : L;
}

constexpr int kStateFloats = 32 + 2;  // o[8][4], max, sum per lane

__global__ __launch_bounds__(64 * kSplits) void kv8_decode_kernel(const DecodeArgs a) {
  __shared__ float xstate[kSplits - 1][kStateFloats][64];
  // Workgroups go to the 8 XCDs in turn, so chunk c of sequence b runs on XCD (c odd + b) % 8: a long sequence's chunks
  // spread over all of them.  (With B itself in odd's place, B = 32 kept each sequence on one XCD: 32 sequences of 128
  // to 32,768 keys 105 us, now 32.)
  const int odd = a.B | 1, b = blockIdx.x % odd, c = blockIdx.x / odd, kvh = blockIdx.y;
  if (b >= a.B) return;
  const int split = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id();
  const int lr = l & 15, lg = l >> 4, G = a.G;
  const int L = seq_len(a, b), ck = chunk_tokens(L), n = chunks_of(L);
  const long long row = (long long)b * a.H + kvh * G + lr;  // this lane's q head
  if (c >= n) {
    if (c == 0 && split == 0 && lr < G) {  // no keys: zeros
#pragma unroll
      for (int cc = 0; cc < 8; cc++) *(uint2 *)(a.out + row * kD + 16 * cc + 4 * lg) = make_uint2(0u, 0u);
    }
    return;
  }
  const int run = ck / kSplits, k_begin = c * ck + split * run, k_end = min(k_begin + run, L);
  const int npg = k_end > k_begin ? (k_end - k_begin + kPage - 1) / kPage : 0;
  // the run's page ids, one per lane; a page outside the pool has its keys left out
  int my_page = l < npg ? a.page_table[(long long)b * a.max_pages + k_begin / kPage + l] : 0;
  const bool bad = my_page < 0 || my_page >= a.num_pages;
  const unsigned long long bad_pages = __ballot(bad);
  if (bad) my_page = 0;

  FragH qf[4];  // (bf16) Q^T: q head lr, dims 64 (f / 2) + 16 lg + 8 (f % 2) ..
#pragma unroll
  for (int f = 0; f < 4; f++)
    qf[f].q = lr < G ? *(const uint4 *)(a.q + row * kD + 64 * (f >> 1) + 16 * lg + 8 * (f & 1)) : make_uint4(0, 0, 0, 0);

  float m_run = kLowest, l_run = 0.0f;
  f32x4 o[8];
#pragma unroll
  for (int cc = 0; cc < 8; cc++) o[cc] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int st = 0; 2 * st < npg; st++) {
    const int k0 = k_begin + 32 * st;
    uint4 kc[2][2], vc[2][2];
    float4 ks[2], vs[2];
#pragma unroll
    for (int p = 0; p < 2; p++) {
      const int i = min(2 * st + p, npg - 1);  // (a page past the run: the last one again, its keys masked)
      const uint8_t *rec = record(a.pool, __builtin_amdgcn_readlane(my_page, i), a.Hkv, kvh);
#pragma unroll
      for (int i2 = 0; i2 < 2; i2++) {
        kc[p][i2] = ld_stream16(rec + 1024 * i2 + 16 * l);
        vc[p][i2] = ld_stream16(rec + kVOff + 1024 * i2 + 16 * l);
      }
      ks[p] = *(const float4 *)(rec + kScaleOff + 16 * lg);
      vs[p] = *(const float4 *)(rec + kScaleOff + 4 * kPage + 16 * lg);
    }
    // keys of this step that count: below k_end, of pages in the pool (lane: 4 of each page)
    int keep[2];
#pragma unroll
    for (int p = 0; p < 2; p++)
      keep[p] = (bad_pages >> min(2 * st + p, 63)) & 1 ? 0 : k_end - (k0 + 16 * p + 4 * lg);
    float t[2][4], iv[2][4];
#pragma unroll
    for (int p = 0; p < 2; p++) {
      f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int f = 0; f < 4; f++) {
        Frag8 kf, qq;
        const uint32_t w0 = (f & 1) ? kc[p][f >> 1].z : kc[p][f >> 1].x, w1 = (f & 1) ? kc[p][f >> 1].w : kc[p][f >> 1].y;
        to_bf16(w0, 1.0f, kf.u[0], kf.u[1]);
        to_bf16(w1, 1.0f, kf.u[2], kf.u[3]);
        qq.q = qf[f].q;
        s = mfma16x16x32(kf, qq, s);
      }
      const float *ksp = (const float *)&ks[p], *vsp = (const float *)&vs[p];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        // V's scale 2^e is part of the exponent, so a row's maximum is that of its contributions; the sum of the
        // probabilities themselves takes 2^-e back out (a scale of 0, a slot never written, as 2^-100)
        const uint32_t vb = i < keep[p] ? max(__float_as_uint(vsp[i]), (uint32_t)(kMinExp + 127) << 23) : 127u << 23;
        const float ev = (float)((int)(vb >> 23) - 127);
        iv[p][i] = __uint_as_float((254u << 23) - vb);
        t[p][i] = i < keep[p] ? fmaf(s[i], ksp[i] * a.qk_scale, ev) : -INFINITY;
      }
    }
    float tmax = fmaxf(t[0][0], t[1][0]);
#pragma unroll
    for (int i = 1; i < 4; i++) tmax = fmaxf(tmax, fmaxf(t[0][i], t[1][i]));
    tmax = max_xor32(max_xor16(tmax));
    const float m_new = fmaxf(m_run, tmax), alpha = __builtin_amdgcn_exp2f(m_run - m_new);
    float psum = 0.0f;
#pragma unroll
    for (int p = 0; p < 2; p++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        t[p][i] = __builtin_amdgcn_exp2f(t[p][i] - (m_new - kPShift));
        psum = fmaf(t[p][i], iv[p][i], psum);
      }
    l_run = fmaf(l_run, alpha, psum);
    m_run = m_new;
    FragH pf;
    pf.u[0] = pack_f16x2(t[0][0], t[0][1]);
    pf.u[1] = pack_f16x2(t[0][2], t[0][3]);
    pf.u[2] = pack_f16x2(t[1][0], t[1][1]);
    pf.u[3] = pack_f16x2(t[1][2], t[1][3]);
    const uint32_t km[2] = {keep_bytes(keep[0]), keep_bytes(keep[1])};  // (a p of 0 does not cancel a NaN code)
#pragma unroll
    for (int cc = 0; cc < 8; cc++) {
      FragH vf;
#pragma unroll
      for (int p = 0; p < 2; p++) to_f16(((const uint32_t *)&vc[p][cc >> 2])[cc & 3] & km[p], vf.u[2 * p], vf.u[2 * p + 1]);
#pragma unroll
      for (int i = 0; i < 4; i++) o[cc][i] *= alpha;
      o[cc] = mfma16x16x32_f16(vf, pf, o[cc]);
    }
  }
  // the runs' states meet in run order
  if (split > 0) {
    float(*st)[64] = xstate[split - 1];
#pragma unroll
    for (int cc = 0; cc < 8; cc++)
#pragma unroll
      for (int i = 0; i < 4; i++) st[4 * cc + i][l] = o[cc][i];
    st[32][l] = m_run;
    st[33][l] = l_run;
  }
  __syncthreads();
  if (split > 0) return;
#pragma unroll
  for (int sp = 1; sp < kSplits; sp++) {
    float(*st)[64] = xstate[sp - 1];
    const float m2 = st[32][l], M = fmaxf(m_run, m2);
    const float f0 = exp2f(m_run - M), f1 = exp2f(m2 - M);
#pragma unroll
    for (int cc = 0; cc < 8; cc++)
#pragma unroll
      for (int i = 0; i < 4; i++) o[cc][i] = fmaf(o[cc][i], f0, st[4 * cc + i][l] * f1);
    l_run = fmaf(l_run, f0, st[33][l] * f1);
    m_run = M;
  }
  const float l_tot = sum_xor32(sum_xor16(l_run));
  if (lr >= G) return;
  if (n == 1) {
    const float inv = l_tot == 0.0f ? 0.0f : 1.0f / l_tot;
#pragma unroll
    for (int cc = 0; cc < 8; cc++) {
      uint2 w;
      w.x = pack_bf16x2(o[cc][0] * inv, o[cc][1] * inv);
      w.y = pack_bf16x2(o[cc][2] * inv, o[cc][3] * inv);
      *(uint2 *)(a.out + row * kD + 16 * cc + 4 * lg) = w;
    }
    return;
  }
  const long long r = ((long long)b * a.ncap + c) * a.H + kvh * G + lr;
#pragma unroll
  for (int cc = 0; cc < 8; cc++)
    *(float4 *)(a.part_o + r * kD + 16 * cc + 4 * lg) = make_float4(o[cc][0], o[cc][1], o[cc][2], o[cc][3]);
  if (lg == 0) *(float2 *)(a.part_ml + 2 * r) = make_float2(m_run, l_tot);
}

// The chunks of a (sequence, q head), in order: thread = chunk lane (16) x 4 dims; lane j takes chunks j, j + 16, ..
constexpr int kMergeLanes = 16;

__global__ __launch_bounds__(32 * kMergeLanes) void kv8_merge_kernel(const DecodeArgs a) {
  const int b = blockIdx.x, h = blockIdx.y, t = threadIdx.x, n = chunks_of(seq_len(a, b));
  if (n <= 1) return;
  __shared__ float4 s_o[kMergeLanes][32];
  __shared__ float s_m[kMergeLanes], s_l[kMergeLanes];
  const int cl = t >> 5, dq = t & 31;
  float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
  float m_run = kLowest, ls = 0.0f;
  for (int c = cl; c < n; c += kMergeLanes) {
    const long long r = ((long long)b * a.ncap + c) * a.H + h;
    const float2 ml = *(const float2 *)(a.part_ml + 2 * r);
    const float4 o = *(const float4 *)(a.part_o + r * kD + 4 * dq);
    const float M = fmaxf(m_run, ml.x), fa = exp2f(m_run - M), fb = exp2f(ml.x - M);
    ls = fmaf(ls, fa, ml.y * fb);
    O.x = fmaf(O.x, fa, o.x * fb);
    O.y = fmaf(O.y, fa, o.y * fb);
    O.z = fmaf(O.z, fa, o.z * fb);
    O.w = fmaf(O.w, fa, o.w * fb);
    m_run = M;
  }
  s_o[cl][dq] = O;
  if (dq == 0) s_m[cl] = m_run, s_l[cl] = ls;
  __syncthreads();
  if (t >= 32) return;
  float M = s_m[0];
  for (int j = 1; j < kMergeLanes; j++) M = fmaxf(M, s_m[j]);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float l_tot = 0.0f;
  for (int j = 0; j < kMergeLanes; j++) {
    const float f = exp2f(s_m[j] - M);
    const float4 v = s_o[j][t];
    acc.x = fmaf(v.x, f, acc.x);
    acc.y = fmaf(v.y, f, acc.y);
    acc.z = fmaf(v.z, f, acc.z);
    acc.w = fmaf(v.w, f, acc.w);
    l_tot = fmaf(s_l[j], f, l_tot);
  }
  const float inv = l_tot == 0.0f ? 0.0f : 1.0f / l_tot;
  uint2 w;
  w.x = pack_bf16x2(acc.x * inv, acc.y * inv);
  w.y = pack_bf16x2(acc.z * inv, acc.w * inv);
  *(uint2 *)(a.out + ((long long)b * a.H + h) * kD + 4 * t) = w;
}

// ---------------------------------------------------------------- causal prompt chunks
// A workgroup owns WAVES x TILES q tiles of 16 rows (16 / G tokens x the G q heads of a kv head) and walks the keys up
// to its last token 128 a step.  A step's codes become bf16 keys (times their scales) and fp16 values in LDS once,
// for all of the workgroup's rows.
constexpr int kPfWaves = 8, kPfTiles = 2;  // a row block (jit_prefill_block_tokens)
constexpr int kStepKeys = 128, kStepPages = kStepKeys / kPage;
constexpr int kPartKeys = 6144;            // key parts (jit_prefill_part_keys)
constexpr int kPartSteps = kPartKeys / kStepKeys;
constexpr int kPfSlot = kD + 4;            // floats of a (token, part, head) partial: o, max, sum, 2 pad
// Values are held in LDS relative to the loudest scale so far, 2^E, times 2^7 (448 x 2^7 < 65,504): a value of a token
// 2^22 times quieter than that still has all its bits.
constexpr int kVShift = 7;

struct PrefillArgs {
  const uint16_t *q;
  const uint8_t *pool;
  const int32_t *page_table;
  const int32_t *blk_chunk, *blk_q0, *blk_part;
  const int32_t *chunk_seq, *chunk_ctx, *chunk_len, *chunk_row;
  uint16_t *out;
  float *part;
  int num_pages, max_pages, H, Hkv, G, pmax;
  float qk_scale;
};

template <int WAVES, int TILES>
__global__ __launch_bounds__(64 * WAVES) void kv8_prefill_kernel(const PrefillArgs a) {
  constexpr int kSub = kPfWaves * kPfTiles / (WAVES * TILES);  // workgroups a row block
  __shared__ __attribute__((aligned(16))) uint4 s_k[kStepPages * 4 * 64];  // [page][fragment][lane] 8 bf16
  __shared__ __attribute__((aligned(16))) uint4 s_v[kStepPages / 2 * 8 * 64];  // [page pair][16 dims][lane] 8 fp16
  const int item = blockIdx.x / (kSub * a.Hkv), kvh = blockIdx.x % a.Hkv;
  const int ch = a.blk_chunk[item], part = a.blk_part[item];
  const int seq = a.chunk_seq[ch], ctx = a.chunk_ctx[ch], len = a.chunk_len[ch], row0 = a.chunk_row[ch];
  const int G = a.G, TR = 16 / G, tpw = TILES * TR;
  int q0 = a.blk_q0[item];
  if constexpr (kSub > 1) q0 += blockIdx.x / a.Hkv % kSub * WAVES * tpw;
  if (q0 >= len) return;  // (uniform)
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id();
  const int lr = l & 15, lg = l >> 4;
  const int kend = ctx + min(q0 + WAVES * tpw, len);  // the workgroup's keys: [0, kend)
  const int nst = (kend + kStepKeys - 1) / kStepKeys, npages = min((kend + kPage - 1) / kPage, a.max_pages);
  const int st0 = part * kPartSteps, st1 = min(nst, st0 + kPartSteps);
  if (st0 >= st1) return;  // (uniform: a piece of a block whose last token alone reaches the part)
  const int32_t *prow = a.page_table + (long long)seq * a.max_pages;

  int tok[TILES];
  bool store[TILES];
  Frag8 qf[TILES][4];
  float m_run[TILES], l_run[TILES];
  f32x4 o[TILES][8];
#pragma unroll
  for (int j = 0; j < TILES; j++) {
    const int t = q0 + wave * tpw + j * TR + lr / G;
    store[j] = t < len;
    tok[j] = min(t, len - 1);
    const uint16_t *qp = a.q + ((long long)(row0 + tok[j]) * a.H + kvh * G + lr % G) * kD + 16 * lg;
#pragma unroll
    for (int f = 0; f < 4; f++) qf[j][f].q = *(const uint4 *)(qp + 64 * (f >> 1) + 8 * (f & 1));
    m_run[j] = kLowest;
    l_run[j] = 0.0f;
#pragma unroll
    for (int cc = 0; cc < 8; cc++) o[j][cc] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  int e_run = kMinExp;  // the exponent of the loudest value so far
  for (int st = st0; st < st1; st++) {
    const int k0 = kStepKeys * st;
    // the step's page ids (lane i: page i % 8) and which of them lie outside the pool
    int my_page = prow[min(kStepPages * st + (l & (kStepPages - 1)), npages - 1)];
    const bool bad = my_page < 0 || my_page >= a.num_pages;
    const uint32_t bad_pages = (uint32_t)__ballot(bad) & 0xffu;
    if (bad) my_page = 0;
    // the loudest live value of the step: lane i's keys 2 i, 2 i + 1
    int e_step = kMinExp;
    {
      const int p = l >> 3;
      const uint8_t *rec = record(a.pool, __shfl(my_page, p, 64), a.Hkv, kvh);
      const float2 s2 = *(const float2 *)(rec + kScaleOff + 4 * kPage + 8 * (l & 7));
      if (!((bad_pages >> p) & 1)) {
        if (k0 + 2 * l < kend) e_step = max(e_step, (int)(__float_as_uint(s2.x) >> 23) - 127);
        if (k0 + 2 * l + 1 < kend) e_step = max(e_step, (int)(__float_as_uint(s2.y) >> 23) - 127);
      }
#pragma unroll
      for (int x = 1; x < 64; x <<= 1) e_step = max(e_step, __shfl_xor(e_step, x, 64));
    }
    const int e_new = max(e_run, min(e_step, kMaxExp));
    const float e_alpha = e_new - e_run > 126 ? 0.0f : exp_bits(e_run - e_new);
    e_run = e_new;
    __syncthreads();  // (the previous step's reads are done)
    for (int u = wave; u < kStepPages; u += WAVES) {  // keys: page u
      const uint8_t *rec = record(a.pool, __builtin_amdgcn_readlane(my_page, u), a.Hkv, kvh);
      const float s = *(const float *)(rec + kScaleOff + 4 * lr);
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const uint4 w = *(const uint4 *)(rec + 1024 * i + 16 * l);
        uint4 f0, f1;
        to_bf16(w.x, s, f0.x, f0.y);
        to_bf16(w.y, s, f0.z, f0.w);
        to_bf16(w.z, s, f1.x, f1.y);
        to_bf16(w.w, s, f1.z, f1.w);
        s_k[(u * 4 + 2 * i) * 64 + l] = f0;
        s_k[(u * 4 + 2 * i + 1) * 64 + l] = f1;
      }
    }
    for (int u = wave; u < kStepPages; u += WAVES) {  // values: page pair u / 2, dims 64 (u % 2) ..
      const int h = u >> 1, qd = u & 1;
      uint32_t w[2][4];
      f16x2_t fac[2][2];
#pragma unroll
      for (int p = 0; p < 2; p++) {
        const uint8_t *rec = record(a.pool, __builtin_amdgcn_readlane(my_page, 2 * h + p), a.Hkv, kvh);
        const uint4 v = *(const uint4 *)(rec + kVOff + 1024 * qd + 16 * l);
        const float4 s = *(const float4 *)(rec + kScaleOff + 4 * kPage + 16 * lg);
        const int keep = (bad_pages >> (2 * h + p)) & 1 ? 0 : kend - (k0 + 32 * h + 16 * p + 4 * lg);
        const uint32_t km = keep_bytes(keep);
        w[p][0] = v.x & km, w[p][1] = v.y & km, w[p][2] = v.z & km, w[p][3] = v.w & km;
        const float *sp = (const float *)&s;
#pragma unroll
        for (int i = 0; i < 4; i++) {  // 2^(e - E + 7) (below fp16's range: 0)
          const int e = i < keep ? (int)(__float_as_uint(sp[i]) >> 23) - 127 - e_run + kVShift : -100;
          fac[p][i >> 1][i & 1] = (_Float16)exp_bits(max(min(e, kVShift), -100));
        }
      }
#pragma unroll
      for (int c = 0; c < 4; c++) {
        uint32_t r[4];
#pragma unroll
        for (int p = 0; p < 2; p++) {
          to_f16(w[p][c], r[2 * p], r[2 * p + 1]);
#pragma unroll
          for (int i = 0; i < 2; i++)
            r[2 * p + i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, r[2 * p + i]) * fac[p][i]);
        }
        s_v[(h * 8 + 4 * qd + c) * 64 + l] = make_uint4(r[0], r[1], r[2], r[3]);
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < TILES; j++) {
      f32x4 sc[kStepPages];
      const int pos = ctx + tok[j];
      float tmax = -INFINITY;
#pragma unroll
      for (int p = 0; p < kStepPages; p++) {
        sc[p] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int f = 0; f < 4; f++) {
          Frag8 kf;
          kf.q = s_k[(p * 4 + f) * 64 + l];
          sc[p] = mfma16x16x32(kf, qf[j][f], sc[p]);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int key = k0 + 16 * p + 4 * lg + i;
          if (key > pos || ((bad_pages >> p) & 1)) sc[p][i] = -INFINITY;
          tmax = fmaxf(tmax, sc[p][i]);
        }
      }
      tmax = max_xor32(max_xor16(tmax)) * a.qk_scale;
      const float m_new = fmaxf(m_run[j], tmax), alpha = __builtin_amdgcn_exp2f(m_run[j] - m_new);
      float psum = 0.0f;
#pragma unroll
      for (int cc = 0; cc < 8; cc++)
#pragma unroll
        for (int i = 0; i < 4; i++) o[j][cc][i] *= alpha * e_alpha;
#pragma unroll
      for (int h = 0; h < kStepPages / 2; h++) {
        FragH pf;
#pragma unroll
        for (int p = 0; p < 2; p++) {
          float t[4];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            t[i] = __builtin_amdgcn_exp2f(fmaf(sc[2 * h + p][i], a.qk_scale, kPShift - m_new));
            psum += t[i];
          }
          pf.u[2 * p] = pack_f16x2(t[0], t[1]);
          pf.u[2 * p + 1] = pack_f16x2(t[2], t[3]);
        }
#pragma unroll
        for (int cc = 0; cc < 8; cc++) {
          FragH vf;
          vf.q = s_v[(h * 8 + cc) * 64 + l];
          o[j][cc] = mfma16x16x32_f16(vf, pf, o[j][cc]);
        }
      }
      l_run[j] = fmaf(l_run[j], alpha, psum);
      m_run[j] = m_new;
    }
  }
  const float unit = exp_bits(e_run - kVShift);
#pragma unroll
  for (int j = 0; j < TILES; j++) {
    const float l_tot = sum_xor32(sum_xor16(l_run[j]));
    if (!store[j]) continue;
    const int parts = (ctx + tok[j]) / kPartKeys + 1;
    if (part >= parts) continue;  // (a token before this part's keys: finished by its own last part)
    const long long hrow = (long long)(row0 + tok[j]) * a.H + kvh * G + lr % G;
    if (parts == 1) {
      const float inv = l_tot == 0.0f ? 0.0f : unit / l_tot;
#pragma unroll
      for (int cc = 0; cc < 8; cc++) {
        uint2 w;
        w.x = pack_bf16x2(o[j][cc][0] * inv, o[j][cc][1] * inv);
        w.y = pack_bf16x2(o[j][cc][2] * inv, o[j][cc][3] * inv);
        *(uint2 *)(a.out + hrow * kD + 16 * cc + 4 * lg) = w;
      }
    } else {
      float *ps = a.part + (((long long)(row0 + tok[j]) * a.pmax + part) * a.H + kvh * G + lr % G) * kPfSlot;
#pragma unroll
      for (int cc = 0; cc < 8; cc++)
        *(float4 *)(ps + 16 * cc + 4 * lg) =
            make_float4(o[j][cc][0] * unit, o[j][cc][1] * unit, o[j][cc][2] * unit, o[j][cc][3] * unit);
      if (lg == 0) *(float2 *)(ps + kD) = make_float2(m_run[j], l_tot);
    }
  }
}

// The parts of a token's keys in order: one workgroup of 8 H threads a token, thread (h, d) 16 dims of head h.
__global__ __launch_bounds__(512) void kv8_prefill_merge_kernel(const PrefillArgs a) {
  const int c = blockIdx.y, t = blockIdx.x;
  if (t >= a.chunk_len[c]) return;
  const int parts = (a.chunk_ctx[c] + t) / kPartKeys + 1;
  if (parts < 2) return;
  const long long row = a.chunk_row[c] + t;
  const int h = threadIdx.x >> 3, d0 = 16 * (threadIdx.x & 7);
  float M = kLowest, ls = 0.0f, O[16];
#pragma unroll
  for (int i = 0; i < 16; i++) O[i] = 0.0f;
  for (int p = 0; p < parts; p++) {
    const float *ps = a.part + ((row * a.pmax + p) * a.H + h) * kPfSlot;
    const float2 ml = *(const float2 *)(ps + kD);
    const float mn = fmaxf(M, ml.x), fa = exp2f(M - mn), fb = exp2f(ml.x - mn);
    ls = fmaf(ls, fa, ml.y * fb);
#pragma unroll
    for (int i = 0; i < 16; i++) O[i] = fmaf(O[i], fa, ps[d0 + i] * fb);
    M = mn;
  }
  const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; i++) w[i] = pack_bf16x2(O[2 * i] * inv, O[2 * i + 1] * inv);
  uint4 *op = (uint4 *)(a.out + (row * a.H + h) * kD + d0);
  op[0] = make_uint4(w[0], w[1], w[2], w[3]);
  op[1] = make_uint4(w[4], w[5], w[6], w[7]);
}

int64_t decode_bytes(int B, int H, int max_len) {
  const int n = max_chunks(max_len);
  return n > 1 ? (int64_t)B * n * H * (kD + 2) * (int64_t)sizeof(float) : 0;
}

}  // namespace

extern "C" int jit_kv8_chunk_tokens(int len) { return len < 1 ? kChunk : chunk_tokens(len); }

extern "C" int64_t jit_kv8_decode_workspace_bytes(int B, int H, int max_len) {
  if (B < 0 || H <= 0 || max_len < 0) return -1;
  return decode_bytes(B, H, max_len);
}

extern "C" int jit_paged_decode_attn_kv8(const uint16_t *q, const void *pool, int num_pages, const int32_t *page_table,
                                         int max_pages, const int32_t *lens, int B, int H, int Hkv, int max_len,
                                         float scale, void *workspace, int64_t workspace_bytes, uint16_t *out,
                                         void *stream) {
  if (B < 0 || H <= 0 || Hkv <= 0 || max_pages <= 0 || num_pages <= 0 || max_len < 0)
    return jit::fail(JIT_EINVAL, "paged_decode_attn_kv8: bad dims B=%d H=%d Hkv=%d max_pages=%d num_pages=%d max_len=%d", B,
                     H, Hkv, max_pages, num_pages, max_len);
  if (H % Hkv != 0) return jit::fail(JIT_EINVAL, "%d query heads do not share %d KV heads evenly", H, Hkv);
  if (H / Hkv > 16) return jit::fail(JIT_EUNSUPPORTED, "paged_decode_attn_kv8 covers H / Hkv <= 16, got %d", H / Hkv);
  if (Hkv > 65535 || H > 65535)
    return jit::fail(JIT_EUNSUPPORTED, "paged_decode_attn_kv8 covers up to 65535 heads, got %d", H);
  if (B == 0) return JIT_OK;
  const int most = (long long)max_pages * kPage < max_len ? max_pages * kPage : max_len;
  const int ncap = max_chunks(most) > 1 ? max_chunks(most) : 1;
  const int64_t need = decode_bytes(B, H, most);
  if (((int64_t)B | 1) * ncap > 0x7fffffff)
    return jit::fail(JIT_EUNSUPPORTED, "paged_decode_attn_kv8: %d sequences of up to %d chunks", B, ncap);
  if (workspace_bytes < need)
    return jit::fail(JIT_EINVAL, "paged_decode_attn_kv8: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                     (long long)need);
  if (!q || !pool || !page_table || !lens || !out || (need > 0 && !workspace))
    return jit::fail(JIT_EINVAL, "paged_decode_attn_kv8: null pointer");
  if (((uintptr_t)q | (uintptr_t)pool | (uintptr_t)out | (uintptr_t)workspace) & 15)
    return jit::fail(JIT_EINVAL, "paged_decode_attn_kv8: q, the pool, the workspace and out must be 16-byte aligned");
  float *part_o = (float *)workspace;
  const DecodeArgs a{q, (const uint8_t *)pool, page_table, lens, part_o, need ? part_o + (int64_t)B * ncap * H * kD : nullptr,
                     out, num_pages, max_pages, B, H, Hkv, H / Hkv, most, ncap, scale * 1.44269504088896341f};
  kv8_decode_kernel<<<dim3((unsigned)(B | 1) * ncap, Hkv), 64 * kSplits, 0, (hipStream_t)stream>>>(a);
  const int rc = jit::check_launch("jit_paged_decode_attn_kv8");
  if (rc || ncap == 1) return rc;
  kv8_merge_kernel<<<dim3(B, H), 32 * kMergeLanes, 0, (hipStream_t)stream>>>(a);
  return jit::check_launch("jit_paged_decode_attn_kv8");
}

extern "C" int jit_paged_prefill_attn_kv8(const uint16_t *q, const void *pool, int num_pages, const int32_t *page_table,
                                          int max_pages, const int32_t *chunk_seq, const int32_t *chunk_ctx,
                                          const int32_t *chunk_len, const int32_t *chunk_row, int C,
                                          const int32_t *blk_chunk, const int32_t *blk_q0, const int32_t *blk_part,
                                          int nblk, int pmax, int max_len, int H, int Hkv, float scale, void *workspace,
                                          uint16_t *out, void *stream) {
  if (C < 0 || nblk < 0 || H <= 0 || Hkv <= 0 || max_pages <= 0 || num_pages <= 0 || pmax < 1 || max_len < 0)
    return jit::fail(JIT_EINVAL, "paged_prefill_attn_kv8: bad dims C=%d nblk=%d H=%d Hkv=%d pmax=%d max_len=%d", C, nblk, H,
                     Hkv, pmax, max_len);
  if (H % Hkv != 0) return jit::fail(JIT_EINVAL, "%d query heads do not share %d KV heads evenly", H, Hkv);
  if (16 % (H / Hkv) != 0)
    return jit::fail(JIT_EUNSUPPORTED, "paged_prefill_attn_kv8 covers H / Hkv in {1, 2, 4, 8, 16}, got %d", H / Hkv);
  if (pmax > 1 && H > 64)
    return jit::fail(JIT_EUNSUPPORTED, "paged_prefill_attn_kv8 merges key parts of up to 64 query heads, got %d", H);
  if (C > 65535) return jit::fail(JIT_EUNSUPPORTED, "paged_prefill_attn_kv8 covers up to 65535 chunks, got %d", C);
  if (C == 0 || nblk == 0) return JIT_OK;
  if (!q || !pool || !page_table || !chunk_seq || !chunk_ctx || !chunk_len || !chunk_row || !blk_chunk || !blk_q0 ||
      !blk_part || !out || (pmax > 1 && !workspace))
    return jit::fail(JIT_EINVAL, "paged_prefill_attn_kv8: null pointer");
  if (((uintptr_t)q | (uintptr_t)pool | (uintptr_t)out | (uintptr_t)workspace) & 15)
    return jit::fail(JIT_EINVAL, "paged_prefill_attn_kv8: q, the pool, the workspace and out must be 16-byte aligned");
  const PrefillArgs a{q, (const uint8_t *)pool, page_table, blk_chunk, blk_q0, blk_part, chunk_seq, chunk_ctx, chunk_len,
                      chunk_row, out, (float *)workspace, num_pages, max_pages, H, Hkv, H / Hkv, pmax,
                      scale * 1.44269504088896341f};
  const hipStream_t st = (hipStream_t)stream;
  kv8_prefill_kernel<kPfWaves, kPfTiles><<<dim3(nblk * Hkv), 64 * kPfWaves, 0, st>>>(a);
  const int rc = jit::check_launch("jit_paged_prefill_attn_kv8");
  if (rc || pmax == 1 || max_len == 0) return rc;
  kv8_prefill_merge_kernel<<<dim3(max_len, C), 8 * H, 0, st>>>(a);
  return jit::check_launch("jit_paged_prefill_attn_kv8");
}
