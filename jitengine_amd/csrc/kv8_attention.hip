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
// A workgroup owns WAVES x 32 rows (32 / G tokens x the G q heads of a kv head a wave) and walks the keys up to its
// last token 128 a step.  A step's codes become bf16 keys (times their scales) and fp16 values in LDS once, for all
// of the workgroup's rows, while the step before is computed: the codes are requested two steps ahead into
// registers, converted one step ahead into the other half of LDS, and a step has one barrier.
//   S^T[32 keys x 32 rows] = K . Q^T        (8 MFMA 32x32x16 bf16)
//   O^T[128 dims x 32 rows] += V^T . P^T    (4 MFMA 32x32x16 fp16 a page)
// A lane owns one row throughout: its scores of a page are its P operand as they are, since the 16 keys of V's
// operand are kept in the order in which the score tile holds them.
constexpr int kRowsWave = 32, kBlockRows = 256;  // a row block (jit_prefill_block_tokens): 256 / G tokens
constexpr int kStepKeys = 128, kStepPages = kStepKeys / kPage;
constexpr int kPartKeys = 6144;                  // key parts (jit_prefill_part_keys)
constexpr int kPartSteps = kPartKeys / kStepKeys;
constexpr int kPfSlot = kD + 4;                  // floats of a (token, part, head) partial: o, max, sum, 2 pad
// Values are held in LDS relative to the loudest scale so far, 2^E, times 2^7 (448 x 2^7 < 65,504): a value of a token
// 2^22 times quieter than that still has all its bits.
constexpr int kVShift = 7;

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mfma32x32x16(const Frag8 &a, const Frag8 &b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32x32x16_f16(const FragH &a, const FragH &b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a.v, b.v, c, 0, 0, 0);
}

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

// What a wave requests of a step: its pages' codes and scales, and the step's V scales (2 keys a lane).
template <int PAGES>
struct Staged {
  uint4 k[PAGES][2], v[PAGES][2];
  float ks[PAGES];
  float4 vs[PAGES][2];
  float2 all_vs;
  uint32_t bad;  // the step's pages outside the pool
};

template <int WAVES>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(WAVES / 4 < 1 ? 1 : WAVES / 4, 2)))
void kv8_prefill_kernel(const PrefillArgs a) {
  constexpr int kSub = kBlockRows / (WAVES * kRowsWave);  // workgroups a row block
  constexpr int kPages = kStepPages / WAVES;              // pages a wave stages a step
  __shared__ __attribute__((aligned(16))) uint4 s_k[2][kStepPages / 2][8][64];  // [page pair][16 dims][lane] 8 bf16
  __shared__ __attribute__((aligned(16))) uint4 s_v[2][kStepPages][4][64];      // [page][32 dims][lane] 8 fp16
  const int item = blockIdx.x / (kSub * a.Hkv), kvh = blockIdx.x % a.Hkv;
  const int ch = a.blk_chunk[item], part = a.blk_part[item];
  const int seq = a.chunk_seq[ch], ctx = a.chunk_ctx[ch], len = a.chunk_len[ch], row0 = a.chunk_row[ch];
  const int G = a.G, tpw = kRowsWave / G;  // tokens a wave
  int q0 = a.blk_q0[item];
  if constexpr (kSub > 1) q0 += blockIdx.x / a.Hkv % kSub * WAVES * tpw;
  if (q0 >= len) return;  // (uniform)
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id();
  const int lr = l & 31, lh = l >> 5;
  const int kend = ctx + min(q0 + WAVES * tpw, len);  // the workgroup's keys: [0, kend)
  const int nst = (kend + kStepKeys - 1) / kStepKeys, npages = min((kend + kPage - 1) / kPage, a.max_pages);
  const int st0 = part * kPartSteps, st1 = min(nst, st0 + kPartSteps);
  if (st0 >= st1) return;  // (uniform: a piece of a block whose last token alone reaches the part)
  const int32_t *prow = a.page_table + (long long)seq * a.max_pages;

  const int t = q0 + wave * tpw + lr / G, tok = min(t, len - 1), pos = ctx + tok;  // the lane's row
  const int first_pos = ctx + min(q0 + wave * tpw, len - 1);                       // the wave's first
  Frag8 qf[8];
  {
    const uint16_t *qp = a.q + ((long long)(row0 + tok) * a.H + kvh * G + lr % G) * kD + 8 * lh;
#pragma unroll
    for (int s = 0; s < 8; s++) qf[s].q = *(const uint4 *)(qp + 16 * s);
  }
  float m_run = kLowest, l_run = 0.0f;
  f32x16 o[4];
#pragma unroll
  for (int c = 0; c < 4; c++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[c][i] = 0.0f;

  // a step's page ids, lane i page i % 8 (past the keys: the last page again, its keys masked)
  auto page_ids = [&](int st) { return prow[min(kStepPages * st + (l & (kStepPages - 1)), npages - 1)]; };
  auto request = [&](Staged<kPages> &r, int pages) {
    const bool bad = pages < 0 || pages >= a.num_pages;
    r.bad = (uint32_t)__ballot(bad) & 0xffu;
    const int ids = bad ? 0 : pages;
#pragma unroll
    for (int p = 0; p < kPages; p++) {
      const uint8_t *rec = record(a.pool, __builtin_amdgcn_readlane(ids, kPages * wave + p), a.Hkv, kvh);
      const float *sc = (const float *)(rec + kScaleOff);
      r.ks[p] = sc[l & 15];
#pragma unroll
      for (int i = 0; i < 2; i++) {
        r.k[p][i] = *(const uint4 *)(rec + 1024 * i + 16 * l);
        // lane (q = l / 32, h = l / 16 % 2, r = l % 16): slots 4 h .. and 8 + 4 h .. of dims 64 q + 16 c + r
        r.v[p][i] = *(const uint4 *)(rec + kVOff + 1024 * (l >> 5) + 512 * i + 16 * (l & 31));
        r.vs[p][i] = *(const float4 *)(sc + kPage + 8 * i + 4 * ((l >> 4) & 1));
      }
    }
    const uint8_t *rec = record(a.pool, __shfl(ids, l >> 3, 64), a.Hkv, kvh);
    r.all_vs = *(const float2 *)(rec + kScaleOff + 4 * kPage + 8 * (l & 7));
  };
  // the step's loudest live value; E over the part so far grows with it, and O's unit with E
  int e_run = kMinExp;
  auto grow_unit = [&](const Staged<kPages> &r, int k0) {
    int e = kMinExp;
    if (!((r.bad >> (l >> 3)) & 1)) {
      if (k0 + 2 * l < kend) e = max(e, (int)(__float_as_uint(r.all_vs.x) >> 23) - 127);
      if (k0 + 2 * l + 1 < kend) e = max(e, (int)(__float_as_uint(r.all_vs.y) >> 23) - 127);
    }
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) e = max(e, __shfl_xor(e, x, 64));
    const int e_new = max(e_run, min(__builtin_amdgcn_readfirstlane(e), kMaxExp));
    const float f = e_new - e_run > 126 ? 0.0f : exp_bits(e_run - e_new);
    e_run = e_new;
    return f;
  };
  auto convert = [&](const Staged<kPages> &r, int st) {
    const int buf = st & 1, k0 = kStepKeys * st;
#pragma unroll
    for (int p = 0; p < kPages; p++) {
      const int pg = kPages * wave + p;
#pragma unroll
      for (int i = 0; i < 2; i++) {  // lane (g = l / 16, slot = l % 16): dims 64 i + 16 g ..
        uint4 f0, f1;
        to_bf16(r.k[p][i].x, r.ks[p], f0.x, f0.y);
        to_bf16(r.k[p][i].y, r.ks[p], f0.z, f0.w);
        to_bf16(r.k[p][i].z, r.ks[p], f1.x, f1.y);
        to_bf16(r.k[p][i].w, r.ks[p], f1.z, f1.w);
        uint4 *dst = &s_k[buf][pg >> 1][4 * i + (l >> 4)][16 * (pg & 1) + (l & 15)];
        dst[0] = f0;
        dst[32] = f1;
      }
      f16x2_t fac[2][2];
      uint32_t w[2][4];
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const int keep = (r.bad >> pg) & 1 ? 0 : kend - (k0 + kPage * pg + 8 * i + 4 * ((l >> 4) & 1));
        const uint32_t km = keep_bytes(keep);  // (what lies past the keys may be anything: no NaN code gets in)
        w[i][0] = r.v[p][i].x & km, w[i][1] = r.v[p][i].y & km, w[i][2] = r.v[p][i].z & km, w[i][3] = r.v[p][i].w & km;
        const float *sp = (const float *)&r.vs[p][i];
#pragma unroll
        for (int j = 0; j < 4; j++) {  // 2^(e - E + 7); below fp16's range 0
          const int e = (int)(__float_as_uint(sp[j]) >> 23) - 127 - e_run + kVShift;
          fac[i][j >> 1][j & 1] = (_Float16)exp_bits(max(min(e, kVShift), -100));
        }
      }
#pragma unroll
      for (int c = 0; c < 4; c++) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 2; i++) {
          to_f16(w[i][c], u[2 * i], u[2 * i + 1]);
#pragma unroll
          for (int j = 0; j < 2; j++)
            u[2 * i + j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, u[2 * i + j]) * fac[i][j]);
        }
        s_v[buf][pg][2 * (l >> 5) + (c >> 1)][32 * ((l >> 4) & 1) + 16 * (c & 1) + (l & 15)] =
            make_uint4(u[0], u[1], u[2], u[3]);
      }
    }
  };

  Staged<kPages> r;
  request(r, page_ids(st0));
  int ids = page_ids(st0 + 1);
  float e_next = grow_unit(r, kStepKeys * st0);
  uint32_t bad = r.bad;
  convert(r, st0);
  request(r, ids);
  ids = page_ids(st0 + 2);
  for (int st = st0; st < st1; st++) {
    const int k0 = kStepKeys * st, buf = st & 1;
    // every wave has written its share of this step and read the step before (a bare barrier: __syncthreads would
    // also wait for the codes in flight)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((15) | (3 << 14) | (7 << 4) | (0 << 8));  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const float e_alpha = e_next;
    const uint32_t bad_pages = bad;
    if (st + 1 < st1) {
      e_next = grow_unit(r, k0 + kStepKeys);
      bad = r.bad;
      convert(r, st + 1);
      request(r, ids);
      ids = page_ids(st + 3);
    }
    f32x16 sc[kStepPages / 2];
#pragma unroll
    for (int g = 0; g < kStepPages / 2; g++) {
#pragma unroll
      for (int i = 0; i < 16; i++) sc[g][i] = 0.0f;
#pragma unroll
      for (int s = 0; s < 8; s++) {
        Frag8 kf;
        kf.q = s_k[buf][g][s][l];
        sc[g] = mfma32x32x16(kf, qf[s], sc[g]);
      }
    }
    // score i of a lane in key group g: key 32 g + 8 (i / 4) + 4 lh + i % 4
    if (k0 + kStepKeys - 1 > first_pos || bad_pages) {
#pragma unroll
      for (int g = 0; g < kStepPages / 2; g++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const int key = k0 + 32 * g + 8 * (i >> 2) + 4 * lh + (i & 3);
          if (key > pos || ((bad_pages >> (2 * g + (i >> 3))) & 1)) sc[g][i] = -INFINITY;
        }
    }
    float tmax = sc[0][0];
#pragma unroll
    for (int g = 0; g < kStepPages / 2; g++)
#pragma unroll
      for (int i = 0; i < 16; i++) tmax = fmaxf(tmax, sc[g][i]);
    tmax = max_xor32(tmax) * a.qk_scale;
    const float m_new = fmaxf(m_run, tmax), alpha = __builtin_amdgcn_exp2f(m_run - m_new), scale_o = alpha * e_alpha;
    if (__any(scale_o != 1.0f)) {
#pragma unroll
      for (int c = 0; c < 4; c++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[c][i] *= scale_o;
    }
    float psum = 0.0f;
    const float off = kPShift - m_new;
#pragma unroll
    for (int p = 0; p < kStepPages; p++) {
      FragH pf;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float x = __builtin_amdgcn_exp2f(fmaf(sc[p >> 1][8 * (p & 1) + 2 * j], a.qk_scale, off));
        const float y = __builtin_amdgcn_exp2f(fmaf(sc[p >> 1][8 * (p & 1) + 2 * j + 1], a.qk_scale, off));
        psum += x + y;
        pf.u[j] = pack_f16x2(x, y);
      }
#pragma unroll
      for (int c = 0; c < 4; c++) {
        FragH vf;
        vf.q = s_v[buf][p][c][l];
        o[c] = mfma32x32x16_f16(vf, pf, o[c]);
      }
    }
    l_run = fmaf(l_run, alpha, psum);
    m_run = m_new;
  }
  const float unit = exp_bits(e_run - kVShift);
  const float l_tot = sum_xor32(l_run);
  const int parts = pos / kPartKeys + 1;
  if (t >= len || part >= parts) return;  // (a token before this part's keys: finished by its own last part)
  const long long hrow = (long long)(row0 + tok) * a.H + kvh * G + lr % G;
  if (parts == 1) {
    const float inv = l_tot == 0.0f ? 0.0f : unit / l_tot;
#pragma unroll
    for (int c = 0; c < 4; c++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        uint2 w;
        w.x = pack_bf16x2(o[c][4 * i] * inv, o[c][4 * i + 1] * inv);
        w.y = pack_bf16x2(o[c][4 * i + 2] * inv, o[c][4 * i + 3] * inv);
        *(uint2 *)(a.out + hrow * kD + 32 * c + 8 * i + 4 * lh) = w;
      }
  } else {
    float *ps = a.part + (((long long)(row0 + tok) * a.pmax + part) * a.H + kvh * G + lr % G) * kPfSlot;
#pragma unroll
    for (int c = 0; c < 4; c++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        *(float4 *)(ps + 32 * c + 8 * i + 4 * lh) = make_float4(o[c][4 * i] * unit, o[c][4 * i + 1] * unit,
                                                                o[c][4 * i + 2] * unit, o[c][4 * i + 3] * unit);
    if (lh == 0) *(float2 *)(ps + kD) = make_float2(m_run, l_tot);
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
  kv8_prefill_kernel<8><<<dim3(nblk * Hkv), 64 * 8, 0, st>>>(a);
  const int rc = jit::check_launch("jit_paged_prefill_attn_kv8");
  if (rc || pmax == 1 || max_len == 0) return rc;
  kv8_prefill_merge_kernel<<<dim3(max_len, C), 8 * H, 0, st>>>(a);
  return jit::check_launch("jit_paged_prefill_attn_kv8");
}
