// Attention over the 8-bit KV cache for gfx950: single tokens (split over the keys) and causal prompt chunks.
// Records and number format: kv8.hpp.
//
// Scores are formed from the codes, K_codes . Q^T in bf16 matrix instructions (codes and q are exact there), and
// take their key's scale afterwards.  Single tokens, bound by memory, keep 16 bits of a probability times V's scale, as
// a high and a low bf16 part (as the bf16 pool's attention does).  Prompt chunks, bound by the matrix instructions, take a
// probability as one fp16, 11 bits: 16 of them would be twice the products with V.
#include "kv8.hpp"

#include <type_traits>

namespace {

using namespace kv8;

// The running maximum before any key: finite, so that rows without a key stay 0, and no finite score lies below it.
constexpr float kLowest = -3.402823466e38f;

// ---------------------------------------------------------------- single tokens
// A sequence is cut into chunks by its own length alone, a chunk into 4 runs of a wave each.  512 keys: with 768 and
// 1,024 64 sequences of 300 keys take 9.9 and 11.5 us a call instead of 8.3, one of 4,096 13.1 and 13.0 instead of 11.1,
// 32 ragged ones 29 to 32 with any of the three.
constexpr int kSplits = 4;
// What meets in a product: a probability times V's scale times 2^8 (2^-92 .. 2^126: both parts are normal numbers down to
// p = 2^-18 of the quietest block), and V's codes times 2^-28.  O is 2^-20 of its size: 2^20 keys of the loudest block
// stay in fp32's range.
constexpr float kVScaleUp = 256.0f, kCodeScale = 0x1p-28f, kOBack = 0x1p20f;
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
  int num_pages, max_pages, B, H, Hkv, G, max_len, ncap;  // max_len: at most the page table's width
  float qk_scale;                                         // scale * log2(e)
};

__device__ __forceinline__ int seq_len(const DecodeArgs &a, int b) { return min(max(a.lens[b], 0), a.max_len); }

constexpr int kStateFloats = 32 + 2;  // o[8][4], max, sum per lane
constexpr int kDecodeWgs = 3;         // workgroups a CU holds (160 registers a lane)
constexpr int kDecodeSeqs = 4096;     // sequences a launch covers (8 bytes of LDS each)

// A bare barrier behind LDS accesses: __syncthreads would also wait for the loads in flight.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((15) | (3 << 14) | (7 << 4) | (0 << 8));  // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Lane J's value of each quad of lanes.
template <int J>
__device__ __forceinline__ float quad(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x55 * J, 0xF, 0xF, true));
}

// What a wave needs of its run of a chunk.
struct Run {
  int b, c, n;         // sequence, chunk, the sequence's chunks
  int k0, k1, pages;   // keys [k0, k1), their pages
  int id;              // lane i: page i's id (a page outside the pool: 0, and its bit in bad)
  unsigned long long bad;
};

// The chunks of all sequences are one list (a sequence without keys has one empty chunk); a workgroup takes every
// gridDim.x-th of them for one kv head, each wave a quarter.  The grid is what the GPU holds at once, whatever the
// lengths: sized by the host's bound (32 sequences of 128 to 32,768 keys: 8,448 workgroups for 1,003 chunks) most
// workgroups only took a CU's place for the microsecond in which they found that they had nothing to do.  A
// wave never runs dry: the first loads of its next chunk are in flight while it ends one.
// Bound by memory: 262,144 keys of 4 kv heads (277 MB) in 45.8 us, 6.0 TB/s; the 32 sequences (133 MB) in 28.4, 4.7 TB/s;
// one of 4,096 keys takes 7.7 us, the latency of a run.  (Reads alone reach 7.1 TB/s here.)
__global__ __launch_bounds__(64 * kSplits) __attribute__((amdgpu_waves_per_eu(kDecodeWgs, kDecodeWgs)))
void kv8_decode_kernel(const DecodeArgs a) {
  __shared__ float xstate[kSplits][kStateFloats][64];
  __shared__ int s_sum[kSplits];
  extern __shared__ int s_seq[];  // [B]: chunks up to and with b; [B]: length
  const int kvh = blockIdx.y;
  const int split = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id();
  const int lr = l & 15, lg = l >> 4, G = a.G;
  int total = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64 * kSplits) {
    const int b = b0 + threadIdx.x, L = b < a.B ? seq_len(a, b) : 0;
    int v = b < a.B ? max(chunks_of(L), 1) : 0;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(v, o, 64);
      if (l >= o) v += u;
    }
    if (l == 63) s_sum[split] = v;
    __syncthreads();
    for (int w = 0; w < kSplits; w++) {
      if (w < split) v += s_sum[w];
    }
    if (b < a.B) s_seq[b] = total + v, s_seq[a.B + b] = L;
    for (int w = 0; w < kSplits; w++) total += s_sum[w];
    __syncthreads();
  }
  auto locate = [&](int item, Run &r) {
    int lo = 0, hi = a.B - 1;  // the first sequence whose chunks end past the item
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (__builtin_amdgcn_readfirstlane(s_seq[mid]) > item) hi = mid;
      else lo = mid + 1;
    }
    const int L = __builtin_amdgcn_readfirstlane(s_seq[a.B + lo]), ck = chunk_tokens(L), run = ck / kSplits;
    r.b = lo;
    r.c = item - (lo ? __builtin_amdgcn_readfirstlane(s_seq[lo - 1]) : 0);
    r.n = chunks_of(L);
    r.k0 = r.c * ck + split * run;
    r.k1 = min(r.k0 + run, L);
    r.pages = r.k1 > r.k0 ? (r.k1 - r.k0 + kPage - 1) / kPage : 0;
    r.id = l < r.pages ? a.page_table[(long long)lo * a.max_pages + r.k0 / kPage + l] : 0;
  };
  auto check_pages = [&](Run &r) {  // (waits for the ids)
    const bool bad = (uint32_t)r.id >= (uint32_t)a.num_pages;
    r.bad = __ballot(bad);
    if (bad) r.id = 0;
  };
  // Q^T (bf16): q head lr, dims 64 (f / 2) + 16 lg + 8 (f % 2) ..
  Frag8 qf[4];
  auto request_q = [&](const Run &r) {
    const uint16_t *qp = a.q + ((long long)r.b * a.H + kvh * G + lr) * kD + 16 * lg;
#pragma unroll
    for (int f = 0; f < 4; f++) qf[f].q = lr < G ? *(const uint4 *)(qp + 64 * (f >> 1) + 8 * (f & 1)) : make_uint4(0, 0, 0, 0);
  };
  // A step's registers are requested again for the next step as soon as they are used: K and the scales once its
  // scores are formed, V once its products are issued.
  uint4 kc[2][2], vc[2][2];
  float ks[2], vs[2];  // lane (lr, lg): of key 4 lg + lr % 4; a lane's four keys are its quad's
  const uint32_t lane16 = 16 * l, lane_s = 16 * lg + 4 * (l & 3);
  auto rec_of = [&](const Run &r, int st, int p) {  // (a page past the run: the last one again, its keys masked)
    return record(a.pool, __builtin_amdgcn_readlane(r.id, min(2 * st + p, r.pages - 1)), a.Hkv, kvh);
  };
  auto request_k = [&](const Run &r, int st) {
#pragma unroll
    for (int p = 0; p < 2; p++) {
      const uint8_t *rec = rec_of(r, st, p);
      kc[p][0] = ld_stream16(rec + lane16);
      kc[p][1] = ld_stream16(rec + 1024 + lane16);
      ks[p] = *(const float *)(rec + kScaleOff + lane_s);
      vs[p] = *(const float *)(rec + kScaleOff + 4 * kPage + lane_s);
    }
  };
  auto request_v = [&](const Run &r, int st) {
#pragma unroll
    for (int p = 0; p < 2; p++) {
      const uint8_t *rec = rec_of(r, st, p) + kVOff;
      vc[p][0] = ld_stream16(rec + lane16);
      vc[p][1] = ld_stream16(rec + 1024 + lane16);
    }
  };

  int item = blockIdx.x;
  if (item >= total) return;  // (uniform)
  Run cur, nxt;
  nxt.pages = 0;
  locate(item, cur);
  request_q(cur);
  check_pages(cur);
  if (cur.pages) {
    request_k(cur, 0);
    asm volatile("" ::: "memory");
    request_v(cur, 0);
  }
  for (;;) {
    const bool more_items = item + (int)gridDim.x < total;
    if (more_items) locate(item + gridDim.x, nxt);
    float m_run = kLowest, l_run = 0.0f;
    f32x4 o[8];
#pragma unroll
    for (int cc = 0; cc < 8; cc++) o[cc] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int nst = (cur.pages + 1) >> 1;
    // LAST: the run's last step, which requests the next run's first
    auto step = [&](const int st, auto last) {
      constexpr bool LAST = decltype(last)::value;
      const int k0 = cur.k0 + 32 * st;
      const bool cut = LAST || cur.bad;  // (keys past the run: in its last step only)
      // keys of this step that count: below k1, of pages in the pool (lane: 4 of each page)
      int keep[2];
#pragma unroll
      for (int p = 0; p < 2; p++)
        keep[p] = !cut ? 4 : (cur.bad >> min(2 * st + p, 63)) & 1 ? 0 : cur.k1 - (k0 + 16 * p + 4 * lg);
      f32x4 s[2];
#pragma unroll
      for (int p = 0; p < 2; p++) {
        s[p] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int f = 0; f < 4; f++) {
          Frag8 kf;
          const uint32_t w0 = (f & 1) ? kc[p][f >> 1].z : kc[p][f >> 1].x, w1 = (f & 1) ? kc[p][f >> 1].w : kc[p][f >> 1].y;
          to_bf16(w0, 1.0f, kf.u[0], kf.u[1]);
          to_bf16(w1, 1.0f, kf.u[2], kf.u[3]);
          s[p] = mfma16x16x32(kf, qf[f], s[p]);
        }
      }
      float t[2][4], v8[2][4];  // scores, then weights; V's scales
#pragma unroll
      for (int p = 0; p < 2; p++) {
        float vb = vs[p] * kVScaleUp;
        if (cut) vb = (l & 3) < keep[p] ? vb : 0.0f;
        const float kq = ks[p] * a.qk_scale;
        const float kqs[4] = {quad<0>(kq), quad<1>(kq), quad<2>(kq), quad<3>(kq)};
        v8[p][0] = quad<0>(vb), v8[p][1] = quad<1>(vb), v8[p][2] = quad<2>(vb), v8[p][3] = quad<3>(vb);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          t[p][i] = s[p][i] * kqs[i];
          if (cut) t[p][i] = i < keep[p] ? t[p][i] : -INFINITY;
        }
      }
      asm volatile("" ::: "memory");
      if constexpr (!LAST) {
        request_k(cur, st + 1);
      } else if (more_items) {
        check_pages(nxt);
        if (nxt.pages) request_k(nxt, 0);
        if (nxt.b != cur.b) request_q(nxt);
      }
      asm volatile("" ::: "memory");
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
          t[p][i] = __builtin_amdgcn_exp2f(t[p][i] - m_new);
          psum += t[p][i];
          t[p][i] *= v8[p][i];
        }
      l_run = fmaf(l_run, alpha, psum);
      m_run = m_new;
      Frag8 high, rest;
#pragma unroll
      for (int i = 0; i < 4; i++) split_bf16x2(t[i >> 1][2 * (i & 1)], t[i >> 1][2 * (i & 1) + 1], high.u[i], rest.u[i]);
      if (cut) {  // (a p of 0 does not cancel a NaN code)
#pragma unroll
        for (int p = 0; p < 2; p++) {
          const uint32_t km = keep_bytes(keep[p]);
#pragma unroll
          for (int i = 0; i < 2; i++) vc[p][i].x &= km, vc[p][i].y &= km, vc[p][i].z &= km, vc[p][i].w &= km;
        }
      }
      if (__any(alpha != 1.0f)) {
#pragma unroll
        for (int cc = 0; cc < 8; cc++)
#pragma unroll
          for (int i = 0; i < 4; i++) o[cc][i] *= alpha;
      }
#pragma unroll
      for (int cc = 0; cc < 8; cc++) {
        Frag8 vf;
#pragma unroll
        for (int p = 0; p < 2; p++)
          to_bf16(((const uint32_t *)&vc[p][cc >> 2])[cc & 3], kCodeScale, vf.u[2 * p], vf.u[2 * p + 1]);
        o[cc] = mfma16x16x32(vf, high, o[cc]);
        o[cc] = mfma16x16x32(vf, rest, o[cc]);
      }
      asm volatile("" ::: "memory");
      if constexpr (!LAST) request_v(cur, st + 1);
      else if (more_items && nxt.pages) request_v(nxt, 0);
      asm volatile("" ::: "memory");
    };
    for (int st = 0; st + 1 < nst; st++) step(st, std::false_type());
    if (nst > 0) {
      step(nst - 1, std::true_type());
    } else if (more_items) {  // (a run without keys)
      check_pages(nxt);
      if (nxt.pages) {
        request_k(nxt, 0);
        asm volatile("" ::: "memory");
        request_v(nxt, 0);
      }
      if (nxt.b != cur.b) request_q(nxt);
    }
    // the runs' states meet, in run order: each wave merges a quarter of the dims
    const long long row = (long long)cur.b * a.H + kvh * G + lr;  // this lane's q head
    lds_barrier();                                               // (the chunk before has been read)
    {
      float(*st)[64] = xstate[split];
#pragma unroll
      for (int cc = 0; cc < 8; cc++)
#pragma unroll
        for (int i = 0; i < 4; i++) st[4 * cc + i][l] = o[cc][i];
      st[32][l] = m_run;
      st[33][l] = l_run;
    }
    lds_barrier();
    {
      float f[kSplits], M = xstate[0][32][l], l_tot = 0.0f;
#pragma unroll
      for (int sp = 0; sp < kSplits; sp++) f[sp] = xstate[sp][32][l];
#pragma unroll
      for (int sp = 1; sp < kSplits; sp++) M = fmaxf(M, f[sp]);
#pragma unroll
      for (int sp = 0; sp < kSplits; sp++) {
        f[sp] = __builtin_amdgcn_exp2f(f[sp] - M);
        l_tot = fmaf(xstate[sp][33][l], f[sp], l_tot);
      }
      l_tot = sum_xor32(sum_xor16(l_tot));
      const float inv = cur.n > 1 ? 1.0f : l_tot == 0.0f ? 0.0f : kOBack / l_tot;
      const long long r = ((long long)cur.b * a.ncap + cur.c) * a.H + kvh * G + lr;
#pragma unroll
      for (int x = 0; x < 2; x++) {
        const int cc = 2 * split + x;
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          y[i] = 0.0f;
#pragma unroll
          for (int sp = 0; sp < kSplits; sp++) y[i] = fmaf(xstate[sp][4 * cc + i][l], f[sp], y[i]);
        }
        if (lr < G && cur.n <= 1)
          *(uint2 *)(a.out + row * kD + 16 * cc + 4 * lg) =
              make_uint2(pack_bf16x2(y[0] * inv, y[1] * inv), pack_bf16x2(y[2] * inv, y[3] * inv));
        else if (lr < G)
          *(float4 *)(a.part_o + r * kD + 16 * cc + 4 * lg) = make_float4(y[0], y[1], y[2], y[3]);
      }
      if (cur.n > 1 && split == 0 && lg == 0 && lr < G) *(float2 *)(a.part_ml + 2 * r) = make_float2(M, l_tot);
    }
    if (!more_items) return;  // (uniform)
    item += gridDim.x;
    cur = nxt;
  }
}

// The chunks of a (sequence, q head), in order: thread = chunk lane (16) x 4 dims; lane j takes chunks j, j + 16, ..
// (3.4 to 5.6 us: an empty launch and two or three trips to memory)
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
  const float inv = l_tot == 0.0f ? 0.0f : kOBack / l_tot;
  uint2 w;
  w.x = pack_bf16x2(acc.x * inv, acc.y * inv);
  w.y = pack_bf16x2(acc.z * inv, acc.w * inv);
  *(uint2 *)(a.out + ((long long)b * a.H + h) * kD + 4 * t) = w;
}

// ---------------------------------------------------------------- causal prompt chunks
// Two launches (three where a token's keys have several parts).  The first expands the keys that the chunks see: K to
// bf16 (times its scale) and V to fp16 (or bf16: kSpread), in the order in which the second launch's matrix instructions
// take them.
// Every row block of a chunk reads all of its keys, so the conversion is done once instead of once a block; inside the
// attention loop it cost as many vector instructions as the softmax (2,048 rows after 8,192 keys: 344 us, without it 328).
//
// The second: a workgroup owns 4 waves x 32 rows (32 / G tokens x the G q heads of a kv head a wave) and walks the keys
// of a part, up to its last token, 64 (a unit) at a time, a unit's 32 KB going straight from memory into LDS.  Two
// workgroups share a CU.
//   S^T[32 keys x 32 rows] = K . Q^T        (8 MFMA 32x32x16 bf16)
//   O^T[128 dims x 32 rows] += V^T . P^T    (4 MFMA 32x32x16 fp16 a page; 8 of bf16 in a part of uneven V)
// Bound by the matrix instructions and the clock they leave (2,048 rows after 8,192 keys: busy 60% of the cycles at 1.9 GHz,
// LDS reads 30%, 298 to 312 us, 1.0 PFLOP/s; a large bf16 product of the library 1.14 to 1.4).  Both workgroups of a CU are
// needed: with one of four waves, however many units are on their way, the same takes 394 us.
// A lane owns one row throughout: its scores of a page are its P operand as they are, since the 16 keys of V's
// operand are kept in the order in which the score tile holds them.
constexpr int kPfWaves = 4, kStages = 2;  // waves a workgroup; units in LDS: the one in use, and those on their way
constexpr int kRowsWave = 32, kBlockRows = kPfWaves * kRowsWave;  // a row block: 128 / G tokens
constexpr int kUnitKeys = JIT_KV8_UNIT_KEYS, kUnitPages = kUnitKeys / kPage;
constexpr int kUnitBytes = 2 * kUnitKeys * kD * 2;  // K, then V
constexpr int kPartMax = 192;  // units of the longest part: every unit's workgroup looks through its part's scales
constexpr int kPfSlot = kD + 4;                  // floats of a (token, part, head) partial: o / sum, max, sum, 2 pad
// A row's reference for the exponentials moves when its maximum passes it by more than 2^4: most units then have no O
// to rescale.  Probabilities are formed 2^11 times too large, at most 2^15: 11 bits down to 2^-25 of the reference.
constexpr float kLazy = 4.0f, kPfShift = 11.0f;
// Two forms of a part, by the scales of V's blocks that its keys hold:
// * within 2^12 of each other: V in fp16 relative to the loudest scale 2^E, times 2^7 (448 x 2^7 < 65,504; the quietest
//   block's least code is 2^-14 then, so every value has all its bits and no row depends on E), probabilities as one fp16.
//   One below fp16's range is off by 2^-25, 2^-36 of the row's sum at least: 12,288 keys 2^12 times louder than what the
//   row is made of lose it 2^(13.6 - 36 + 12), less than a fifth of a bf16 rounding.
// * further apart: V in bf16 as it is (4 bits, 2^-109 .. 2^127: exact) and probabilities as a high and a low bf16 part, 16
//   bits at any magnitude, 2^-20 of their size so that no sum passes fp32's range: half as many matrix instructions again
//   (2,048 rows after 8,192 keys: 408 us instead of 298).
constexpr int kVShift = 7, kSpread = 12;
constexpr float kWideShift = -20.0f;

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
  const int32_t *chunk_unit, *chunk_part, *chunk_slot;  // [C + 1]: first unit of each; units a part; first partial slot
  uint16_t *out;
  uint8_t *units;  // [units][Hkv][kUnitBytes]
  int32_t *info;   // [units][Hkv][2]: E of the unit's part, its pages outside the pool (4 bits; 16: some in the part;
                   // 32: NaN codes of V in the unit; 64: the part's V scales are more than 2^kSpread apart)
  float *part;     // (token, part, head): o / sum, the maximum, the sum
  int num_pages, max_pages, H, Hkv, G, C, num_units, num_slots;
  float qk_scale;
};

// The tables of units, parts, slots and work items lie in the caller's device memory: each kernel leaves out an entry that
// does not belong to its chunk before it becomes an address.  Here: the first slot of token t's partials, or -1.
__device__ __forceinline__ long long first_slot(const PrefillArgs &a, int ch, int part_units, int t, int parts) {
  const uint32_t units = (uint32_t)a.chunk_unit[ch + 1] - (uint32_t)a.chunk_unit[ch];
  const uint32_t most = (units + (uint32_t)part_units - 1u) / (uint32_t)part_units;
  const long long s = a.chunk_slot[ch] + (long long)t * most;
  return most >= (uint32_t)parts && s >= 0 && s + parts <= a.num_slots ? s : -1;
}

// One workgroup expands a unit of one kv head, wave w its page w: 10,240 keys of 4 heads, 11 MB to 21 MB, in 16 to 18 us,
// most of it the latency of its part's scales (parts of 96 units: 11 us).  Its codes are requested first; meanwhile the part's
// loudest and quietest live V scales are found (by every workgroup of a part for itself: a line of 64 bytes a page).
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(8))) void kv8_expand_kernel(const PrefillArgs a) {
  __shared__ int s_e[4], s_bad[4], s_ids[kPartMax * kUnitPages];
  __shared__ uint32_t s_least[4];
  const int gu = blockIdx.x, kvh = blockIdx.y, l = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int lo = 0, hi = a.C - 1;  // the chunk whose units hold gu
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.chunk_unit[mid] <= gu) lo = mid;
    else hi = mid - 1;
  }
  const int u = gu - a.chunk_unit[lo], kend = a.chunk_ctx[lo] + a.chunk_len[lo];
  if (u < 0 || u > (kend - 1) / kUnitKeys) return;  // (uniform: no such unit of a chunk)
  const int32_t *prow = a.page_table + (long long)a.chunk_seq[lo] * a.max_pages;
  const int npages = min((kend + kPage - 1) / kPage, a.max_pages);
  // the part's pages
  const int part = min(max(a.chunk_part[lo], 1), kPartMax), pg0 = u / part * part * kUnitPages;
  const int np = min(part * kUnitPages, npages - pg0);
  for (int i = threadIdx.x; i < np; i += 256) s_ids[i] = prow[pg0 + i];
  // this wave's page
  const int pg = kUnitPages * u + wave, page = pg < npages ? prow[pg] : -1;
  const bool out_of_pool = (uint32_t)page >= (uint32_t)a.num_pages;
  const uint8_t *rec = record(a.pool, out_of_pool ? 0 : page, a.Hkv, kvh);
  const float *sc = (const float *)(rec + kScaleOff);
  // K: lane (g = l / 16, slot = l % 16), dims 64 i + 16 g ..
  // V: lane (q = l / 32, h = l / 16 % 2, r = l % 16): slots 4 h .. and 8 + 4 h .. of dims 64 q + 16 c + r
  const int vh = (l >> 4) & 1;
  uint4 wk[2], wv[2];
  float4 sv[2];
  const float sk = sc[l & 15];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    wk[i] = *(const uint4 *)(rec + 1024 * i + 16 * l);
    wv[i] = *(const uint4 *)(rec + kVOff + 1024 * (l >> 5) + 512 * i + 16 * (l & 31));
    sv[i] = *(const float4 *)(sc + kPage + 8 * i + 4 * vh);
  }
  // E: thread = page of the part x quarter of its slots (a bare barrier: the codes stay in flight)
  int e = 0, bad = 0;    // (positive powers of two are ordered as their bits)
  uint32_t least = ~0u;  // (bits - 1: a slot never written, scale 0, is the last of all)
  lds_barrier();
#pragma unroll 6
  for (int i = threadIdx.x; i < 4 * np; i += 256) {
    const int p = pg0 + (i >> 2), id = s_ids[i >> 2];
    const bool off = (uint32_t)id >= (uint32_t)a.num_pages;
    const float4 s = *(const float4 *)(record(a.pool, off ? 0 : id, a.Hkv, kvh) + kScaleOff + 4 * kPage + 16 * (i & 3));
    const int left = off ? 0 : kend - (kPage * p + 4 * (i & 3));
    const float *sp = (const float *)&s;
    bad |= off;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      e = j < left ? max(e, __float_as_int(sp[j])) : e;
      least = j < left ? min(least, __float_as_uint(sp[j]) - 1u) : least;
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    e = max(e, __shfl_xor(e, o, 64));
    least = min(least, (uint32_t)__shfl_xor((int)least, o, 64));
  }
  const int any = __any(bad), here = __any(out_of_pool && pg < npages);
  // What lies past the keys or in a page outside the pool may be anything (0 x NaN): it counts as 0.  So do NaN codes
  // of V, which rows that do not see their key must not get either: kv8_prefill_kernel puts them back.
  int keep[2];
  uint32_t nan = 0;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    keep[i] = out_of_pool ? 0 : kend - (kPage * pg + 8 * i + 4 * vh);
    const uint32_t km = keep_bytes(keep[i]);
    uint32_t *w = (uint32_t *)&wv[i];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      w[j] &= km;
      const uint32_t n = (((w[j] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;  // 1 in the bytes 0x7f and 0xff
      w[j] &= ~(n * 255u);
      nan |= n;
    }
  }
  const int any_nan = __any(nan != 0);
  if (l == 0) s_e[wave] = e, s_least[wave] = least, s_bad[wave] = (any ? 16 : 0) | (here ? 1 << wave : 0) | (any_nan ? 32 : 0);
  __syncthreads();
  e = max(max(s_e[0], s_e[1]), max(s_e[2], s_e[3]));
  least = min(min(s_least[0], s_least[1]), min(s_least[2], s_least[3]));
  const int E = min(max((e >> 23) - 127, kMinExp), kMaxExp);
  const bool wide = e && (e >> 23) - (int)((least + 1u) >> 23) > kSpread;
  if (threadIdx.x == 0)
    *(int2 *)(a.info + 2 * ((long long)gu * a.Hkv + kvh)) =
        make_int2(E, s_bad[0] | s_bad[1] | s_bad[2] | s_bad[3] | (wide ? 64 : 0));
  uint4 *dst_k = (uint4 *)(a.units + ((long long)gu * a.Hkv + kvh) * kUnitBytes), *dst_v = dst_k + kUnitBytes / 32;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    uint4 f0, f1;
    to_bf16(wk[i].x, sk, f0.x, f0.y);
    to_bf16(wk[i].y, sk, f0.z, f0.w);
    to_bf16(wk[i].z, sk, f1.x, f1.y);
    to_bf16(wk[i].w, sk, f1.z, f1.w);
    uint4 *d = dst_k + (8 * (wave >> 1) + 4 * i + (l >> 4)) * 64 + 16 * (wave & 1) + (l & 15);
    d[0] = f0;
    d[32] = f1;
  }
  // value (i, j) of dims c: slot 8 i + 4 vh + j
  auto v_out = [&](int c) { return dst_v + (4 * wave + 2 * (l >> 5) + (c >> 1)) * 64 + 32 * vh + 16 * (c & 1) + (l & 15); };
  if (wide) {  // (uniform; rare)
#pragma unroll
    for (int c = 0; c < 4; c++) {
      uint32_t r[4];
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const float *sp = (const float *)&sv[i];
        uint32_t w[2];
        to_bf16(((const uint32_t *)&wv[i])[c], 1.0f, w[0], w[1]);
#pragma unroll
        for (int j = 0; j < 2; j++)
          r[2 * i + j] = pack_bf16x2_rne(2 * j < keep[i] ? bf2f(w[j] & 0xffffu) * sp[2 * j] : 0.0f,
                                         2 * j + 1 < keep[i] ? bf2f_hi(w[j]) * sp[2 * j + 1] : 0.0f);
      }
      *v_out(c) = make_uint4(r[0], r[1], r[2], r[3]);
    }
    return;
  }
  const float unit = exp_bits(kVShift - E);
  f16x2_t fac[2][2];  // 2^(e - E + 7); of a slot never written 0
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const float *sp = (const float *)&sv[i];
#pragma unroll
    for (int j = 0; j < 4; j++) fac[i][j >> 1][j & 1] = (_Float16)(j < keep[i] ? sp[j] * unit : 0.0f);
  }
#pragma unroll
  for (int c = 0; c < 4; c++) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 2; i++) to_f16(((const uint32_t *)&wv[i])[c], r[2 * i], r[2 * i + 1]);
#pragma unroll
    for (int i = 0; i < 4; i++)
      r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, r[i]) * fac[i >> 1][i & 1]);
    *v_out(c) = make_uint4(r[0], r[1], r[2], r[3]);
  }
}

// 16 bytes a lane from base + off straight into LDS at byte dst + 16 lane.  Written in assembly, so that the compiler's
// waits for LDS reads do not include these.  (s_nop: the load takes M0 one wait state after a scalar write of it at the
// earliest, which the compiler does not see to inside a string)
__device__ __forceinline__ void load_lds16(const uint8_t *base, uint32_t off, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(dst) : "memory", "m0");
}

__global__ __launch_bounds__(64 * kPfWaves) __attribute__((amdgpu_waves_per_eu(2, 2)))
void kv8_prefill_kernel(const PrefillArgs a) {
  constexpr int kLoads = 16 / kPfWaves;  // 1 KB loads of a wave for a unit's K (and V)
  __shared__ __attribute__((aligned(16))) uint4 s_k[kStages][16][64];              // [page pair, 16 dims][lane] 8 bf16
  __shared__ __attribute__((aligned(16))) uint4 s_v[kStages][kUnitPages * 4][64];  // [page, 32 dims][lane] 8 fp16
  const int item = blockIdx.x / a.Hkv, kvh = blockIdx.x % a.Hkv;
  const int ch = a.blk_chunk[item], q0 = a.blk_q0[item], part = a.blk_part[item];
  if (ch < 0 || ch >= a.C || q0 < 0 || part < 0) return;  // (uniform, as below)
  const int part_units = a.chunk_part[ch], unit0 = a.chunk_unit[ch];  // (loads on one trip to memory)
  const int ctx = a.chunk_ctx[ch], len = a.chunk_len[ch], row0 = a.chunk_row[ch];
  const int G = a.G, tpw = kRowsWave / G;  // tokens a wave
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id();
  const int lr = l & 31, lh = l >> 5;
  const int kend = ctx + min(q0 + kPfWaves * tpw, len);  // the workgroup's keys: [0, kend)
  const int all = (kend + kUnitKeys - 1) / kUnitKeys;
  if ((q0 >= len) | (unit0 < 0) | (all > a.num_units - unit0) | (part_units < 1) | (part_units > kPartMax)) return;
  if ((long long)part * part_units >= all) return;  // (no such item)
  const int u0 = part * part_units, u1 = min(all, u0 + part_units);
  const long long first_unit = (long long)unit0 * a.Hkv + kvh;  // (units of a head lie Hkv apart)
  const uint8_t *units = a.units + first_unit * kUnitBytes;
  const int32_t *info = a.info + 2 * first_unit;
  const uint32_t k_lds = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)&s_k[0][kLoads * wave][0]);
  const uint32_t v_lds = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)&s_v[0][kLoads * wave][0]);
  const uint32_t lane_at = 1024 * kLoads * wave + 16 * l;
  const long long unit_step_bytes = (long long)a.Hkv * kUnitBytes;
  // (a unit past the last: the last again, whose place in LDS is free and never read)
  auto request_k = [&](int u, int slot) __attribute__((always_inline)) {
    const uint8_t *p = units + min(u, u1 - 1) * unit_step_bytes;
#pragma unroll
    for (int i = 0; i < kLoads; i++) load_lds16(p, lane_at + 1024 * i, k_lds + 16384 * slot + 1024 * i);
  };
  auto request_v = [&](int u, int slot) __attribute__((always_inline)) {
    const uint8_t *p = units + min(u, u1 - 1) * unit_step_bytes + kUnitBytes / 2;
#pragma unroll
    for (int i = 0; i < kLoads; i++) load_lds16(p, lane_at + 1024 * i, v_lds + 16384 * slot + 1024 * i);
  };
  // K(u0) .. K(u0 + kStages - 1) and V(u0) .. V(u0 + kStages - 2), in the order of the loop's requests; q and the units'
  // infos come in behind them, on one trip to memory
  request_k(u0, 0);
#pragma unroll
  for (int i = 1; i < kStages; i++) {
    request_k(u0 + i, i);
    request_v(u0 + i - 1, i - 1);
  }
  const int t = q0 + wave * tpw + lr / G, tok = min(t, len - 1), pos = ctx + tok;  // the lane's row
  const int first_pos = ctx + min(q0 + wave * tpw, len - 1);                       // the wave's first
  Frag8 qf[8];
  {
    const uint16_t *qp = a.q + ((long long)(row0 + tok) * a.H + kvh * G + lr % G) * kD + 8 * lh;
#pragma unroll
    for (int s = 0; s < 8; s++) qf[s].q = *(const uint4 *)(qp + 16 * s);
  }
  const int E = info[2 * (long long)u0 * a.Hkv], flags = info[2 * (long long)u0 * a.Hkv + 1], some_bad = flags & 16;
  const bool wide = __builtin_amdgcn_readfirstlane(flags & 64) != 0;
  const float p_shift = wide ? kWideShift : kPfShift;
  int nan = 0;
  for (int u = u0 + l; u < u1; u += 64) nan |= info[2 * (long long)u * a.Hkv + 1] & 32;
  const bool some_nan = __any(nan);
  // (q is there before the loop, whose direct loads the compiler's waits for it would include)
#pragma unroll
  for (int s = 0; s < 8; s++)
    asm volatile("" ::"v"(qf[s].u[0]), "v"(qf[s].u[1]), "v"(qf[s].u[2]), "v"(qf[s].u[3]));
  float m_run = kLowest, l_run = 0.0f, top = 0.0f;
  f32x16 o[4];
#pragma unroll
  for (int c = 0; c < 4; c++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[c][i] = 0.0f;

  // The loads of units up to the one that is next are there, for every wave, and the units behind it are read: the newest
  // kStages - 2 units' loads stay in flight (vmcnt is split over bits 3:0 and 15:14), and a bare barrier follows.
  constexpr int kVm = (kStages - 2) * 2 * kLoads;
  auto meet = [&]() __attribute__((always_inline)) {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((kVm & 15) | ((kVm >> 4) << 14) | (7 << 4) | (0 << 8));  // vmcnt(kVm) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  constexpr int kAhead = 4;  // operand fragments requested from LDS ahead of their instructions
  f32x16 sc[2][2];  // scores of two units (u % 2) of two page pairs; lane: key 32 g + 8 (i / 4) + 4 lh + i % 4
  auto read_k = [&](int slot, int j) __attribute__((always_inline)) {  // page pair j % 2, dims 16 (j / 2)
    Frag8 f;
    f.q = s_k[slot][8 * (j & 1) + (j >> 1)][l];
    return f;
  };
  auto read_v = [&](int slot, int j) __attribute__((always_inline)) {  // page j / 4, dims 32 (j % 4)
    FragH f;
    f.q = s_v[slot][j][l];
    return f;
  };
  auto score = [&](f32x16 (&s)[2], const Frag8 &kf, int j) __attribute__((always_inline)) {
    const f32x16 z = {};
    s[j & 1] = mfma32x32x16(kf, qf[j >> 1], j < 2 ? z : s[j & 1]);
  };
  auto largest = [&](const f32x16 (&s)[2]) __attribute__((always_inline)) {
    top = s[0][0];
#pragma unroll
    for (int g = 0; g < 2; g++)
#pragma unroll
      for (int i = 0; i < 16; i++) top = fmaxf(top, s[g][i]);
  };
  // What of unit u's softmax waits for its scores' maximum, and O's rescaling.
  float off = 0.0f;
  auto settle = [&](int u, f32x16 (&s)[2]) __attribute__((always_inline)) {
    const int k0 = kUnitKeys * u;
    if (k0 + kUnitKeys - 1 > first_pos || some_bad) {
      const int bad = some_bad ? info[2 * (long long)u * a.Hkv + 1] : 0;
#pragma unroll
      for (int g = 0; g < 2; g++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const int key = k0 + 32 * g + 8 * (i >> 2) + 4 * lh + (i & 3);
          if (key > pos || ((bad >> (2 * g + (i >> 3))) & 1)) s[g][i] = -INFINITY;
        }
      largest(s);
    }
    top = max_xor32(top) * a.qk_scale;
    const float m_new = top > m_run + kLazy ? top : m_run;
    const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
    off = p_shift - m_new;
    l_run *= alpha;
    m_run = m_new;
    if (__any(alpha != 1.0f)) {
#pragma unroll
      for (int c = 0; c < 4; c++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[c][i] *= alpha;
    }
  };
  auto next = [](int slot, int by) { return slot + by >= kStages ? slot + by - kStages : slot + by; };
  int slot = 0;  // unit u's place in both rings
  // Unit u: its softmax beside the scores of unit u + 1, then its products with V beside the maximum of the new scores;
  // cut into groups of a matrix instruction and the vector work that runs during it.
  auto unit_step = [&](int u, f32x16 (&s)[2], f32x16 (&s_next)[2], bool more) __attribute__((always_inline)) {
    meet();
    const int k_slot = next(slot, 1);
    Frag8 kf[kAhead];
    FragH vf[kAhead], pf[kUnitPages];
#pragma unroll
    for (int j = 0; j < kAhead; j++) kf[j] = read_k(k_slot, j);
    request_k(u + kStages, slot);  // (K(u)'s and V(u - 1)'s places are free)
    request_v(u + kStages - 1, next(slot, kStages - 1));
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < 16; j++) {
      score(s_next, kf[j % kAhead], j);
      if (j + kAhead < 16) kf[j % kAhead] = read_k(k_slot, j + kAhead);
      else vf[j % kAhead] = read_v(slot, j + kAhead - 16);
      const float p0 = __builtin_amdgcn_exp2f(fmaf(s[j >> 3][2 * (j & 7)], a.qk_scale, off));
      const float p1 = __builtin_amdgcn_exp2f(fmaf(s[j >> 3][2 * (j & 7) + 1], a.qk_scale, off));
      pf[j >> 2].u[j & 3] = pack_f16x2(p0, p1);
      // (the sum of the rounded probabilities, which the products take too)
      l_run = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, pf[j >> 2].u[j & 3]), f16x2_t{1, 1}, l_run, false);
      asm volatile("" : "+v"(pf[j >> 2].u[j & 3]));  // (here, not where they are used)
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int j = 0; j < 16; j++) {
      o[j & 3] = mfma32x32x16_f16(vf[j % kAhead], pf[j >> 2], o[j & 3]);
      if (j + kAhead < 16) vf[j % kAhead] = read_v(slot, j + kAhead);
      if (j >= 3 && j < 11) {
        const int i0 = 4 * ((j - 3) & 3), g = (j - 3) >> 2;
        float x = j == 3 ? s_next[0][0] : top;
#pragma unroll
        for (int i = 0; i < 4; i++) x = fmaxf(x, s_next[g][i0 + i]);
        top = x;
        asm volatile("" : "+v"(top));
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    slot = k_slot;
    if (more) settle(u + 1, s_next);
  };

  // unit_step of a part of uneven V: bf16 V, a page's probabilities in two parts at a time (all four pages' do not fit the
  // registers)
  auto wide_step = [&](int u, f32x16 (&s)[2], f32x16 (&s_next)[2], bool more) __attribute__((always_inline)) {
    meet();
    const int k_slot = next(slot, 1);
    request_k(u + kStages, slot);
    request_v(u + kStages - 1, next(slot, kStages - 1));
#pragma unroll
    for (int j = 0; j < 16; j++) score(s_next, read_k(k_slot, j), j);
#pragma unroll
    for (int pg = 0; pg < kUnitPages; pg++) {
      Frag8 high, rest;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int i = 8 * (pg & 1) + 2 * j;
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[pg >> 1][i], a.qk_scale, off));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[pg >> 1][i + 1], a.qk_scale, off));
        split_bf16x2(p0, p1, high.u[j], rest.u[j]);
        l_run += p0 + p1;
      }
#pragma unroll
      for (int c = 0; c < 4; c++) {
        Frag8 v;
        v.q = s_v[slot][4 * pg + c][l];
        o[c] = mfma32x32x16(v, high, o[c]);
        o[c] = mfma32x32x16(v, rest, o[c]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    largest(s_next);
    slot = k_slot;
    if (more) settle(u + 1, s_next);
  };

  meet();
#pragma unroll
  for (int j = 0; j < 16; j++) score(sc[0], read_k(0, j), j);
  largest(sc[0]);
  settle(u0, sc[0]);
  int u = u0;
  if (!wide) {
    for (; u + 1 < u1; u += 2) {
      unit_step(u, sc[0], sc[1], true);
      unit_step(u + 1, sc[1], sc[0], u + 2 < u1);
    }
    if (u < u1) unit_step(u, sc[0], sc[1], false);
  } else {
    for (; u + 1 < u1; u += 2) {
      wide_step(u, sc[0], sc[1], true);
      wide_step(u + 1, sc[1], sc[0], u + 2 < u1);
    }
    if (u < u1) wide_step(u, sc[0], sc[1], false);
  }
  __builtin_amdgcn_s_waitcnt(0);  // no load may still write the LDS when the workgroup ends
  if (some_nan) {  // (rare) V's NaN codes, to the rows that see their keys
    const int32_t *prow = a.page_table + (long long)a.chunk_seq[ch] * a.max_pages;
    for (int u = u0; u < u1; u++) {
      if (!(info[2 * (long long)u * a.Hkv + 1] & 32)) continue;
      for (int k = 0; k < kUnitKeys; k++) {
        const int key = kUnitKeys * u + k;
        if (key > pos) break;
        const int page = key / kPage < a.max_pages ? prow[key / kPage] : -1;
        if ((uint32_t)page >= (uint32_t)a.num_pages) continue;
        const uint8_t *v = record(a.pool, page, a.Hkv, kvh) + kVOff + (k % kPage / 4) * 256 + k % 4;
#pragma unroll
        for (int c = 0; c < 4; c++)
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const int d = 32 * c + 8 * (i >> 2) + 4 * lh + (i & 3);  // (byte of (slot, d): 16 (4 q + c) + r)
            if ((v[(d >> 6) * 1024 + (d & 15) * 16 + ((d >> 4) & 3) * 4] & 127) == 127) o[c][i] = __builtin_nanf("");
          }
      }
    }
  }
  const float unit = wide ? 1.0f : exp_bits(E - kVShift);
  const float l_tot = sum_xor32(l_run);
  const int parts = pos / (kUnitKeys * part_units) + 1;
  if (t >= len || part >= parts) return;  // (a token before this part's keys: finished by its own last part)
  const long long hrow = (long long)(row0 + tok) * a.H + kvh * G + lr % G;
  // (divided by the part's own sum, so that a partial, too, is a mean of values of the cache: the undivided sum of loud
  // ones would pass fp32's range)
  const float inv = l_tot == 0.0f ? 0.0f : unit / l_tot;
  if (parts == 1) {
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
    const long long slot0 = first_slot(a, ch, part_units, tok, parts);
    if (slot0 < 0) return;
    float *ps = a.part + ((slot0 + part) * a.H + kvh * G + lr % G) * kPfSlot;
#pragma unroll
    for (int c = 0; c < 4; c++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        *(float4 *)(ps + 32 * c + 8 * i + 4 * lh) = make_float4(o[c][4 * i] * inv, o[c][4 * i + 1] * inv,
                                                                o[c][4 * i + 2] * inv, o[c][4 * i + 3] * inv);
    // (the sums of both forms at one size)
    if (lh == 0) *(float2 *)(ps + kD) = make_float2(m_run, wide ? l_tot * 0x1p31f : l_tot);
  }
}

// The parts of a token's keys in order, four at a time in flight: 16 heads a workgroup, thread (h, x) dims 32 i + 4 x .. + 3.
// O is the mean over the parts so far throughout: a part with the share w of the weight moves it by w (o - O).
__global__ __launch_bounds__(128) void kv8_prefill_merge_kernel(const PrefillArgs a) {
  const int c = blockIdx.y, t = blockIdx.x, h = 16 * blockIdx.z + (threadIdx.x >> 3);
  if (t >= a.chunk_len[c] || h >= a.H) return;
  const int pu = a.chunk_part[c], d0 = 4 * (threadIdx.x & 7);
  if (pu < 1 || pu > kPartMax) return;
  const int parts = (a.chunk_ctx[c] + t) / (kUnitKeys * pu) + 1;
  if (parts < 2) return;
  const long long slot0 = first_slot(a, c, pu, t, parts);
  if (slot0 < 0) return;
  const float *first = a.part + (slot0 * a.H + h) * kPfSlot;
  float M = kLowest, ls = 0.0f, O[16];
#pragma unroll
  for (int i = 0; i < 16; i++) O[i] = 0.0f;
  constexpr int kBatch = 4;
  for (int p0 = 0; p0 < parts; p0 += kBatch) {
    float4 v[kBatch][4];
    float2 ml[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; j++) {
      if (p0 + j >= parts) break;  // (uniform)
      const float *ps = first + (long long)(p0 + j) * a.H * kPfSlot;
      ml[j] = *(const float2 *)(ps + kD);
#pragma unroll
      for (int i = 0; i < 4; i++) v[j][i] = *(const float4 *)(ps + d0 + 32 * i);
    }
#pragma unroll
    for (int j = 0; j < kBatch; j++) {
      if (p0 + j >= parts) break;
      const float mn = fmaxf(M, ml[j].x), here = ml[j].y * exp2f(ml[j].x - mn);
      ls = fmaf(ls, exp2f(M - mn), here);
      const float w = ls == 0.0f ? 0.0f : here / ls;
      const float *x = (const float *)v[j];
#pragma unroll
      for (int i = 0; i < 16; i++) O[i] = fmaf(w, x[i] - O[i], O[i]);
      M = mn;
    }
  }
  uint16_t *op = a.out + ((long long)(a.chunk_row[c] + t) * a.H + h) * kD + d0;
#pragma unroll
  for (int i = 0; i < 4; i++)
    *(uint2 *)(op + 32 * i) = make_uint2(pack_bf16x2(O[4 * i], O[4 * i + 1]), pack_bf16x2(O[4 * i + 2], O[4 * i + 3]));
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
  if (workspace_bytes < need)
    return jit::fail(JIT_EINVAL, "paged_decode_attn_kv8: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                     (long long)need);
  if (!q || !pool || !page_table || !lens || !out || (need > 0 && !workspace))
    return jit::fail(JIT_EINVAL, "paged_decode_attn_kv8: null pointer");
  if (((uintptr_t)q | (uintptr_t)pool | (uintptr_t)out | (uintptr_t)workspace) & 15)
    return jit::fail(JIT_EINVAL, "paged_decode_attn_kv8: q, the pool, the workspace and out must be 16-byte aligned");
  const int slots = kDecodeWgs * jit::cu_count();
  for (int b0 = 0; b0 < B; b0 += kDecodeSeqs) {
    const int nb = B - b0 < kDecodeSeqs ? B - b0 : kDecodeSeqs;
    const int64_t rows = (int64_t)b0 * H, parts = (int64_t)nb * ncap * H;
    float *part_o = (float *)workspace + rows * ncap * (kD + 2);
    const DecodeArgs a{q + rows * kD, (const uint8_t *)pool, page_table + (int64_t)b0 * max_pages, lens + b0, part_o,
                       need ? part_o + parts * kD : nullptr, out + rows * kD, num_pages, max_pages, nb, H, Hkv, H / Hkv,
                       most, ncap, scale * 1.44269504088896341f};
    const int64_t chunks = (int64_t)nb * ncap, at_once = slots / Hkv > 1 ? slots / Hkv : 1;
    kv8_decode_kernel<<<dim3((unsigned)(chunks < at_once ? chunks : at_once), Hkv), 64 * kSplits, 8 * nb,
                        (hipStream_t)stream>>>(a);
    int rc = jit::check_launch("jit_paged_decode_attn_kv8");
    if (rc) return rc;
    if (ncap == 1) continue;
    kv8_merge_kernel<<<dim3(nb, H), 32 * kMergeLanes, 0, (hipStream_t)stream>>>(a);
    rc = jit::check_launch("jit_paged_decode_attn_kv8");
    if (rc) return rc;
  }
  return JIT_OK;
}

namespace {
// (infos padded to 16 bytes: the partials behind them are read 16 bytes at a time)
int64_t units_bytes(int units, int Hkv) { return (int64_t)units * Hkv * kUnitBytes + ((int64_t)units * Hkv * 8 + 15) / 16 * 16; }
}  // namespace

extern "C" int jit_kv8_prefill_block_tokens(int H, int Hkv) {
  if (H <= 0 || Hkv <= 0 || H % Hkv != 0 || 16 % (H / Hkv) != 0) return -1;
  return kBlockRows / (H / Hkv);
}

// Keys are cut where a chunk has too few row blocks to fill 256 CUs evenly.  `lines` row blocks of n parts are
// lines x n workgroups, whose time is that of the rounds they take on 256 CUs: about 1.88 us a unit for the two that
// share a CU and 1.15 us for one alone, 4 units' time for a workgroup's start and end, and 3 us and 0.02 a workgroup for
// the partials and their merge.  The n with the least of that, by the chunk alone, so that a row's bits do not depend on
// the call's other chunks.  All three launches, against parts of a fixed 6,144 keys (32 query heads over 4): 16 rows after
// 8,000 keys 35 us in 15 parts, 115 us; 512 rows after 8,000 90 us in 4, 116 us; 512 of 16 heads over 16 after 4,000 49 us
// in 4, 92 us; 2,048 rows after 8,192 305 to 316 us in one, 318 to 329 in two.
extern "C" int jit_kv8_prefill_part_units(int ctx, int len, int H, int Hkv) {
  const int bt = jit_kv8_prefill_block_tokens(H, Hkv);
  if (bt < 0 || ctx < 0 || len < 1) return -1;
  const int64_t lines = ((int64_t)len + bt - 1) / bt * Hkv, units = ((int64_t)ctx + len + kUnitKeys - 1) / kUnitKeys;
  int64_t best = 0, pu = 0;
  for (int64_t n = (units + kPartMax - 1) / kPartMax; n == 1 || 8 * n <= units; n++) {
    const int64_t part = (units + n - 1) / n, jobs = lines * n, rounds = (jobs + 255) / 256;
    const int64_t cost = (rounds / 2 * 188 + rounds % 2 * 115) * (part + 4) + (n > 1 ? 300 + 2 * jobs : 0);  // (us / 100)
    if (!pu || cost < best) best = cost, pu = part;
    if (jobs > 4 * 256) break;  // (more rounds of shorter workgroups: nothing left to even out)
  }
  return (int)pu;
}

extern "C" int jit_kv8_prefill_plan(const int32_t *ctx, const int32_t *len, int C, int H, int Hkv, int32_t *tables,
                                    int32_t *blocks, int n) {
  const int bt = jit_kv8_prefill_block_tokens(H, Hkv);
  if (bt < 0)
    return jit::fail(JIT_EUNSUPPORTED, "kv8_prefill_plan covers H / Hkv in {1, 2, 4, 8, 16}, got %d / %d", H, Hkv);
  if (C < 0 || (C > 0 && (!ctx || !len)) || !tables) return jit::fail(JIT_EINVAL, "kv8_prefill_plan: null pointer or C=%d", C);
  int64_t units = 0, slots = 0, at[kPartMax + 1] = {};  // at[w]: items of w units, then where the next of them goes
  auto items = [&](auto &&f) {
    for (int c = 0; c < C; c++) {
      const int pu = tables[C + 1 + c];
      for (int64_t q0 = 0; q0 < len[c]; q0 += bt) {
        const int64_t keys = (int64_t)ctx[c] + (q0 + bt < len[c] ? q0 + bt : len[c]), nu = (keys + kUnitKeys - 1) / kUnitKeys;
        for (int64_t u = 0; u < nu; u += pu) f(c, (int)q0, (int)(u / pu), (int)(nu - u < pu ? nu - u : pu));
      }
    }
  };
  for (int c = 0; c < C; c++) {
    const int pu = jit_kv8_prefill_part_units(ctx[c], len[c], H, Hkv);
    if (pu < 0) return jit::fail(JIT_EINVAL, "kv8_prefill_plan: chunk %d of %d rows after %d", c, len[c], ctx[c]);
    const int64_t nu = ((int64_t)ctx[c] + len[c] + kUnitKeys - 1) / kUnitKeys, parts = (nu + pu - 1) / pu;
    tables[c] = (int32_t)units, tables[C + 1 + c] = pu, tables[2 * (C + 1) + c] = (int32_t)slots;
    units += nu;
    slots += parts > 1 ? parts * len[c] : 0;
    if (units > 0x7fffffff || slots > 0x7fffffff)
      return jit::fail(JIT_EUNSUPPORTED, "kv8_prefill_plan covers up to 2^31 - 1 units and partials");
  }
  tables[C] = (int32_t)units, tables[2 * C + 1] = 0, tables[3 * C + 2] = (int32_t)slots;
  int64_t total = 0;
  items([&](int, int, int, int w) { at[w]++, total++; });
  if (total > 0x7fffffff) return jit::fail(JIT_EUNSUPPORTED, "kv8_prefill_plan: %lld work items", (long long)total);
  if (!blocks) return (int)total;
  if (n != total) return jit::fail(JIT_EINVAL, "kv8_prefill_plan: %d work items, %lld needed", n, (long long)total);
  for (int64_t w = kPartMax, next = 0; w > 0; w--) {  // the items with the most units first
    const int64_t of = at[w];
    at[w] = next;
    next += of;
  }
  items([&](int c, int q0, int part, int w) {
    const int64_t i = at[w]++;
    blocks[i] = c, blocks[n + i] = q0, blocks[2 * (int64_t)n + i] = part;
  });
  return (int)total;
}

extern "C" int64_t jit_kv8_prefill_workspace_bytes(int H, int Hkv, int units, int slots) {
  if (H <= 0 || Hkv <= 0 || units < 0 || slots < 0) return -1;
  return units_bytes(units, Hkv) + (int64_t)slots * H * kPfSlot * (int64_t)sizeof(float);
}

extern "C" int jit_paged_prefill_attn_kv8(const uint16_t *q, const void *pool, int num_pages, const int32_t *page_table,
                                          int max_pages, const int32_t *chunk_seq, const int32_t *chunk_ctx,
                                          const int32_t *chunk_len, const int32_t *chunk_row, const int32_t *chunk_unit,
                                          const int32_t *chunk_part, const int32_t *chunk_slot, int C, int units,
                                          int slots, const int32_t *blk_chunk, const int32_t *blk_q0,
                                          const int32_t *blk_part, int nblk, int max_len, int H, int Hkv, float scale,
                                          void *workspace, int64_t workspace_bytes, uint16_t *out, void *stream) {
  if (C < 0 || nblk < 0 || units < 0 || slots < 0 || H <= 0 || Hkv <= 0 || max_pages <= 0 || num_pages <= 0 || max_len < 0)
    return jit::fail(JIT_EINVAL, "paged_prefill_attn_kv8: bad dims C=%d nblk=%d H=%d Hkv=%d max_len=%d units=%d slots=%d", C,
                     nblk, H, Hkv, max_len, units, slots);
  if (H % Hkv != 0) return jit::fail(JIT_EINVAL, "%d query heads do not share %d KV heads evenly", H, Hkv);
  if (!(scale > 0.0f)) return jit::fail(JIT_EINVAL, "paged_prefill_attn_kv8: the scale must be positive");
  if (16 % (H / Hkv) != 0)
    return jit::fail(JIT_EUNSUPPORTED, "paged_prefill_attn_kv8 covers H / Hkv in {1, 2, 4, 8, 16}, got %d", H / Hkv);
  if (C > 65535 || Hkv > 65535 || (int64_t)nblk * Hkv > 0x7fffffff)
    return jit::fail(JIT_EUNSUPPORTED, "paged_prefill_attn_kv8 covers up to 65535 chunks and heads, got %d and %d", C, Hkv);
  if (C == 0 || nblk == 0) return JIT_OK;
  const int64_t need = jit_kv8_prefill_workspace_bytes(H, Hkv, units, slots);
  if (units == 0 || workspace_bytes < need)
    return jit::fail(JIT_EINVAL, "paged_prefill_attn_kv8: workspace of %lld bytes for %d units, %lld needed",
                     (long long)workspace_bytes, units, (long long)need);
  if (!q || !pool || !page_table || !chunk_seq || !chunk_ctx || !chunk_len || !chunk_row || !chunk_unit || !chunk_part ||
      !chunk_slot || !blk_chunk || !blk_q0 || !blk_part || !out || !workspace)
    return jit::fail(JIT_EINVAL, "paged_prefill_attn_kv8: null pointer");
  if (((uintptr_t)q | (uintptr_t)pool | (uintptr_t)out | (uintptr_t)workspace) & 15)
    return jit::fail(JIT_EINVAL, "paged_prefill_attn_kv8: q, the pool, the workspace and out must be 16-byte aligned");
  uint8_t *ws = (uint8_t *)workspace;
  int32_t *info = (int32_t *)(ws + (int64_t)units * Hkv * kUnitBytes);
  const PrefillArgs a{q, (const uint8_t *)pool, page_table, blk_chunk, blk_q0, blk_part, chunk_seq, chunk_ctx, chunk_len,
                      chunk_row, chunk_unit, chunk_part, chunk_slot, out, ws, info,
                      (float *)(ws + units_bytes(units, Hkv)), num_pages, max_pages, H, Hkv, H / Hkv, C, units, slots,
                      scale * 1.44269504088896341f};
  const hipStream_t st = (hipStream_t)stream;
  kv8_expand_kernel<<<dim3(units, Hkv), 256, 0, st>>>(a);
  int rc = jit::check_launch("jit_paged_prefill_attn_kv8");
  if (rc) return rc;
  kv8_prefill_kernel<<<dim3(nblk * Hkv), 64 * kPfWaves, 0, st>>>(a);
  rc = jit::check_launch("jit_paged_prefill_attn_kv8");
  if (rc || slots == 0 || max_len == 0) return rc;
  kv8_prefill_merge_kernel<<<dim3(max_len, C, (H + 15) / 16), 128, 0, st>>>(a);
  return jit::check_launch("jit_paged_prefill_attn_kv8");
}
