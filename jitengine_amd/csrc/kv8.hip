// The 8-bit KV cache's writes, page copies and step tables for gfx950 (records and number format: kv8.hpp).
#include "kv8.hpp"

namespace {

using namespace kv8;

// A wave writes one head of 4 consecutive rows (tokens), 16 lanes a row: lane x of a row has dims 4 x .. + 3 and 64 + 4 x ..
// + 3, so RoPE's pairs (i, i + 64) are its own, and a norm or a largest magnitude is four lane exchanges.  Bound by
// latency up to some hundred rows (32 rows of 32 + 2 x 4 heads: 3.4 us, an empty launch 2.5), past that by memory: 2,108
// such rows read 21.6 MB and write 17.3 MB of q and 2.2 MB of codes in 12.4 us (3.3 TB/s; a copy reaches 4.8), 11.3 to 11.7 at
// consecutive slots: V's byte stores are 1 us of it.  A wave a row, two dims a lane, took 20.7 us: its V codes went out
// two bytes a lane, and every wave formed 64 sines.

// Sum or maximum over the 16 lanes of a row (lanes l ^ 1, l ^ 2, then mirrored in 8 and in 16).
template <bool MAX>
__device__ __forceinline__ float row16(float v) {
  auto op = [](float a, float b) { return MAX ? fmaxf(a, b) : a + b; };
  v = op(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, true)));
  v = op(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, true)));
  v = op(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xF, 0xF, true)));
  return op(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xF, 0xF, true)));
}

struct Raw8 {
  uint2 w[2];
};
__device__ __forceinline__ Raw8 load8(const uint16_t *src, int x) {
  return {{*(const uint2 *)(src + 4 * x), *(const uint2 *)(src + 64 + 4 * x)}};
}
__device__ __forceinline__ void widen8(const Raw8 &r, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 2; i++) {
    v[4 * i] = bf2f(r.w[i].x & 0xffffu), v[4 * i + 1] = bf2f_hi(r.w[i].x);
    v[4 * i + 2] = bf2f(r.w[i].y & 0xffffu), v[4 * i + 3] = bf2f_hi(r.w[i].y);
  }
}

// cos and sin of a row's position times the lane's four inverse frequencies.  The angle is formed in fp64 and brought
// there into [-pi/4, pi/4] about a quarter turn k (at position 262,143 an fp32 product is off by up to 0.016 rad);
// sine and cosine of the rest are their Taylor series to r^9 and r^10 (2e-9 off at most, 9e-8 with fp32's roundings).
__device__ __forceinline__ void rotation(int pos, const float *inv_freq, int x, float (&cs)[4], float (&sn)[4]) {
  const float4 f = *(const float4 *)(inv_freq + 4 * x);
  const float *fp = (const float *)&f;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const double ang = (double)pos * (double)fp[i], k = __builtin_rint(ang * 0.6366197723675814);
    const float r = (float)__builtin_fma(-k, 6.123233995736766e-17, __builtin_fma(-k, 1.5707963267948966, ang));
    const int quarter = (int)(long long)k;
    const float z = r * r;
    const float s = fmaf(r * z, fmaf(z, fmaf(z, fmaf(z, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), r);
    const float c = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
    const float a = quarter & 1 ? c : s, b = quarter & 1 ? s : c;  // sine and cosine but for their signs
    sn[i] = quarter & 2 ? -a : a;
    cs[i] = (quarter + 1) & 2 ? -b : b;
  }
}

// RMSNorm with weights w and the rotation, in fp32 with no rounding in between (q is rounded to bf16, k to its codes,
// once).
__device__ __forceinline__ void norm_rope(float (&v)[8], const float (&w)[8], float eps, const float (&cs)[4],
                                          const float (&sn)[4]) {
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; i++) ss = fmaf(v[i], v[i], ss);
  const float r = rsqrtf(row16<false>(ss) * (1.0f / 128.0f) + eps);
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float a = v[i] * r * w[i], b = v[i + 4] * r * w[i + 4];
    v[i] = a * cs[i] - b * sn[i];
    v[i + 4] = a * sn[i] + b * cs[i];
  }
}

// Byte k of four words, in order.
__device__ __forceinline__ uint32_t byte_of(uint32_t t0, uint32_t t1, uint32_t t2, uint32_t t3, int k) {
  const uint32_t lo = __builtin_amdgcn_perm(t1, t0, 0x0c0c0400u + 0x0101u * k);  // (0x0c: a zero byte)
  const uint32_t hi = __builtin_amdgcn_perm(t3, t2, 0x0c0c0400u + 0x0101u * k);
  return lo | (hi << 16);
}

template <int J>
__device__ __forceinline__ uint32_t lane_of_quad(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x55 * J, 0xF, 0xF, true);
}

// The wave's blocks into their records: rec and slot of the lane's row (on: whether it is written); quad: the rows are
// the 4 slots of one of V's words (uniform), which then go as words of 4 slots, else V's codes go byte by byte (1,001
// rows of 16 + 16 heads at consecutive slots: 4.9 us as words; 6.0 as bytes, where the run's first row of the call is not a
// word's first slot; at scattered slots 7.0).
__device__ __forceinline__ void store_blocks(uint8_t *rec, int slot, bool on, bool is_v, bool quad, int l, const float (&v)[8]) {
  const int x = l & 15, k = l >> 4;
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; i++) amax = fmaxf(amax, mag(v[i]));
  amax = row16<true>(amax);
  const int e = scale_exp(amax);
  const float inv = exp_bits(-e);
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; i++) y[i] = to_code_range(v[i], inv);
  uint32_t c[2];
#pragma unroll
  for (int i = 0; i < 2; i++) c[i] = codes2(y[4 * i], y[4 * i + 1]) | (codes2(y[4 * i + 2], y[4 * i + 3]) << 16);
  if (on && x == 0) ((float *)(rec + kScaleOff))[(is_v ? kPage : 0) + slot] = exp_bits(e);
  if (!is_v) {
    if (on) {
      uint8_t *p = rec + (x >> 2) * 256 + slot * 16 + 4 * (x & 3);
      *(uint32_t *)p = c[0];
      *(uint32_t *)(p + 1024) = c[1];
    }
  } else if (quad) {
    // every lane gets the four rows' words of its dims; row k stores dim 4 x + k (of each 64)
    uint8_t *p = rec + kVOff + (slot >> 2) * 256 + (4 * (x & 3) + k) * 16 + (x >> 2) * 4;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const auto a = __builtin_amdgcn_permlane16_swap(c[i], c[i], false, false);  // rows 0 (2) and 1 (3)
      const auto b = __builtin_amdgcn_permlane32_swap(a[0], a[0], false, false);  // rows 0 and 2
      const auto d = __builtin_amdgcn_permlane32_swap(a[1], a[1], false, false);  // rows 1 and 3
      *(uint32_t *)(p + 1024 * i) = byte_of(b[0], d[0], b[1], d[1], k);
    }
  } else {
    // Byte stores: a lane first gets byte x % 4 of its four lanes' words, so that a store instruction writes 16 bytes of
    // one 64-byte segment a row and not 4 of each of four.
    uint8_t *p = rec + kVOff + (slot >> 2) * 256 + (x & 3) * 16 + (x >> 2) * 4 + (slot & 3);
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const uint32_t t = byte_of(lane_of_quad<0>(c[i]), lane_of_quad<1>(c[i]), lane_of_quad<2>(c[i]), lane_of_quad<3>(c[i]), x & 3);
      if (on) {
#pragma unroll
        for (int j = 0; j < 4; j++) p[1024 * i + 64 * j] = (uint8_t)(t >> (8 * j));
      }
    }
  }
}

// A lane's row of 4 rows from row0: its place in the pool.
struct Place {
  int b, slot, page;
  bool in, on, quad;  // a row of the call; written; the four are a word's slots
};
__device__ __forceinline__ Place place_of(int row0, int B, const int32_t *slots, int num_pages, int l) {
  Place p;
  p.b = min(row0 + (l >> 4), B - 1);
  p.in = row0 + (l >> 4) < B;
  const int s = slots[p.b];
  p.page = s / kPage;
  p.slot = s % kPage;
  p.on = p.in && s >= 0 && p.page < num_pages;
  const int s0 = __builtin_amdgcn_readfirstlane(s);
  p.quad = __all(p.on && s == s0 + (l >> 4) && s0 % 4 == 0);
  if (!p.on) p.page = p.slot = 0;
  return p;
}

__global__ __launch_bounds__(256) void kv8_append_kernel(const uint16_t *__restrict__ k, const uint16_t *__restrict__ v,
                                                         int B, int Hkv, const int32_t *__restrict__ slots,
                                                         uint8_t *__restrict__ pool, int num_pages) {
  const int l = lane_id(), unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (unit >= 2 * Hkv) return;
  const Place p = place_of(4 * blockIdx.y, B, slots, num_pages, l);
  auto src = [&](int head) {
    return (head >= Hkv ? v : k) + ((long long)p.b * Hkv + (head >= Hkv ? head - Hkv : head)) * kD;
  };
  const int step = 4 * gridDim.x;
  Raw8 next = load8(src(unit), l & 15);
  for (int head = unit; head < 2 * Hkv; head += step) {
    float x[8];
    widen8(next, x);
    if (head + step < 2 * Hkv) next = load8(src(head + step), l & 15);
    const bool is_v = head >= Hkv;
    store_blocks(record(pool, p.page, Hkv, is_v ? head - Hkv : head), p.slot, p.on, is_v, p.quad, l, x);
  }
}

// The fused rows [q: H * 128 | k: Hkv * 128 | v: Hkv * 128].
__global__ __launch_bounds__(256) void qk_norm_rope_append_kv8_kernel(
    const uint16_t *__restrict__ qkv, int B, int H, int Hkv, const uint16_t *__restrict__ qn_w,
    const uint16_t *__restrict__ kn_w, float eps, const float *__restrict__ inv_freq, const int32_t *__restrict__ pos,
    const int32_t *__restrict__ slots, uint8_t *__restrict__ pool, int num_pages, uint16_t *__restrict__ q_out) {
  const int l = lane_id(), unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nh = H + 2 * Hkv;
  if (unit >= nh) return;
  const Place p = place_of(4 * blockIdx.y, B, slots, num_pages, l);
  const int step = 4 * gridDim.x;
  const uint16_t *row = qkv + (long long)p.b * nh * kD;
  Raw8 next = load8(row + unit * kD, l & 15);
  float w[8], cs[4], sn[4];
  widen8(load8(unit < H ? qn_w : kn_w, l & 15), w);
  if (unit < H + Hkv) rotation(pos[p.b], inv_freq, l & 15, cs, sn);
  for (int head = unit; head < nh; head += step) {
    float x[8];
    widen8(next, x);
    if (head + step < nh) next = load8(row + (head + step) * kD, l & 15);  // (in flight beside this head's work)
    if (head < H + Hkv) {
      if (head >= H && head - step < H && head > unit) widen8(load8(kn_w, l & 15), w);
      norm_rope(x, w, eps, cs, sn);
    }
    if (head < H) {
      if (!p.in) continue;
      uint16_t *qo = q_out + ((long long)p.b * H + head) * kD + 4 * (l & 15);
#pragma unroll
      for (int i = 0; i < 2; i++)
        *(uint2 *)(qo + 64 * i) =
            make_uint2(pack_bf16x2(x[4 * i], x[4 * i + 1]), pack_bf16x2(x[4 * i + 2], x[4 * i + 3]));
    } else {
      const bool is_v = head >= H + Hkv;
      store_blocks(record(pool, p.page, Hkv, head - H - (is_v ? Hkv : 0)), p.slot, p.on, is_v, p.quad, l, x);
    }
  }
}

// Blocks of 4 waves a group of rows: one head a wave up to 1,024 blocks (what 256 CUs hold of them at once), else that
// many, whose waves loop over the heads and form their rows' rotations once.  2,108 rows of 32 + 2 x 4 heads with 512,
// 1,024, 2,048 and 4,096 blocks: 14.1, 12.2, 15.3 and 19.5 us; 300 rows: 5.2, 4.6, 4.6 and 4.5.
int head_blocks(int rows, int heads) {
  const int groups = (rows + 3) / 4, all = (heads + 3) / 4, want = (1024 + groups - 1) / groups;
  return want < all ? want : all;
}

// Workgroup i copies page src[i] to page dst[i]; a page id outside the pool copies nothing.
__global__ __launch_bounds__(256) void kv8_copy_pages_kernel(uint4 *__restrict__ pool, const int32_t *__restrict__ src,
                                                             const int32_t *__restrict__ dst, int page_words,
                                                             int num_pages) {
  const int ps = src[blockIdx.x], pd = dst[blockIdx.x];
  if (ps < 0 || ps >= num_pages || pd < 0 || pd >= num_pages) return;
  const long long s = (long long)ps * page_words, d = (long long)pd * page_words;
  for (int j = threadIdx.x; j < page_words; j += blockDim.x) pool[d + j] = pool[s + j];
}

// ---------------------------------------------------------------- step tables
// Every workgroup scans all S sequences itself (a few thousand integers out of L2) and then writes the entries of
// its own rows: no workgroup waits for another, and the tables take one launch.  Bound by latency (the lengths, two
// scans, a table entry): 4.1 us for one sequence, 6.1 for 1,024 with 9,208 rows; an empty launch takes 2.5.
constexpr int kTabThreads = 1024, kTabRows = 1024, kTabSeqs = JIT_STEP_TABLES_MAX_SEQS;

struct TableArgs {
  const int32_t *ctx, *fresh, *free_pages, *free_at;
  int32_t *table, *row_start, *row_seq, *pos, *slots, *lens, *status;
  int S, max_pages, rows, n_free;  // n_free < 0: the tables hold the step's pages already
};

// Inclusive scan of one value a thread over the workgroup (red: 16 words of LDS).
__device__ __forceinline__ long long block_scan(long long v, long long *red) {
  const int l = lane_id(), w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long long u = __shfl_up(v, o, 64);
    if (l >= o) v += u;
  }
  if (l == 63) red[w] = v;
  __syncthreads();
  long long add = 0;
  for (int i = 0; i < w; i++) add += red[i];
  __syncthreads();
  return v + add;
}

__device__ __forceinline__ int sat(long long v) { return v > 0x7fffffffLL ? 0x7fffffff : (int)v; }

__global__ __launch_bounds__(kTabThreads) void step_tables_kernel(const TableArgs a) {
  __shared__ int32_t s_end[kTabSeqs], s_base[kTabSeqs];  // rows up to and with b; pages before b (-1: refused)
  __shared__ long long red[kTabThreads / 64];
  __shared__ int s_refused, s_next;
  const int t = threadIdx.x;
  const bool first = blockIdx.x == 0;
  const int free_at = a.free_at ? max(*a.free_at, 0) : 0;
  if (t == 0) s_refused = 0, s_next = free_at;
  long long rows0 = 0, pages0 = free_at;  // of the sequences of earlier rounds
  for (int b0 = 0; b0 < a.S; b0 += kTabThreads) {
    const int b = b0 + t;
    const bool on = b < a.S;
    const long long ctx = on ? max(a.ctx[b], 0) : 0, add = on ? max(a.fresh[b], 0) : 0;
    const long long end = rows0 + block_scan(add, red);
    const long long have = (ctx + kPage - 1) / kPage, tot = (ctx + add + kPage - 1) / kPage;
    const bool fits = tot <= a.max_pages && end <= a.rows;
    const long long need = on && fits && a.n_free >= 0 ? tot - have : 0;
    const long long cum = pages0 + block_scan(need, red);
    const bool served = fits && (need == 0 || cum <= a.n_free);
    if (on) {
      s_end[b] = sat(end);
      s_base[b] = served ? sat(cum - need) : -1;
      if (first) {
        a.row_start[b + 1] = sat(end);
        a.lens[b] = sat(ctx + (served ? add : 0));
        if (!served) atomicAdd(&s_refused, 1);
        if (served && need) atomicMax(&s_next, sat(cum));
      }
    }
    if (t == kTabThreads - 1) red[0] = end, red[1] = cum;
    __syncthreads();
    rows0 = red[0];
    pages0 = red[1];
    __syncthreads();
  }
  if (first && t == 0) {
    a.row_start[0] = 0;
    a.status[0] = sat(rows0);
    a.status[1] = s_next;
    a.status[2] = s_refused;
    a.status[3] = 0;
  }
  const int r = blockIdx.x * kTabRows + t;
  if (r >= a.rows) return;
  int lo = 0, hi = a.S;  // the first sequence whose rows end past r
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (s_end[mid] > r) hi = mid;
    else lo = mid + 1;
  }
  const int b = lo;
  if (b >= a.S) {
    a.row_seq[r] = -1;
    a.pos[r] = 0;
    a.slots[r] = -1;
    return;
  }
  const int ctx = max(a.ctx[b], 0), pos = sat((long long)ctx + r - (b ? s_end[b - 1] : 0));
  const int base = s_base[b], pi = pos / kPage, have = (int)(((long long)ctx + kPage - 1) / kPage);
  int slot = -1;
  if (base >= 0) {  // (served: pi < max_pages, and its new pages lie in the list)
    int32_t *entry = a.table + (long long)b * a.max_pages + pi;
    int page;
    if (a.n_free >= 0 && pi >= have) {
      page = a.free_pages[base + pi - have];
      if (pos % kPage == 0) *entry = page;
    } else {
      page = *entry;
    }
    if (page >= 0 && page < (1 << 27)) slot = page * kPage + pos % kPage;
  }
  a.row_seq[r] = b;
  a.pos[r] = pos;
  a.slots[r] = slot;
}

}  // namespace

extern "C" int jit_kv8_append_paged(const uint16_t *k, const uint16_t *v, int B, int Hkv, const int32_t *slots, void *pool,
                                    int num_pages, void *stream) {
  if (B < 0 || Hkv <= 0 || num_pages <= 0)
    return jit::fail(JIT_EINVAL, "kv8_append_paged: bad dims B=%d Hkv=%d num_pages=%d", B, Hkv, num_pages);
  if (B > 65535) return jit::fail(JIT_EUNSUPPORTED, "kv8_append_paged covers up to 65535 rows, got %d", B);
  if (B == 0) return JIT_OK;
  if (!k || !v || !slots || !pool) return jit::fail(JIT_EINVAL, "kv8_append_paged: null pointer");
  if (((uintptr_t)pool & 15) || (((uintptr_t)k | (uintptr_t)v) & 7))
    return jit::fail(JIT_EINVAL, "kv8_append_paged: the pool must be 16-byte, k and v 8-byte aligned");
  kv8_append_kernel<<<dim3(head_blocks(B, 2 * Hkv), (B + 3) / 4), 256, 0, (hipStream_t)stream>>>(
      k, v, B, Hkv, slots, (uint8_t *)pool, num_pages);
  return jit::check_launch("jit_kv8_append_paged");
}

extern "C" int jit_qk_norm_rope_append_kv8(const uint16_t *qkv, int B, int H, int Hkv, const uint16_t *q_norm_w,
                                           const uint16_t *k_norm_w, float eps, const float *inv_freq,
                                           const int32_t *pos, const int32_t *slots, void *pool, int num_pages,
                                           uint16_t *q_out, void *stream) {
  if (B < 0 || H <= 0 || Hkv <= 0 || num_pages <= 0)
    return jit::fail(JIT_EINVAL, "qk_norm_rope_append_kv8: bad dims B=%d H=%d Hkv=%d num_pages=%d", B, H, Hkv, num_pages);
  if (H % Hkv != 0) return jit::fail(JIT_EINVAL, "%d query heads do not share %d KV heads evenly", H, Hkv);
  if (B > 65535) return jit::fail(JIT_EUNSUPPORTED, "qk_norm_rope_append_kv8 covers up to 65535 rows, got %d", B);
  if (B == 0) return JIT_OK;
  if (!qkv || !q_norm_w || !k_norm_w || !inv_freq || !pos || !slots || !pool || !q_out)
    return jit::fail(JIT_EINVAL, "qk_norm_rope_append_kv8: null pointer");
  if ((((uintptr_t)pool | (uintptr_t)inv_freq) & 15) ||
      (((uintptr_t)qkv | (uintptr_t)q_norm_w | (uintptr_t)k_norm_w | (uintptr_t)q_out) & 7))
    return jit::fail(JIT_EINVAL, "qk_norm_rope_append_kv8: the pool and inv_freq must be 16-byte, the rows and norms "
                                 "8-byte aligned");
  qk_norm_rope_append_kv8_kernel<<<dim3(head_blocks(B, H + 2 * Hkv), (B + 3) / 4), 256, 0, (hipStream_t)stream>>>(
      qkv, B, H, Hkv, q_norm_w, k_norm_w, eps, inv_freq, pos, slots, (uint8_t *)pool, num_pages, q_out);
  return jit::check_launch("jit_qk_norm_rope_append_kv8");
}

extern "C" int jit_kv8_copy_pages(void *pool, int num_pages, int Hkv, const int32_t *src, const int32_t *dst, int n,
                                  void *stream) {
  if (n < 0 || Hkv <= 0 || num_pages <= 0)
    return jit::fail(JIT_EINVAL, "kv8_copy_pages: bad dims n=%d Hkv=%d num_pages=%d", n, Hkv, num_pages);
  if (n == 0) return JIT_OK;
  if (!pool || !src || !dst) return jit::fail(JIT_EINVAL, "kv8_copy_pages: null pointer");
  if ((uintptr_t)pool & 15) return jit::fail(JIT_EINVAL, "kv8_copy_pages: the pool must be 16-byte aligned");
  kv8_copy_pages_kernel<<<n, 256, 0, (hipStream_t)stream>>>((uint4 *)pool, src, dst, Hkv * (kRec / 16), num_pages);
  return jit::check_launch("jit_kv8_copy_pages");
}

extern "C" int jit_step_tables(const int32_t *ctx, const int32_t *new_rows, int S, int32_t *page_table, int max_pages,
                               int rows, const int32_t *free_pages, int n_free, const int32_t *free_at,
                               int32_t *row_start, int32_t *row_seq, int32_t *pos, int32_t *slots, int32_t *lens,
                               int32_t *status, void *stream) {
  if (S < 0 || max_pages <= 0 || rows < 0)
    return jit::fail(JIT_EINVAL, "step_tables: bad dims S=%d max_pages=%d rows=%d", S, max_pages, rows);
  if (S > kTabSeqs)
    return jit::fail(JIT_EUNSUPPORTED, "step_tables covers up to %d sequences, got %d", kTabSeqs, S);
  if (!row_start || !status || (S > 0 && (!ctx || !new_rows || !page_table || !lens)) ||
      (rows > 0 && (!row_seq || !pos || !slots)) || (n_free > 0 && !free_pages))
    return jit::fail(JIT_EINVAL, "step_tables: null pointer");
  const TableArgs a{ctx, new_rows, free_pages, free_at, page_table, row_start, row_seq, pos, slots, lens, status,
                    S, max_pages, rows, n_free};
  const int blocks = rows > kTabRows ? (int)(((long long)rows + kTabRows - 1) / kTabRows) : 1;
  step_tables_kernel<<<blocks, kTabThreads, 0, (hipStream_t)stream>>>(a);
  return jit::check_launch("jit_step_tables");
}
