// The 8-bit KV cache's writes, page copies and step tables for gfx950 (records and number format: kv8.hpp).
#include "kv8.hpp"

namespace {

using namespace kv8;

// One token's block of one head on a wave (lane l: dims l, l + 64): its codes and scale into the record.
__device__ __forceinline__ void store_block(uint8_t *rec, int slot, bool is_v, int l, float x1, float x2) {
  const float amax = wave_butterfly<true>(fmaxf(mag(x1), mag(x2)));
  const int e = scale_exp(amax);
  const float inv = exp_bits(-e);
  const uint32_t c = codes2(to_code_range(x1, inv), to_code_range(x2, inv));
  const int at = is_v ? v_at(slot, l) : k_at(slot, l);  // (dim l + 64 lies 1,024 bytes on in either part)
  rec[at] = (uint8_t)c;
  rec[at + 1024] = (uint8_t)(c >> 8);
  if (l == 0) ((float *)(rec + kScaleOff))[(is_v ? kPage : 0) + slot] = exp_bits(e);
}

// One head of one token: RMSNorm with weights w1, w2 (dims l, l + 64) and the rotation by pos * f, in fp32 with no
// rounding in between (q is rounded to bf16, k to its codes, once).  The angle is formed and brought into one turn
// in fp64: at position 262,143 an fp32 product is off by up to 0.016 rad.
__device__ __forceinline__ void norm_rope(float &x1, float &x2, float w1, float w2, float eps, int pos, float f) {
  float ss = __builtin_fmaf(x1, x1, x2 * x2);
  ss = wave_butterfly<false>(ss);
  const float r = rsqrtf(ss * (1.0f / 128.0f) + eps);
  const float y1 = x1 * r * w1, y2 = x2 * r * w2;
  const double ang = (double)pos * (double)f;
  const double turns = __builtin_rint(ang * 0.15915494309189535);
  double red = __builtin_fma(-turns, 6.283185307179586, ang);
  red = __builtin_fma(-turns, 2.4492935982947064e-16, red);
  float sn, cs;
  sincosf((float)red, &sn, &cs);
  x1 = y1 * cs - y2 * sn;
  x2 = y1 * sn + y2 * cs;
}

// One wave per (token, kv head, K or V).
__global__ __launch_bounds__(256) void kv8_append_kernel(const uint16_t *__restrict__ k, const uint16_t *__restrict__ v,
                                                         int Hkv, const int32_t *__restrict__ slots,
                                                         uint8_t *__restrict__ pool, int num_pages) {
  const int b = blockIdx.y, l = lane_id();
  const int head = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int s = slots[b];
  if (head >= 2 * Hkv || s < 0 || s / kPage >= num_pages) return;
  const bool is_v = head >= Hkv;
  const int h = is_v ? head - Hkv : head;
  const uint16_t *src = (is_v ? v : k) + ((long long)b * Hkv + h) * kD;
  store_block(record(pool, s / kPage, Hkv, h), s % kPage, is_v, l, bf2f(src[l]), bf2f(src[l + 64]));
}

// One wave per (token, head) of the fused row [q: H * 128 | k: Hkv * 128 | v: Hkv * 128].
__global__ __launch_bounds__(256) void qk_norm_rope_append_kv8_kernel(
    const uint16_t *__restrict__ qkv, int H, int Hkv, const uint16_t *__restrict__ qn_w,
    const uint16_t *__restrict__ kn_w, float eps, const float *__restrict__ inv_freq, const int32_t *__restrict__ pos,
    const int32_t *__restrict__ slots, uint8_t *__restrict__ pool, int num_pages, uint16_t *__restrict__ q_out) {
  const int b = blockIdx.y, l = lane_id();
  const int head = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int nh = H + 2 * Hkv;
  if (head >= nh) return;
  const uint16_t *src = qkv + ((long long)b * nh + head) * kD;
  float x1 = bf2f(src[l]), x2 = bf2f(src[l + 64]);
  const bool is_v = head >= H + Hkv;
  if (!is_v) {
    const uint16_t *nw = head < H ? qn_w : kn_w;
    norm_rope(x1, x2, bf2f(nw[l]), bf2f(nw[l + 64]), eps, pos[b], inv_freq[l]);
    if (head < H) {
      uint16_t *qo = q_out + ((long long)b * H + head) * kD;
      qo[l] = (uint16_t)f2bf(x1);
      qo[l + 64] = (uint16_t)f2bf(x2);
      return;
    }
  }
  const int s = slots[b];
  if (s < 0 || s / kPage >= num_pages) return;
  const int h = head - H - (is_v ? Hkv : 0);
  store_block(record(pool, s / kPage, Hkv, h), s % kPage, is_v, l, x1, x2);
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
// its own rows: no workgroup waits for another, and the tables take one launch.
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
  if ((uintptr_t)pool & 15) return jit::fail(JIT_EINVAL, "kv8_append_paged: the pool must be 16-byte aligned");
  kv8_append_kernel<<<dim3((2 * Hkv + 3) / 4, B), 256, 0, (hipStream_t)stream>>>(k, v, Hkv, slots, (uint8_t *)pool,
                                                                                 num_pages);
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
  if ((uintptr_t)pool & 15) return jit::fail(JIT_EINVAL, "qk_norm_rope_append_kv8: the pool must be 16-byte aligned");
  qk_norm_rope_append_kv8_kernel<<<dim3((H + 2 * Hkv + 3) / 4, B), 256, 0, (hipStream_t)stream>>>(
      qkv, H, Hkv, q_norm_w, k_norm_w, eps, inv_freq, pos, slots, (uint8_t *)pool, num_pages, q_out);
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
