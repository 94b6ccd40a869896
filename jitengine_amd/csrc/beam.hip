// Sequences that are continued several times, for gfx950: the choice among their continuations, the page tables,
// reference counts and free list of the sequences that go on, and page copies in every layer.
#include "common.hpp"

namespace {

// ------------------------------------------------------------------ choice of continuations
// A group's candidates are (beam b, alternative j), c = b m + j, with score_b + logprob_bj (score_b alone, as alternative
// 0, for a beam that has ended).  One wave a group, candidate c in lane c % 64: the w-th largest score is found bit by bit
// from the top (up to 32 counts by ballot over order-preserving keys, until just w are left), candidates that tie with it
// are taken from the lowest c on, and the w chosen ones count how many of them stand before each.  Latency bounds it: one
// group of 4 x 8 candidates 3 us, 64 groups of 16 x 32 12 us.
constexpr int kMaxWidth = 64, kMaxCands = 4096;
constexpr long long kMaxLaunch = 0xffffffffLL;  // threads of a launch

struct BeamArgs {
  const float *scores, *lp;
  const int32_t *ids, *done, *eos;
  int32_t *parents, *tokens, *done_out;
  float *out;
  int G, n, m, w, n_eos;
};

// Keys rise with the value; 0 is no candidate (NaN and -inf are none).
__device__ __forceinline__ uint32_t key_of(float v) {
  if (!(v > -__builtin_inff())) return 0u;
  const uint32_t u = __float_as_uint(v + 0.0f);  // (-0 ties +0)
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

template <int NV>
__global__ __launch_bounds__(64) void beam_select_kernel(const BeamArgs a) {
  __shared__ uint32_t s_key[kMaxWidth];
  __shared__ int s_c[kMaxWidth];
  __shared__ float s_score[64 * NV];
  __shared__ bool s_done[64 * NV];
  const int g = blockIdx.x, l = lane_id(), cands = a.n * a.m;
  uint32_t key[NV];
  // (every load before the first use: clamped addresses in place of branches)
  float lp[NV];
  int32_t id[NV];
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const long long at = (long long)g * cands + min(64 * i + l, cands - 1);
    lp[i] = a.lp[at];
    id[i] = a.ids[at];
  }
  for (int b = l; b < a.n; b += 64) {  // (a beam that has ended: its score, and no other candidate)
    s_score[b] = a.scores[(long long)g * a.n + b];
    s_done[b] = a.done && a.done[(long long)g * a.n + b] != 0;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const int c = 64 * i + l, b = min(c, cands - 1) / a.m;
    const float s = s_score[b];
    const bool ended = s_done[b], is = ended ? c == b * a.m : id[i] >= 0;
    key[i] = c < cands && is ? key_of(ended ? s : s + lp[i]) : 0u;
  }
  auto count = [&](uint32_t least) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < NV; i++) n += __builtin_popcountll(__ballot(key[i] >= least));
    return n;
  };
  uint32_t least = 0u;  // the w-th largest key, or 1 where there are fewer candidates
  if (count(1u) > a.w) {
    for (int bit = 31; bit >= 0; bit--) {
      const int n = count(least | (1u << bit));
      if (n >= a.w) least |= 1u << bit;
      if (n == a.w) break;
    }
  } else {
    least = 1u;
  }
  // (left early, all that is not below `least` is wanted: ties are none too many then)
  int above = 0;
#pragma unroll
  for (int i = 0; i < NV; i++) above += __builtin_popcountll(__ballot(key[i] > least));
  const uint64_t below = ((uint64_t)1 << l) - 1;
  int at = 0, tied = a.w - above;  // places taken; candidates of key `least` still wanted
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const uint64_t tie = __ballot(key[i] == least);
    const bool take = key[i] > least || (key[i] == least && __builtin_popcountll(tie & below) < tied);
    const uint64_t all = __ballot(take);
    if (take) {
      const int p = at + __builtin_popcountll(all & below);
      s_key[p] = key[i];
      s_c[p] = 64 * i + l;
    }
    at += __builtin_popcountll(all);
    tied -= min(tied, __builtin_popcountll(tie));
  }
  __syncthreads();
  const long long o = (long long)g * a.w;
  if (l < at) {
    const uint32_t k = s_key[l];
    const int c = s_c[l];
    int r = 0;
    for (int j = 0; j < at; j++) r += s_key[j] > k || (s_key[j] == k && s_c[j] < c) ? 1 : 0;
    const int b = c / a.m;
    const bool ended = s_done[b];
    const int tok = ended ? -1 : a.ids[(long long)g * cands + c];
    bool end = ended;
    for (int e = 0; e < a.n_eos; e++) end |= tok == a.eos[e];
    a.parents[o + r] = g * a.n + b;
    a.tokens[o + r] = tok;
    a.out[o + r] = value_of(k);
    a.done_out[o + r] = end ? 1 : 0;
  } else if (l < a.w) {
    a.parents[o + l] = -1;
    a.tokens[o + l] = -1;
    a.out[o + l] = -__builtin_inff();
    a.done_out[o + l] = 1;
  }
}

// ------------------------------------------------------------------ forks
// Child i continues sequence parents[i].  Full pages are shared; a last page that is part full stays with the first
// child if no one else holds it, and the other children get copies from the free list.  A table's entry gives its page
// (the children that keep it) - 1 references; pages that lost their last one go back before the list's next free page,
// in ascending order.  Three launches: the children (one workgroup), the tables' entries (every workgroup), the pages
// that came free (one workgroup); one launch for small tables.  Latency and the order among the parts bound it: 8 tables of 272
// pages 12 us (13 as three launches, each of which costs the host some 3 more), 512 of 544 pages 5 + 8 + 11.
constexpr int kForkThreads = 1024, kPage = JIT_PAGE_TOKENS;
// Entries of the tables that one workgroup takes.  8 tables over a pool of 65,536 pages, in a graph with a copy of its counts,
// as one launch and as three: 2,096 entries 15.7 and 16.6 us, 2,752 17.1 and 16.5, 3,952 18.6 and 16.6, 6,048 20.4 and 16.4.
// As calls of their own, which the host bounds, one launch takes 21.4 us at all of them, three 25 to 28; of more tables 4,032
// entries take 24.4 and 27.5, 5,120 26.7 and 27.4.  The rule stands between the two uses.
constexpr int kSmallFork = 4096;

struct ForkArgs {
  const int32_t *table, *lens, *parents, *free_at;
  int32_t *refs, *free_pages, *new_table, *new_lens, *src, *dst, *status;
  int32_t *kids;    // [2 S] children, and children that keep the last page
  int32_t *from;    // [N] the row a child copies (-1: none)
  uint32_t *lost;   // [ceil(P / 32)] pages that lost a reference
  int S, W, N, P, F;
};

__device__ __forceinline__ int load_now(const int32_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// inclusive sum over the workgroup's threads; every thread gets the total
__device__ __forceinline__ int block_incl(int v, int *red, int &total) {
  const int l = lane_id(), w = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (l >= o) x += y;
  }
  __syncthreads();  // (red's earlier readers)
  if (l == 63) red[w] = x;
  __syncthreads();
  int base = 0;
  total = 0;
  for (int i = 0; i < (int)(blockDim.x >> 6); i++) {
    if (i < w) base += red[i];
    total += red[i];
  }
  return base + x;
}

__device__ __forceinline__ int fork_len(const ForkArgs &a, int s) {
  const int n = max(a.lens[s], 0);
  return n / kPage >= a.W ? a.W * kPage : n;  // (positions past the table are not there)
}

__device__ __forceinline__ void fork_children(const ForkArgs &a, int *s_first, int *red) {  // s_first [S]: first child
  const int t = threadIdx.x;
  for (int w = t; w < (a.P + 31) / 32; w += kForkThreads) a.lost[w] = 0u;
  for (int s = t; s < a.S; s += kForkThreads) s_first[s] = a.N, a.kids[s] = a.kids[a.S + s] = 0;
  __syncthreads();
  for (int i = t; i < a.N; i += kForkThreads) {
    const int p = a.parents[i];
    if (p >= 0 && p < a.S) atomicMin(&s_first[p], i);
  }
  __syncthreads();
  const int at = min(max(*a.free_at, 0), a.F);
  int taken = 0, refused = 0;
  for (int i0 = 0; i0 < a.N; i0 += kForkThreads) {
    const int i = i0 + t;
    const int p = i < a.N ? a.parents[i] : -1;
    const bool live = p >= 0 && p < a.S;
    const int n = live ? fork_len(a, p) : 0;
    int tail = -1;
    bool need = false;
    if (n % kPage != 0) {
      tail = a.table[(long long)p * a.W + n / kPage];
      need = tail >= 0 && tail < a.P && !(s_first[p] == i && a.refs[tail] == 1);
    }
    int total;
    const int k = block_incl(need ? 1 : 0, red, total) - 1 + taken;
    taken += total;
    int page = -1;
    if (need && k < a.F - at) page = a.free_pages[at + k];
    const bool got = need && page >= 0 && page < a.P, on = live && (!need || got);
    block_incl(need && !got ? 1 : 0, red, total);
    refused += total;
    if (i < a.N) {
      a.from[i] = on ? p : -1;
      a.new_lens[i] = on ? n : 0;
      a.src[i] = got ? tail : -1;
      a.dst[i] = got ? page : -1;
      if (on) atomicAdd(&a.kids[p], 1);
      if (on && !got) atomicAdd(&a.kids[a.S + p], 1);
    }
  }
  if (t == 0) {
    a.status[0] = 0;
    a.status[1] = at + min(taken, a.F - at);
    a.status[2] = refused;
    a.status[3] = 0;
  }
}

// Entry (row, j) of the old tables changes its page's count; of the new ones is copied.
__device__ __forceinline__ void fork_entry(const ForkArgs &a, int row, int j) {
  if (row < a.S) {
    const int n = fork_len(a, row), held = (n + kPage - 1) / kPage;
    if (j < held) {
      const int page = a.table[(long long)row * a.W + j];
      const int gain = load_now(&a.kids[n % kPage != 0 && j == held - 1 ? a.S + row : row]) - 1;
      if (page >= 0 && page < a.P && gain > 0) atomicAdd(&a.refs[page], gain);
      // (whoever takes the last reference sees a count that is not above 0 after it)
      if (page >= 0 && page < a.P && gain < 0 && atomicAdd(&a.refs[page], gain) + gain <= 0)
        atomicOr(&a.lost[page >> 5], 1u << (page & 31));
    }
  }
  if (row < a.N) {
    const int from = a.from[row], n = a.new_lens[row], held = (n + kPage - 1) / kPage;
    int page = 0;
    if (j < held) {
      page = a.table[(long long)from * a.W + j];
      if (j == held - 1 && a.dst[row] >= 0) page = a.dst[row];
    }
    a.new_table[(long long)row * a.W + j] = page;
  }
}

__device__ __forceinline__ void fork_free(const ForkArgs &a, int *red) {
  const int t = threadIdx.x, words = (a.P + 31) / 32;
  int gone = 0;  // pages that came free, all rounds
  const int here = a.status[1];
  // the count first: the list ends where it went on before
  for (int w0 = 0; w0 < words; w0 += kForkThreads) {
    const int w = w0 + t;
    const uint32_t bits = w < words ? load_now((const int32_t *)&a.lost[w]) : 0u;
    uint32_t kept = 0u;
    if (__any(bits != 0)) {  // a wave's 64 words, two at a time: the counts of 64 pages next to each other by one load
      const int l = lane_id(), first = 32 * (w - l);
      int32_t refs[32];
#pragma unroll
      for (int i = 0; i < 32; i++) refs[i] = load_now(&a.refs[min(first + 64 * i + l, a.P - 1)]);
#pragma unroll
      for (int i = 0; i < 32; i++) {
        const uint64_t free = __ballot(refs[i] == 0);
        if (l >> 1 == i) kept = bits & (uint32_t)(l & 1 ? free >> 32 : free);
      }
      if (w < words) a.lost[w] = kept;
    }
    int total;
    block_incl(__builtin_popcount(kept), red, total);
    gone += total;
  }
  __syncthreads();
  const int back = max(here - gone, 0), room = here - back;  // (a list with no room keeps the lowest pages)
  int before = 0;
  for (int w0 = 0; w0 < words; w0 += kForkThreads) {
    const int w = w0 + t;
    uint32_t bits = w < words ? load_now((const int32_t *)&a.lost[w]) : 0u;
    int total;
    int k = before + block_incl(__builtin_popcount(bits), red, total) - __builtin_popcount(bits);
    before += total;
    while (bits) {
      const int i = __builtin_ctz(bits);
      bits &= bits - 1;
      if (k < room) a.free_pages[back + k] = 32 * w + i;
      k++;
    }
  }
  int copies = 0;
  for (int i = t; i < a.N; i += kForkThreads)
    if (a.dst[i] >= 0) a.refs[a.dst[i]] = 1, copies++;
  int total;
  block_incl(copies, red, total);
  if (t == 0) {
    a.status[0] = total;
    a.status[1] = back;
    a.status[3] = gone - room;
  }
}

__global__ __launch_bounds__(kForkThreads) void fork_children_kernel(const ForkArgs a) {
  extern __shared__ int s_first[];
  __shared__ int red[kForkThreads / 64];
  fork_children(a, s_first, red);
}

__global__ __launch_bounds__(256) void fork_entries_kernel(const ForkArgs a) {
  const int cols = (a.W + 255) / 256;
  const int row = blockIdx.x / cols, j = (blockIdx.x % cols) * 256 + threadIdx.x;
  if (j < a.W) fork_entry(a, row, j);
}

__global__ __launch_bounds__(kForkThreads) void fork_free_kernel(const ForkArgs a) {
  __shared__ int red[kForkThreads / 64];
  fork_free(a, red);
}

// The three by one workgroup, for tables of few entries.  What atomics changed is read by load_now, past the L1.
__global__ __launch_bounds__(kForkThreads) void fork_small_kernel(const ForkArgs a) {
  extern __shared__ int s_first[];
  __shared__ int red[kForkThreads / 64];
  fork_children(a, s_first, red);
  __syncthreads();
  const int rows = max(a.S, a.N);
  for (int e = threadIdx.x; e < rows * a.W; e += kForkThreads) fork_entry(a, e / a.W, e % a.W);
  __syncthreads();
  fork_free(a, red);
}

// ------------------------------------------------------------------ page copies in every layer
// A workgroup copies one part of one page of one layer, 16 bytes a thread and step.  256 pages of 48 layers (805 MB read
// and written) take 166 us, 4.85 TB/s, what a large copy reaches; 7 pages 5.5 us.
constexpr int kMaxLayers = 128;  // of a launch: the layers' pointers are its arguments

struct CopyArgs {
  uint4 *pool[kMaxLayers];
  const int32_t *src, *dst;
  int page_words, num_pages, parts, part_words, layers;
};

__global__ __launch_bounds__(256) void copy_layers_kernel(const CopyArgs a) {
  const int part = blockIdx.x % a.parts, rest = blockIdx.x / a.parts, layer = rest % a.layers, i = rest / a.layers;
  const int ps = a.src[i], pd = a.dst[i];
  if (ps < 0 || ps >= a.num_pages || pd < 0 || pd >= a.num_pages) return;
  const uint4 *s = a.pool[layer] + (long long)ps * a.page_words;
  uint4 *d = a.pool[layer] + (long long)pd * a.page_words;
  const int end = min(a.page_words, (part + 1) * a.part_words);
  for (int j = part * a.part_words + threadIdx.x; j < end; j += 256) d[j] = s[j];
}

}  // namespace

extern "C" int jit_beam_select(const float *scores, const float *logprobs, const int32_t *ids, const int32_t *done,
                               const int32_t *eos, int n_eos, int groups, int beams, int alternatives, int width,
                               int32_t *parents, int32_t *tokens, float *out_scores, int32_t *out_done, void *stream) {
  if (groups < 0 || beams <= 0 || alternatives <= 0 || width <= 0 || n_eos < 0)
    return jit::fail(JIT_EINVAL, "beam_select: bad dims groups=%d beams=%d alternatives=%d width=%d n_eos=%d", groups, beams,
                     alternatives, width, n_eos);
  const long long cands = (long long)beams * alternatives;
  if (cands > kMaxCands || width > kMaxWidth)
    return jit::fail(JIT_EUNSUPPORTED, "beam_select covers up to %d candidates a group and a width of %d, got %lld and %d",
                     kMaxCands, kMaxWidth, cands, width);
  if ((long long)groups * beams > 0x7fffffffLL || (long long)groups * 64 > kMaxLaunch)
    return jit::fail(JIT_EUNSUPPORTED, "beam_select covers up to 2^31 - 1 beams of 2^26 - 1 groups, got %d x %d", groups, beams);
  if (groups == 0) return JIT_OK;
  if (!scores || !logprobs || !ids || (n_eos && !eos) || !parents || !tokens || !out_scores || !out_done)
    return jit::fail(JIT_EINVAL, "beam_select: null pointer");
  const BeamArgs a{scores, logprobs, ids, done, eos, parents, tokens, out_done, out_scores, groups, beams, alternatives, width, n_eos};
  const hipStream_t st = (hipStream_t)stream;
  if (cands <= 64)
    beam_select_kernel<1><<<groups, 64, 0, st>>>(a);
  else if (cands <= 256)
    beam_select_kernel<4><<<groups, 64, 0, st>>>(a);
  else if (cands <= 1024)
    beam_select_kernel<16><<<groups, 64, 0, st>>>(a);
  else
    beam_select_kernel<64><<<groups, 64, 0, st>>>(a);
  return jit::check_launch("jit_beam_select");
}

extern "C" long long jit_pages_fork_workspace_bytes(int S, int N, int num_pages) {
  if (S < 0 || N < 0 || num_pages <= 0) return -1;
  return 4LL * (2LL * S + N + (num_pages + 31LL) / 32);
}

extern "C" int jit_pages_fork(const int32_t *page_table, const int32_t *lens, int S, int max_pages, const int32_t *parents,
                              int N, int32_t *refs, int num_pages, int32_t *free_pages, int n_free,
                              const int32_t *free_at, int32_t *new_table, int32_t *new_lens, int32_t *src, int32_t *dst,
                              int32_t *status, void *workspace, long long workspace_bytes, void *stream) {
  if (S < 0 || N < 0 || max_pages <= 0 || num_pages <= 0 || n_free < 0)
    return jit::fail(JIT_EINVAL, "pages_fork: bad dims S=%d N=%d max_pages=%d num_pages=%d n_free=%d", S, N, max_pages,
                     num_pages, n_free);
  if (S > JIT_STEP_TABLES_MAX_SEQS || N > JIT_STEP_TABLES_MAX_SEQS || max_pages > (1 << 26) || num_pages > (1 << 27))
    return jit::fail(JIT_EUNSUPPORTED, "pages_fork covers up to %d sequences and children of up to 2^26 pages of 2^27, got %d, %d, %d and %d",
                     JIT_STEP_TABLES_MAX_SEQS, S, N, max_pages, num_pages);
  const long long blocks = (long long)(S > N ? S : N) * ((max_pages + 255) / 256);
  if (blocks * 256 > kMaxLaunch) return jit::fail(JIT_EUNSUPPORTED, "pages_fork: tables of %d x %d", S > N ? S : N, max_pages);
  if (!refs || !free_at || !status || (S && (!page_table || !lens)) || (N && (!parents || !new_table || !new_lens || !src || !dst)) ||
      (n_free && !free_pages))
    return jit::fail(JIT_EINVAL, "pages_fork: null pointer");
  const long long need = jit_pages_fork_workspace_bytes(S, N, num_pages);
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))
    return jit::fail(JIT_EINVAL, "pages_fork: a workspace of %lld bytes, 16-byte aligned, is needed", need);
  int32_t *ws = (int32_t *)workspace;
  const ForkArgs a{page_table, lens, parents, free_at, refs, free_pages, new_table, new_lens, src, dst, status,
                   ws, ws + 2 * S, (uint32_t *)(ws + 2 * S + N), S, max_pages, N, num_pages, n_free};
  const hipStream_t st = (hipStream_t)stream;
  if ((long long)(S > N ? S : N) * max_pages <= kSmallFork) {
    fork_small_kernel<<<1, kForkThreads, (size_t)S * 4, st>>>(a);
    return jit::check_launch("jit_pages_fork");
  }
  fork_children_kernel<<<1, kForkThreads, (size_t)S * 4, st>>>(a);
  int rc = jit::check_launch("jit_pages_fork (children)");
  if (rc != JIT_OK) return rc;
  if (blocks) {
    fork_entries_kernel<<<(unsigned)blocks, 256, 0, st>>>(a);
    if ((rc = jit::check_launch("jit_pages_fork (entries)")) != JIT_OK) return rc;
  }
  fork_free_kernel<<<1, kForkThreads, 0, st>>>(a);
  return jit::check_launch("jit_pages_fork (free)");
}

extern "C" int jit_kv_copy_pages_layers(void *const *pools, int layers, int num_pages, long long page_bytes,
                                        const int32_t *src, const int32_t *dst, int n, void *stream) {
  if (layers < 0 || n < 0 || num_pages <= 0 || page_bytes <= 0)
    return jit::fail(JIT_EINVAL, "kv_copy_pages_layers: bad dims layers=%d n=%d num_pages=%d page_bytes=%lld", layers, n,
                     num_pages, page_bytes);
  if (page_bytes % 16 || page_bytes > (1LL << 30))
    return jit::fail(JIT_EUNSUPPORTED, "kv_copy_pages_layers covers pages of whole 16-byte words up to 2^30 bytes, got %lld", page_bytes);
  if (layers == 0 || n == 0) return JIT_OK;
  if (!pools || !src || !dst) return jit::fail(JIT_EINVAL, "kv_copy_pages_layers: null pointer");
  for (int i = 0; i < layers; i++)
    if (!pools[i] || ((uintptr_t)pools[i] & 15))
      return jit::fail(JIT_EINVAL, "kv_copy_pages_layers: layer %d's pool must be 16-byte aligned and not null", i);
  CopyArgs a;
  a.num_pages = num_pages;
  a.page_words = (int)(page_bytes / 16);
  // parts of a page, none of fewer than 1,024 words, until 1,024 workgroups copy (1 page of 64 KB in 48 layers: 2.6 us in a
  // graph, 4.4 whole; 7 of 32 KB: 3.8 and 4.1)
  const long long pages = (long long)n * (layers < kMaxLayers ? layers : kMaxLayers), most_parts = (a.page_words + 1023) / 1024;
  a.parts = (int)(pages >= 1024 ? 1 : (1024 + pages - 1) / pages < most_parts ? (1024 + pages - 1) / pages : most_parts);
  a.part_words = (a.page_words + a.parts - 1) / a.parts;
  for (int at = 0; at < layers; at += kMaxLayers) {
    a.layers = layers - at < kMaxLayers ? layers - at : kMaxLayers;
    for (int i = 0; i < a.layers; i++) a.pool[i] = (uint4 *)pools[at + i];
    const long long most = kMaxLaunch / 256 / ((long long)a.layers * a.parts);  // pages of a launch
    for (long long i0 = 0; i0 < n; i0 += most) {
      const long long m = n - i0 < most ? n - i0 : most;
      a.src = src + i0, a.dst = dst + i0;
      copy_layers_kernel<<<(unsigned)(m * a.layers * a.parts), 256, 0, (hipStream_t)stream>>>(a);
      const int rc = jit::check_launch("jit_kv_copy_pages_layers");
      if (rc != JIT_OK) return rc;
    }
  }
  return JIT_OK;
}
