// Filling a paged context: block table and slots of a step's new tokens, and their rows'
// copy into the pages.
//
// Block table.  With old_b tokens cached and new_b to store, request b lacks need_b =
// ceil((old_b + new_b) / 64) - ceil(old_b / 64) pages and takes them from the free list
// behind those of the requests before it, so one prefix sum over the requests gives every
// page, and every token's slot follows from its request's entry of that sum.  The work is a
// few bytes per token and table entry: what it costs is the launches and the latency of
// its dependent loads.
//
// 64 requests of one token, tables of 94 pages: 7.5 us in one workgroup; 512 requests of up to 32
// tokens with a keep mask, tables of 129 pages: 5.0 + 3.6 + 5.4 us.
//
// Append.  A copy of rows; the slot of a token is read once and used for several heads.  32 sequences
// of 256-1024 tokens, 16 heads of k and v, D = 128: 355 MB in 71 us, 5.0 TB/s (a large copy: 5.16).
#include "fmlm_common.h"

#include <algorithm>

namespace fmlm {

typedef fmlm_block_table_params BtParams;
constexpr int kBtThreads = 1024;
constexpr int kBtFillThreads = 256;

FMLM_DEV int64_t bt_index(const void* a, bool i64, int64_t i) {
  return i64 ? ((const int64_t*)a)[i] : (int64_t)((const int32_t*)a)[i];
}
// packed tokens [c0, c1) of request b, within the call's whatever the offsets hold
FMLM_DEV void bt_tokens(const BtParams& p, int b, int& c0, int& c1) {
  c0 = min(max(p.cu_seqlens[b], 0), p.T);
  c1 = min(max(p.cu_seqlens[b + 1], c0), p.T);
}
FMLM_DEV int pages_of(int n) { return (n + FMLM_PAGE_ROWS - 1) / FMLM_PAGE_ROWS; }

// workspace: per request its old length (clamped), the place of its first new page in the
// free list, the tokens it may store and, with keep, the kept tokens before each token (T + 1
// entries): of the whole call (small calls), or of its request, the requests' own ends then
// being in `kept`
struct BtSpace {
  int32_t *old, *base, *count, *kept, *rank;
};
__host__ __device__ inline BtSpace bt_space(const BtParams& p) {
  BtSpace s;
  s.old = (int32_t*)p.workspace;
  s.base = s.old + p.B;
  s.count = s.base + p.B;
  s.kept = s.count + p.B;
  s.rank = s.kept + p.B;
  return s;
}

// inclusive sums over the workgroup's threads of two values at once; s holds NT / 64 pairs
template <int NT>
FMLM_DEV int2 block_scan(int2 v, int2* s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int x = __shfl_up(v.x, off), y = __shfl_up(v.y, off);
    if (lane >= off) {
      v.x += x;
      v.y += y;
    }
  }
  if (lane == 63) s[wave] = v;
  __syncthreads();
  for (int w = 0; w < wave; ++w) {
    v.x += s[w].x;
    v.y += s[w].y;
  }
  __syncthreads();
  return v;
}

// Kept tokens of [t0, t1) before each of them, into rank[t0 .. t1); returns their number.  By a
// workgroup of NT threads, 16 tokens a thread: up to 16 NT tokens take one round.
template <int NT>
FMLM_DEV int bt_rank(const BtParams& p, int t0, int t1, int32_t* rank, int2* part, int* last) {
  constexpr int PER = 16;
  int before = 0;
  for (int base = t0; base < t1; base += PER * NT) {
    const int first = base + PER * threadIdx.x;
    uint32_t bits = 0;
    const bool wide = first + PER <= t1;
    if (wide && ((uintptr_t)(p.keep + first) & 15) == 0) {
      const u32x4 x = *(const u32x4*)(p.keep + first);
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (x[i / 4] >> (8 * (i % 4)) & 0xffu) bits |= 1u << i;
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (first + i < t1 && p.keep[first + i]) bits |= 1u << i;
    }
    const int n = __popc(bits);
    const int2 v = block_scan<NT>(make_int2(n, 0), part);
    const int r0 = before + v.x - n;
    if (wide && ((uintptr_t)(rank + first) & 15) == 0) {
#pragma unroll
      for (int i = 0; i < PER; i += 4) {
        u32x4 x;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = (uint32_t)(r0 + __popc(bits & ((1u << (i + j)) - 1u)));
        *(u32x4*)(rank + first + i) = x;
      }
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (first + i < t1) rank[first + i] = r0 + __popc(bits & ((1u << i) - 1u));
    }
    if (threadIdx.x == NT - 1) *last = v.x;
    __syncthreads();
    before += *last;
    __syncthreads();
  }
  return before;
}

// The requests' prefix sums, by one workgroup of kBtThreads threads.  Each round scans the
// pages that kBtThreads requests lack beside their old lengths, then the rows they end up
// with (the free list may have cut them).  SMALL: ranks are the whole call's.
template <bool SMALL>
FMLM_DEV void bt_scan(const BtParams& p, const BtSpace& w, int2* part) {
  __shared__ int2 total;
  __shared__ int bad;
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  const int cap_in = p.table_in ? min(p.in_pages, p.max_pages) * FMLM_PAGE_ROWS : 0;
  const int cap_out = p.max_pages * FMLM_PAGE_ROWS;
  int pages = 0, rows = 0, rows_old = 0;  // of the requests before
  for (int b0 = 0; b0 < p.B; b0 += kBtThreads) {
    const int b = b0 + threadIdx.x;
    int old = 0, cnt = 0, need = 0, have = 0;
    bool over = false;
    if (b < p.B) {
      const int64_t raw = bt_index(p.old_lens, p.flags & FMLM_BT_OLD_I64, b);
      int c0, c1;
      bt_tokens(p, b, c0, c1);
      old = (int)(raw < 0 ? 0 : raw > cap_in ? cap_in : raw);
      cnt = !p.keep ? c1 - c0 : SMALL ? w.rank[c1] - w.rank[c0] : w.kept[b];
      over = raw != old || cnt > cap_out - old;
      cnt = min(cnt, cap_out - old);
      have = pages_of(old);
      need = pages_of(old + cnt) - have;
    }
    const uint64_t m = __builtin_amdgcn_ballot_w64(over);
    if (m && (threadIdx.x & 63) == 0) atomicAdd(&bad, __popcll(m));
    const int2 v = block_scan<kBtThreads>(make_int2(need, old), part);
    const int base = pages + v.x - need;
    // what the free list lacks, the request's later tokens cannot be stored in
    const int got = max(0, min(need, p.n_free - base));
    if (got < need) cnt = max(0, min(cnt, (have + got) * FMLM_PAGE_ROWS - old));
    const int2 r = block_scan<kBtThreads>(make_int2(cnt, 0), part);
    if (b < p.B) {
      w.old[b] = old;
      w.base[b] = base;
      w.count[b] = cnt;
      p.new_lens[b] = old + cnt;
      p.cu_kv[b + 1] = rows + v.y + r.x;
    }
    if (b0 + kBtThreads < p.B) {  // the next round's start
      if (threadIdx.x == kBtThreads - 1) total = make_int2(v.x, v.y);
      __syncthreads();
      pages += total.x;
      rows_old += total.y;
      rows += total.y;
      __syncthreads();
      if (threadIdx.x == kBtThreads - 1) total.x = r.x;
      __syncthreads();
      rows += total.x;
      __syncthreads();
    } else if (threadIdx.x == kBtThreads - 1) {
      const int need_all = pages + v.x, taken = min(need_all, p.n_free);
      p.summary[0] = taken;
      p.summary[1] = need_all - taken;
      p.summary[2] = bad;  // the scans' barriers lie between
      p.summary[3] = rows + v.y + r.x - (rows_old + v.y);
    }
  }
  if (threadIdx.x == 0) {
    p.cu_kv[0] = 0;
    if (p.B == 0) p.summary[0] = p.summary[1] = p.summary[2] = p.summary[3] = 0;
  }
}

// Table entries and tokens, kBtUnroll at a time per thread, `step` apart, so that the loads of a
// stage overlap: an entry waits for its request's sums and then for its page, a token for its
// index before that.
constexpr int kBtUnroll = 4;
struct BtPlace {
  int b, i;  // page i of request b
};
FMLM_DEV void bt_pages(const BtParams& p, const BtSpace& w, const BtPlace (&at)[kBtUnroll], const bool (&want)[kBtUnroll],
                       int (&page)[kBtUnroll]) {
  int old[kBtUnroll], count[kBtUnroll], base[kBtUnroll];
#pragma unroll
  for (int u = 0; u < kBtUnroll; ++u) {
    old[u] = w.old[at[u].b];
    count[u] = w.count[at[u].b];
    base[u] = w.base[at[u].b];
  }
#pragma unroll
  for (int u = 0; u < kBtUnroll; ++u) {
    const int have = pages_of(old[u]), all = pages_of(old[u] + count[u]), i = at[u].i;
    page[u] = -1;
    if (want[u] && i < have)
      page[u] = (int)bt_index(p.table_in, p.flags & FMLM_BT_TABLE_I64, (int64_t)at[u].b * p.in_pages + i);
    else if (want[u] && i < all)
      page[u] = (int)bt_index(p.free_pages, p.flags & FMLM_BT_FREE_I64, base[u] + i - have);
  }
}

template <bool SMALL>
FMLM_DEV void bt_fill(const BtParams& p, const BtSpace& w, int64_t first, int64_t step) {
  const int64_t entries = (int64_t)p.B * p.max_pages;
  for (int64_t e0 = first; e0 < entries; e0 += kBtUnroll * step) {
    BtPlace at[kBtUnroll];
    bool want[kBtUnroll];
    int page[kBtUnroll];
#pragma unroll
    for (int u = 0; u < kBtUnroll; ++u) {
      const int64_t e = e0 + u * step;
      want[u] = e < entries;
      const int64_t x = want[u] ? e : 0;
      // (64-bit divisions take some hundred instructions)
      at[u].b = entries <= 0x7fffffff ? (int)((uint32_t)x / (uint32_t)p.max_pages) : (int)(x / p.max_pages);
      at[u].i = (int)(x - (int64_t)at[u].b * p.max_pages);
    }
    bt_pages(p, w, at, want, page);
#pragma unroll
    for (int u = 0; u < kBtUnroll; ++u)
      if (want[u]) p.block_table[e0 + u * step] = page[u];
  }
  for (int64_t t0 = first; t0 < p.T; t0 += kBtUnroll * step) {
    uint32_t tok[kBtUnroll];
    int rank[kBtUnroll], old[kBtUnroll], count[kBtUnroll], pos[kBtUnroll], page[kBtUnroll];
    bool real[kBtUnroll], kept[kBtUnroll];
    BtPlace at[kBtUnroll];
#pragma unroll
    for (int u = 0; u < kBtUnroll; ++u) {
      const int64_t t = t0 + u * step;
      real[u] = t < p.T;
      tok[u] = (uint32_t)p.token_indices[real[u] ? t : 0];
      kept[u] = real[u] && (!p.keep || p.keep[t]);
      rank[u] = p.keep && real[u] ? w.rank[t] : 0;
    }
#pragma unroll
    for (int u = 0; u < kBtUnroll; ++u) {
      at[u].b = (int)min(tok[u] / (uint32_t)p.N, (uint32_t)p.B - 1u);
      pos[u] = (int)min(tok[u] - (uint32_t)at[u].b * (uint32_t)p.N, (uint32_t)p.N - 1u);
      if (!p.keep) rank[u] = pos[u];
      else if (SMALL && kept[u]) rank[u] -= w.rank[max(t0 + u * step - pos[u], (int64_t)0)];
      rank[u] = max(rank[u], 0);  // (not so only where the metadata contradicts itself)
      old[u] = w.old[at[u].b];
      count[u] = w.count[at[u].b];
    }
#pragma unroll
    for (int u = 0; u < kBtUnroll; ++u) {
      kept[u] = kept[u] && rank[u] < count[u];
      at[u].i = (old[u] + rank[u]) / FMLM_PAGE_ROWS;
    }
    bt_pages(p, w, at, kept, page);
#pragma unroll
    for (int u = 0; u < kBtUnroll; ++u) {
      if (!real[u]) continue;
      const int64_t t = t0 + u * step;
      p.slot_mapping[t] =
          page[u] >= 0 ? (int64_t)page[u] * FMLM_PAGE_ROWS + (old[u] + rank[u]) % FMLM_PAGE_ROWS : (int64_t)-1;
      p.positions[t] = old[u] + pos[u];
    }
  }
}

// all of it in one workgroup
__global__ __launch_bounds__(kBtThreads) void block_table_small_kernel(const BtParams p) {
  __shared__ int2 part[kBtThreads / 64];
  __shared__ int last;
  const BtSpace w = bt_space(p);
  if (p.keep) {
    const int all = bt_rank<kBtThreads>(p, 0, p.T, w.rank, part, &last);
    if (threadIdx.x == 0) w.rank[p.T] = all;
    __syncthreads();
  }
  bt_scan<true>(p, w, part);
  __syncthreads();
  bt_fill<true>(p, w, threadIdx.x, kBtThreads);
}

// one workgroup per request
__global__ __launch_bounds__(kBtFillThreads) void block_table_rank_kernel(const BtParams p) {
  __shared__ int2 part[kBtFillThreads / 64];
  __shared__ int last;
  const BtSpace w = bt_space(p);
  const int b = blockIdx.x;
  int c0, c1;
  bt_tokens(p, b, c0, c1);
  const int n = bt_rank<kBtFillThreads>(p, c0, c1, w.rank, part, &last);
  if (threadIdx.x == 0) w.kept[b] = n;
}
__global__ __launch_bounds__(kBtThreads) void block_table_scan_kernel(const BtParams p) {
  __shared__ int2 part[kBtThreads / 64];
  bt_scan<false>(p, bt_space(p), part);
}
__global__ __launch_bounds__(kBtFillThreads) void block_table_fill_kernel(const BtParams p) {
  bt_fill<false>(p, bt_space(p), (int64_t)blockIdx.x * kBtFillThreads + threadIdx.x, (int64_t)gridDim.x * kBtFillThreads);
}

// One workgroup for two rounds of table entries and one of tokens (a round: what its threads fill at
// once).  A further round of entries takes it 1.2 to 1.8 us, one of tokens 2 and with keep 3; the other kernels
// cost 1 to 1.5 us more to begin with (with keep, one more, 2), and as much again where the host's launches
// are what counts.  us a call, one workgroup against the others, in a graph (on a stream):
//   entries, no keep: 4096 6.3 : 7.1 (6.3 : 8.7), 8192 7.5-8.0 : 7.2-7.5 (7.5-8.0 : 8.7), 9024 8.8 : 7.2 (8.8 : 8.7)
//   with keep:        8192 10.0-10.5 : 10.4-10.8 (10.0-10.5 : 11.2), 9024 11.3 : 10.7 (11.2 : 11.0)
//   tokens, no keep:  3100 7.1 : 8.3 (7.1 : 8.7), 6200 8.7 : 7.3 (8.6 : 9.0)
//   with keep:        3100 10.2 : 12.3 (10.2 : 12.7), 6200 13.0 : 11.5 (12.9 : 11.8)
constexpr int64_t kBtRound = kBtUnroll * kBtThreads;
static bool bt_small(int64_t entries, int64_t tokens) { return entries <= 2 * kBtRound && tokens <= kBtRound; }

static int bt_check(const BtParams& p) {
  if (p.B < 0 || p.N < 0 || p.T < 0 || p.max_pages < 0 || p.in_pages < 0 || p.n_free < 0) return FMLM_E_ARG;
  if ((int64_t)p.B * p.N > 0x7fffffff || p.T > (int64_t)p.B * p.N) return FMLM_E_ARG;
  // lengths are 32-bit
  if (p.max_pages > 0x7fffffff / FMLM_PAGE_ROWS || p.in_pages > 0x7fffffff / FMLM_PAGE_ROWS) return FMLM_E_ARG;
  return 0;
}

// ---------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------
struct AppendPagedArgs {
  fmlm_paged_tensor t[2];
};
constexpr int kApThreads = 256;
constexpr int kApHeads = 4;  // heads per thread

// VB bytes a lane; a row is cpr lanes.  blockIdx.y: chunk of heads, z: tensor
template <typename V>
__global__ __launch_bounds__(kApThreads) void paged_append_kernel(const AppendPagedArgs args, int es, int heads, int cpr,
                                                                  int64_t row_bytes, int T, int N, int layout,
                                                                  const int64_t* __restrict__ token_indices,
                                                                  const int64_t* __restrict__ slots, int64_t pool_rows) {
  const fmlm_paged_tensor& a = args.t[blockIdx.z];
  const int64_t at = (int64_t)blockIdx.x * kApThreads + threadIdx.x;
  const int64_t t = at / cpr;
  if (t >= T) return;
  const int c = (int)(at - t * cpr);
  const int64_t slot = slots[t];
  int64_t off = t * a.s_sn;
  if (layout == FMLM_LAYOUT_PADDED) {
    const uint32_t tok = (uint32_t)token_indices[t];
    uint32_t b = tok / (uint32_t)N;
    const uint32_t p = tok - b * (uint32_t)N;
    if (a.batch > 0) b = min(b, (uint32_t)a.batch - 1u);
    off = (int64_t)b * a.s_sb + (int64_t)p * a.s_sn;
  }
  if (slot < 0 || slot >= pool_rows) return;
  const char* src = (const char*)a.src + off * es + (int64_t)c * sizeof(V);
  char* dst = (char*)a.pool + slot * row_bytes + (int64_t)c * sizeof(V);
  const int64_t ss = a.s_sh * es, ds = pool_rows * row_bytes;
  const int h0 = blockIdx.y * kApHeads;
  V v[kApHeads];
#pragma unroll
  for (int u = 0; u < kApHeads; ++u)
    if (h0 + u < heads) v[u] = *(const V*)(src + (h0 + u) * ss);
#pragma unroll
  for (int u = 0; u < kApHeads; ++u)
    if (h0 + u < heads) *(V*)(dst + (h0 + u) * ds) = v[u];
}

}  // namespace fmlm

using namespace fmlm;

extern "C" int fmlm_block_table_params_size(void) { return (int)sizeof(fmlm_block_table_params); }

extern "C" int64_t fmlm_block_table_workspace_bytes(const fmlm_block_table_params* pp) {
  if (!pp) return FMLM_E_ARG;
  const int rc = bt_check(*pp);
  if (rc) return rc;
  return 4 * (4 * (int64_t)pp->B + (pp->keep ? (int64_t)pp->T + 1 : 0));
}

extern "C" int fmlm_block_table(const fmlm_block_table_params* pp, void* stream) {
  if (!pp) return FMLM_E_ARG;
  const BtParams& p = *pp;
  const int64_t need = fmlm_block_table_workspace_bytes(pp);
  if (need < 0) return (int)need;
  if (!p.cu_kv || !p.summary) return FMLM_E_ARG;
  if (p.B > 0 && (!p.old_lens || !p.cu_seqlens || !p.new_lens)) return FMLM_E_ARG;
  if (p.T > 0 && (!p.token_indices || !p.slot_mapping || !p.positions)) return FMLM_E_ARG;
  if (((int64_t)p.B * p.max_pages > 0 && !p.block_table) || (p.n_free > 0 && !p.free_pages)) return FMLM_E_ARG;
  if (need > 0 && (!p.workspace || p.workspace_bytes < need)) return FMLM_E_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  const int64_t entries = (int64_t)p.B * p.max_pages, work = std::max<int64_t>(entries, p.T);
  if (bt_small(entries, p.T)) {
    hipLaunchKernelGGL(block_table_small_kernel, dim3(1), dim3(kBtThreads), 0, s, p);
    return launch_status();
  }
  if (p.keep) {
    hipLaunchKernelGGL(block_table_rank_kernel, dim3(p.B), dim3(kBtFillThreads), 0, s, p);
  }
  hipLaunchKernelGGL(block_table_scan_kernel, dim3(1), dim3(kBtThreads), 0, s, p);
  const unsigned blocks = (unsigned)std::min<int64_t>((work + kBtFillThreads - 1) / kBtFillThreads, 4096);
  hipLaunchKernelGGL(block_table_fill_kernel, dim3(blocks), dim3(kBtFillThreads), 0, s, p);
  return launch_status();
}

template <typename V>
static int paged_append(const fmlm_paged_tensor* tensors, int n, int es, int heads, int64_t row_bytes, int T, int N,
                        int layout, const int64_t* token_indices, const int64_t* slots, int64_t pool_rows,
                        hipStream_t s) {
  AppendPagedArgs args{};
  for (int i = 0; i < n; ++i) args.t[i] = tensors[i];
  const int64_t cpr = row_bytes / (int64_t)sizeof(V), blocks = (cpr * T + kApThreads - 1) / kApThreads;
  if (blocks > 0x7fffffff || cpr > 0x7fffffff) return FMLM_E_ARG;
  hipLaunchKernelGGL(paged_append_kernel<V>, dim3((unsigned)blocks, (heads + kApHeads - 1) / kApHeads, n),
                     dim3(kApThreads), 0, s, args, es, heads, (int)cpr, row_bytes, T, N, layout, token_indices, slots,
                     pool_rows);
  return launch_status();
}

extern "C" int fmlm_paged_append(const fmlm_paged_tensor* tensors, int32_t n_tensors, int32_t elem_bytes, int32_t heads,
                                 int32_t D, int32_t T, int32_t N, int32_t layout, const int64_t* token_indices,
                                 const int64_t* slots, int64_t pool_rows, void* stream) {
  if (elem_bytes != 1 && elem_bytes != 2 && elem_bytes != 4 && elem_bytes != 8) return FMLM_E_DTYPE;
  if (!tensors || n_tensors < 1 || n_tensors > 2 || heads < 0 || D < 1 || T < 0 || pool_rows < 0) return FMLM_E_ARG;
  if (layout != FMLM_LAYOUT_PADDED && layout != FMLM_LAYOUT_PACKED) return FMLM_E_ARG;
  if (heads > 65535 * kApHeads) return FMLM_E_ARG;
  if (T == 0 || heads == 0 || pool_rows == 0) return 0;
  if (!slots || (layout == FMLM_LAYOUT_PADDED && (!token_indices || N < 1))) return FMLM_E_ARG;
  const int64_t row_bytes = (int64_t)D * elem_bytes;
  uint64_t all = (uint64_t)row_bytes;  // low bits common to every address
  for (int i = 0; i < n_tensors; ++i) {
    const fmlm_paged_tensor& t = tensors[i];
    if (!t.src || !t.pool) return FMLM_E_ARG;
    all |= (uint64_t)t.src | (uint64_t)t.pool | (uint64_t)(t.s_sb * elem_bytes) | (uint64_t)(t.s_sh * elem_bytes) |
           (uint64_t)(t.s_sn * elem_bytes);
  }
  if (all % elem_bytes) return FMLM_E_ALIGN;
  hipStream_t s = (hipStream_t)stream;
  if (all % 16 == 0) return paged_append<u32x4>(tensors, n_tensors, elem_bytes, heads, row_bytes, T, N, layout, token_indices, slots, pool_rows, s);
  if (all % 4 == 0) return paged_append<uint32_t>(tensors, n_tensors, elem_bytes, heads, row_bytes, T, N, layout, token_indices, slots, pool_rows, s);
  if (all % 2 == 0) return paged_append<uint16_t>(tensors, n_tensors, elem_bytes, heads, row_bytes, T, N, layout, token_indices, slots, pool_rows, s);
  return paged_append<uint8_t>(tensors, n_tensors, elem_bytes, heads, row_bytes, T, N, layout, token_indices, slots, pool_rows, s);
}
