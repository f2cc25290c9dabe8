// Drafted trees: ancestor masks, and the tree's part of the attention calls whose main kernel
// does not mask its keys itself.
//
// Query i of a sequence attends to the sequence's context and to those tokens j of its own
// draft that are i or an ancestor of i.  The MFMA kernels up to D = 256 do all of it
// (fmlm_attn.hip).  For the 512-wide latent the context's part runs by itself and
// leaves, per row, its own softmax's output o_c (fp32) and l_c = log2(sum 2^z), z =
// scale log2(e) q.k.  A kernel here computes m = max z and l = sum 2^(z - m) over the ancestors
// and writes
//   (2^(l_c - M) o_c + 2^(m - M) sum 2^(z - m) v) / (2^(l_c - M) + 2^(m - M) l),  M = max(l_c, m).
//
// A draft has at most 256 tokens, so its keys are few beside the context's: these kernels are
// bound by latency, not by bandwidth or products.  Steps in which no row has an ancestor are
// skipped (an ancestor precedes its descendants, so the later ones).
#include "fmlm_common.h"

#include <algorithm>
#include <type_traits>

namespace fmlm {

// ---------------------------------------------------------------------------
// Ancestor masks: one workgroup per sequence, thread i is token i.  After round k a token
// knows its nearest 2^k ancestors, and the next one beyond them.  512 sequences of up to 32 tokens:
// 3.2 us, a launch's latency.
// ---------------------------------------------------------------------------
constexpr int kTreeWords = FMLM_MAX_TREE / 64;

__global__ __launch_bounds__(FMLM_MAX_TREE) void tree_mask_kernel(const void* parents, int parents_i64,
                                                                  const int32_t* __restrict__ cu, int N, int T, int words,
                                                                  const void* ctx_lens, int ctx_i64,
                                                                  uint64_t* __restrict__ mask,
                                                                  int32_t* __restrict__ positions, int32_t* n_bad) {
  __shared__ uint64_t s_bits[FMLM_MAX_TREE][kTreeWords];
  __shared__ int s_next[FMLM_MAX_TREE];
  const int b = blockIdx.x, i = threadIdx.x;
  const int c0 = min(max(cu[b], 0), T), n = max(0, min(min(cu[b + 1], T) - c0, min(N, FMLM_MAX_TREE)));
  uint64_t bits[kTreeWords];
  int next = -1;
  if (i < n) {
    const int64_t up = parents_i64 ? ((const int64_t*)parents)[c0 + i] : (int64_t)((const int32_t*)parents)[c0 + i];
    if (up >= 0 && up < i) next = (int)up;
    else if (up != -1 && n_bad) atomicAdd(n_bad, 1);
#pragma unroll
    for (int w = 0; w < kTreeWords; ++w) bits[w] = i / 64 == w ? 1ull << (i % 64) : 0;
  }
  for (int span = 1; span < n; span *= 2) {
    if (i < n) {
#pragma unroll
      for (int w = 0; w < kTreeWords; ++w) s_bits[i][w] = bits[w];
      s_next[i] = next;
    }
    __syncthreads();
    if (i < n && next >= 0) {
#pragma unroll
      for (int w = 0; w < kTreeWords; ++w) bits[w] |= s_bits[next][w];
      next = s_next[next];
    }
    __syncthreads();
  }
  if (i < n) {
    int seen = 0;
#pragma unroll
    for (int w = 0; w < kTreeWords; ++w) {
      if (w < words) mask[(int64_t)(c0 + i) * words + w] = bits[w];
      seen += __popcll(bits[w]);
    }
    for (int w = kTreeWords; w < words; ++w) mask[(int64_t)(c0 + i) * words + w] = 0;
    const int64_t ctx = !ctx_lens ? 0 : ctx_i64 ? ((const int64_t*)ctx_lens)[b] : (int64_t)((const int32_t*)ctx_lens)[b];
    positions[c0 + i] = (int)ctx + seen - 1;
  }
}

// ---------------------------------------------------------------------------
// What the two tree kernels share: the sequence, and the context's part of a row.
// ---------------------------------------------------------------------------
struct TreeSeq {
  int q0, len;
  bool has_ctx;
  int64_t k0, v0;  // element offsets of the sequence's first main key and value of the head
  int64_t k_sn, v_sn;
};
FMLM_DEV TreeSeq tree_seq(const fmlm_attn_params& p, int b, int h) {
  const SeqInfo si = seq_info(p, b);
  TreeSeq s;
  s.q0 = si.q0;
  s.len = min(si.len, FMLM_MAX_TREE);
  s.has_ctx = si.ctx > 0;
  const bool mla = p.flags & FMLM_FLAG_MLA, packed = p.kv_layout == FMLM_LAYOUT_PACKED;
  const int64_t v_sb = mla ? p.k_sb : p.v_sb, v_sh = mla ? p.k_sh : p.v_sh;
  s.k_sn = p.k_sn;
  s.v_sn = mla ? p.k_sn : p.v_sn;
  s.k0 = (packed ? (int64_t)s.q0 * s.k_sn : (int64_t)b * p.k_sb) + (int64_t)h * p.k_sh;
  s.v0 = (packed ? (int64_t)s.q0 * s.v_sn : (int64_t)b * v_sb) + (int64_t)h * v_sh;
  return s;
}
FMLM_DEV int64_t tree_row(int layout, int b, int h, int q0, int pos, int64_t sb, int64_t sh, int64_t sn) {
  return layout == FMLM_LAYOUT_PACKED ? (int64_t)h * sh + (int64_t)(q0 + pos) * sn
                                      : (int64_t)b * sb + (int64_t)h * sh + (int64_t)pos * sn;
}
// the weights of the two parts of a row, already divided by their sum (m, l: the tree's)
struct TreeJoin {
  float wc, wt;
};
FMLM_DEV TreeJoin tree_join(bool has_ctx, float lc, float m, float l) {
  TreeJoin j{0.f, 0.f};
  if (!has_ctx) {
    if (l != 0.f) j.wt = 1.f / l;  // (NaN too; no key at all: 0)
    return j;
  }
  const float top = vmax(lc, m);
  j.wc = fast_exp2(lc - top);  // an infinite top: NaN, as inf - inf is
  j.wt = m == -INFINITY ? 0.f : fast_exp2(m - top);
  const float inv = 1.f / fmaf(j.wt, l, j.wc);
  j.wc *= inv;
  j.wt *= inv;
  return j;
}

// ---------------------------------------------------------------------------
// bf16 / fp16, the 512-wide latent (K = V = one row for all heads).  A workgroup of 4 waves takes 16 of
// a sequence's (head, position) rows: all heads have the same keys, and a tile of one head would be
// mostly empty for a draft of a few tokens.  As in the forward kernels S^T = K Q^T and
// O^T = V^T P^T, so that a lane (q + 16 g) holds keys 4g .. 4g+3 of query q and then columns
// 16 db + 4g .. of its output.  Steps of 32 keys pass through LDS once and serve both products: b128
// reads make K's operand, transposing reads V's.  Every wave computes all scores (32 MFMAs)
// and the output of its own 128 columns, which needs no exchange.  What the kernel takes is the
// latency of its loads: those of a step and of the context's rows are issued together at the start, and
// the queries pass through LDS so that three workgroups fit a CU.  P is rounded to the input type
// for the product, and its row sum is taken of the rounded values.
// 16 sequences of up to 16 tokens, 64 heads: one wave a tile of one head, keys and values read apart
// and the context's rows at the end took 22.4 us, four waves with all of it at the start 16.9, tiles over
// heads with two workgroups a CU 17.5, with three 12.5.
// Merging the parts of a split context here as well, instead of the 15 us of a launch of its own, took
// 40: these workgroups are too few to read the parts' records.
// ---------------------------------------------------------------------------
constexpr int kLatentD = 512, kLatentWaves = 4;

template <typename T>
__global__ __launch_bounds__(kLatentWaves * 64, 3) void attn_tree_latent_kernel(const fmlm_attn_params p,
                                                                             const float* __restrict__ octx,
                                                                             const float* __restrict__ lse,
                                                                             const uint64_t* __restrict__ mask,
                                                                             int words) {
  typedef typename Mfma<T>::v8 v8;
  constexpr int D = kLatentD, NW = kLatentWaves, KC = D / 32, NDB = D / 16 / NW, BK = 32;
  constexpr int PITCH = D * 2 + 16;  // 16 bytes apart: a column's rows fall into different banks
  constexpr int NL = BK / NW;        // rows (1 KiB, one load) per wave and step
  __shared__ __align__(16) char tile[BK * PITCH];
  __shared__ __align__(16) char qs[16 * PITCH];
  __shared__ uint32_t s_bad[NW];
  const int b = blockIdx.y, r0 = blockIdx.x * 16;
  const TreeSeq s = tree_seq(p, b, 0);
  const int rows = p.H * s.len;
  if (r0 >= rows) return;
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = r0 + l16, c0 = wave * NDB * 16;
  const bool ok = row < rows;
  const int h = min(row, rows - 1) / s.len, pos = min(row, rows - 1) - h * s.len;
  const float c = p.scale * kLog2e;
  const T* const kp = (const T*)p.k + s.k0;

  u32x4 v[NL];
  auto load = [&](int j0) {  // this wave's rows of a step; rows past the sequence are zero
#pragma unroll
    for (int n = 0; n < NL; ++n) {
      const int j = j0 + wave * NL + n;
      v[n] = u32x4{0u, 0u, 0u, 0u};
      if (j < s.len) v[n] = *(const u32x4*)(kp + (int64_t)j * s.k_sn + lane * 8);
    }
  };
  load(0);
  // the queries (in registers they would cost a CU a workgroup)
#pragma unroll
  for (int n = 0; n < 16 / NW; ++n) {
    const int i = wave * (16 / NW) + n, r = min(r0 + i, rows - 1), hq = r / s.len;
    const T* q = (const T*)p.q + tree_row(p.q_layout, b, hq, s.q0, r - hq * s.len, p.q_sb, p.q_sh, p.q_sn);
    *(u32x4*)(qs + i * PITCH + lane * 16) = *(const u32x4*)(q + lane * 8);
  }
  f32x4 oc[NDB];
  float lc = 0.f;
  if (s.has_ctx) {
    const int64_t at = (int64_t)h * p.total_q + s.q0 + pos;
    lc = lse[at];
#pragma unroll
    for (int db = 0; db < NDB; ++db) oc[db] = *(const f32x4*)(octx + at * D + c0 + db * 16 + 4 * g);
  }
  f32x4 o[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  const uint32_t qaddr = lds_addr(qs) + l16 * PITCH + 16 * g, kaddr = lds_addr(tile) + l16 * PITCH + 16 * g;
  const uint32_t vaddr = lds_addr(tile) + (4 * g + (l16 >> 2)) * PITCH + 8 * (l16 & 3) + 2 * c0;
  for (int j0 = 0; j0 < s.len; j0 += BK) {
    uint32_t seen = 0;  // keys j0 + bit that the lane's row attends to
    if (ok && j0 / 64 < words) seen = (uint32_t)(mask[(int64_t)(s.q0 + pos) * words + j0 / 64] >> (j0 % 64));
    if (s.len - j0 < BK) seen &= (1u << (s.len - j0)) - 1u;
    // (the same in every wave)
    if (j0 > 0 && !__builtin_amdgcn_ballot_w64(seen != 0)) continue;
    if (j0 > 0) {
      load(j0);
      __syncthreads();  // the tile's last readers are done
    }
    // ---- the tile, and which of its rows have an element that is not finite: 0 times it would
    // not be 0 in the rows that do not see it (below)
    constexpr uint32_t E = std::is_same<T, bf16>::value ? 0x7f80u : 0x7c00u;  // exponent of inf and NaN
    uint32_t mine = 0;
#pragma unroll
    for (int n = 0; n < NL; ++n) {
      const int row = wave * NL + n;
      bool inf = false;
#pragma unroll
      for (int w = 0; w < 4; ++w) inf |= (v[n][w] & E) == E || (v[n][w] >> 16 & E) == E;
      if (__builtin_amdgcn_ballot_w64(inf)) mine |= 1u << row;
      *(u32x4*)(tile + row * PITCH + lane * 16) = v[n];
    }
    if (lane == 0) s_bad[wave] = mine;
    __syncthreads();
    // ---- scores
    f32x4 sc[2];
    sc[0] = sc[1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      const v8 q = *(const FMLM_LDS v8*)(uintptr_t)(qaddr + kc * 64);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
        sc[kb] = Mfma<T>::run(*(const FMLM_LDS v8*)(uintptr_t)(kaddr + kb * 16 * PITCH + kc * 64), q, sc[kb]);
    }
    uint32_t bad = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) bad |= s_bad[w];
    bad = __builtin_amdgcn_readfirstlane(bad);
    if (bad) {
      __syncthreads();  // every wave has its scores
#pragma unroll
      for (int n = 0; n < NL; ++n)
        if (bad >> (wave * NL + n) & 1) *(u32x4*)(tile + (wave * NL + n) * PITCH + lane * 16) = u32x4{0u, 0u, 0u, 0u};
      __syncthreads();
    }
    float mx = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        sc[kb][r] = (seen >> (kb * 16 + 4 * g + r) & 1) ? sc[kb][r] * c : -INFINITY;
        mx = vmax(mx, sc[kb][r]);
      }
    const float m_new = vmax(m, lane_max_xor16_32(mx));
    const float ref = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = fast_exp2(m - ref);
    m = m_new;
    v8 pf;
    float sum = 0.f;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const T x = (T)fast_exp2(sc[kb][r] - ref);
        pf[kb * 4 + r] = x;
        sum += (float)x;
      }
    l = l * alpha + sum;
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
      const s16x4 lo = lds_read_tr16_at(vaddr + db * 32), hi = lds_read_tr16_at(vaddr + db * 32 + 16 * PITCH);
      const v8 a = __builtin_bit_cast(v8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
      o[db] = Mfma<T>::run(a, pf, o[db] * alpha);
    }
    // ---- values that are not finite: by the rows that see them alone
    for (uint32_t left = bad; left; left &= left - 1) {
      const int j = __builtin_ctz(left), from = l16 + 16 * ((j & 15) >> 2);
      float x = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e == (j >> 4) * 4 + (j & 3)) x = (float)pf[e];
      x = __shfl(x, from);
      if (seen >> j & 1) {
        const T* vj = kp + (int64_t)(j0 + j) * s.k_sn + c0 + 4 * g;
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[db][r] = fmaf(x, (float)vj[db * 16 + r], o[db][r]);
      }
    }
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (!ok) return;
  const TreeJoin j = tree_join(s.has_ctx, lc, m, l);
  T* const dst = (T*)p.o + tree_row(p.o_layout, b, h, s.q0, pos, p.o_sb, p.o_sh, p.o_sn) + c0 + 4 * g;
#pragma unroll
  for (int db = 0; db < NDB; ++db) {
    f32x4 x = o[db] * j.wt;
    if (s.has_ctx) x += j.wc * oc[db];
    T y[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = (T)x[r];
    u32x2 raw;
    __builtin_memcpy(&raw, y, 8);
    *(u32x2*)(dst + db * 16) = raw;
  }
}

// ---------------------------------------------------------------------------
// fp32 latent (whose context runs on the SIMT kernel): one wave per row.  Lane j scores key j of a step of 64 keys; then the row's keys are
// taken one by one, a lane holding D / 64 columns.
// Keys that the row does not see are not read.  Chains of 8 tokens, 4 sequences, 16 heads: 15 us beside the
// 1156 of their 1000 context rows; of 64 tokens, 8 sequences: 156 beside 1972.  The context's SIMT kernel,
// which plain fp32 latent calls have too, is what such calls take (floors: 7 and 112 us).
// ---------------------------------------------------------------------------
template <int D>
__global__ __launch_bounds__(64) void attn_tree_f32_kernel(const fmlm_attn_params p, const float* __restrict__ octx,
                                                           const float* __restrict__ lse,
                                                           const uint64_t* __restrict__ mask, int words) {
  constexpr int NC = D / 64;
  __shared__ __align__(16) float qs[D];
  const int b = blockIdx.z, h = blockIdx.y, pos = blockIdx.x, lane = threadIdx.x;
  const TreeSeq s = tree_seq(p, b, h);
  if (pos >= s.len) return;
  const float c = p.scale * kLog2e;
  const float* const q = (const float*)p.q + tree_row(p.q_layout, b, h, s.q0, pos, p.q_sb, p.q_sh, p.q_sn);
  const float* const kp = (const float*)p.k + s.k0;
  const float* const vp = (const float*)((p.flags & FMLM_FLAG_MLA) ? p.k : p.v) + s.v0;
  for (int d = lane; d < D; d += 64) qs[d] = q[d];
  __syncthreads();
  float o[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) o[i] = 0.f;
  float m = -INFINITY, l = 0.f;
  for (int w = 0; w < words && w * 64 < s.len; ++w) {
    uint64_t seen = mask[(int64_t)(s.q0 + pos) * words + w];
    if (s.len - w * 64 < 64) seen &= (1ull << (s.len - w * 64)) - 1ull;
    if (!seen) continue;
    float z = -INFINITY;
    if (seen >> lane & 1) {
      const float* k = kp + (int64_t)(w * 64 + lane) * s.k_sn;
      f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int d = 0; d < D; d += 4) acc += *(const f32x4*)(qs + d) * *(const f32x4*)(k + d);
      z = ((acc[0] + acc[1]) + (acc[2] + acc[3])) * c;
    }
    float mx = z;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) mx = vmax(mx, __shfl_xor(mx, off));
    const float m_new = vmax(m, mx);
    const float ref = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = fast_exp2(m - ref);
    const float x = fast_exp2(z - ref);
    m = m_new;
    l = l * alpha + x;
#pragma unroll
    for (int i = 0; i < NC; ++i) o[i] *= alpha;
    for (uint64_t left = seen; left; left &= left - 1) {
      const int j = __builtin_ctzll(left);
      const float pj = __shfl(x, j);
      const float* v = vp + (int64_t)(w * 64 + j) * s.v_sn;
#pragma unroll
      for (int i = 0; i < NC; ++i)
        o[i] = fmaf(pj, v[lane + 64 * i], o[i]);
    }
  }
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) l += __shfl_xor(l, off);
  const TreeJoin j = tree_join(s.has_ctx, s.has_ctx ? lse[(int64_t)h * p.total_q + s.q0 + pos] : 0.f, m, l);
  float* const dst = (float*)p.o + tree_row(p.o_layout, b, h, s.q0, pos, p.o_sb, p.o_sh, p.o_sn);
  const float* const oc = octx + ((int64_t)h * p.total_q + s.q0 + pos) * D;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    float x = o[i] * j.wt;
    if (s.has_ctx) x = fmaf(j.wc, oc[lane + 64 * i], x);
    dst[lane + 64 * i] = x;
  }
}

bool tree_part_aligned(const fmlm_attn_params& p) {
  const int es = elem_size(p.dtype);
  const bool mla = p.flags & FMLM_FLAG_MLA;
  for (int64_t st : {p.q_sb, p.q_sh, p.q_sn, p.k_sb, p.k_sh, p.k_sn, p.o_sb, p.o_sh, p.o_sn})
    if ((st * es) % 16) return false;
  if (!mla && ((p.v_sb * es) % 16 || (p.v_sh * es) % 16 || (p.v_sn * es) % 16)) return false;
  return (((uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.o | (mla ? 0 : (uintptr_t)p.v)) & 15) == 0;
}

int launch_tree_part(const fmlm_attn_params& ctx, const fmlm_attn_params& p, const uint64_t* mask, int words,
                     int longest, void* stream) {
  const hipStream_t s = (hipStream_t)stream;
  const float* const octx = (const float*)ctx.o;
  if (p.dtype != FMLM_DTYPE_F32) {
    const dim3 grid((unsigned)(((int64_t)longest * p.H + 15) / 16), (unsigned)p.B);
    const dim3 block(kLatentWaves * 64);
    if (p.D != kLatentD || !(p.flags & FMLM_FLAG_MLA)) return FMLM_E_HEAD_DIM;
    if (p.dtype == FMLM_DTYPE_BF16)
      hipLaunchKernelGGL(attn_tree_latent_kernel<bf16>, grid, block, 0, s, p, octx, ctx.lse, mask, words);
    else
      hipLaunchKernelGGL(attn_tree_latent_kernel<f16>, grid, block, 0, s, p, octx, ctx.lse, mask, words);
    return launch_status();
  }
  const dim3 grid((unsigned)longest, (unsigned)p.H, (unsigned)p.B);
  if (p.D != kLatentD) return FMLM_E_HEAD_DIM;
  hipLaunchKernelGGL(attn_tree_f32_kernel<kLatentD>, grid, dim3(64), 0, s, p, octx, ctx.lse, mask, words);
  return launch_status();
}

}  // namespace fmlm

using namespace fmlm;

extern "C" int fmlm_tree_mask(const void* parents, int32_t parents_i64, const int32_t* cu_seqlens, int32_t B, int32_t N,
                              int32_t T, int32_t words, const void* ctx_lens, int32_t ctx_lens_i64, uint64_t* mask,
                              int32_t* positions, int32_t* n_bad, void* stream) {
  if (B < 0 || N < 0 || T < 0 || words < 0 || N > FMLM_MAX_TREE || (int64_t)words * 64 < N) return FMLM_E_ARG;
  if (B == 0 || T == 0) return 0;
  if (!parents || !cu_seqlens || !mask || !positions) return FMLM_E_ARG;
  const int threads = std::max(64, (N + 63) / 64 * 64);
  hipLaunchKernelGGL(tree_mask_kernel, dim3(B), dim3(threads), 0, (hipStream_t)stream, parents, parents_i64, cu_seqlens,
                     N, T, words, ctx_lens, ctx_lens_i64, mask, positions, n_bad);
  return launch_status();
}
