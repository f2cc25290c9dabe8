// Norms of queries and keys for each head with the position rotation, and their gradients.
//
// A row is one head's D elements x of one token at position s.  Forward, in fp32:
//   r = (mean(x^2) + eps)^-1/2,  n_d = x_d r w_d,
//   pairs (a, b) of the first R elements of n:  (a c - b s, a s + b c),
//   c = cos[s, i], s = sin[s, i] of pair i: elements (i, i + R/2) or (2i, 2i + 1)
// and one rounding to the input type.  Backward, with g = dy rotated back by the same
// angles, u_d = g_d w_d and xh = x r:
//   dx = r (u - xh mean(u xh)),   dw_d = sum over rows of g_d xh_d.
// The norm is recomputed from x: x has to be read anyway.
//
// Each pass is bound by memory: a row is read once and written once (forward), x and dy
// read and dx written (backward).  A row belongs to D / 8 neighbouring lanes, 8 elements (one
// 16-byte load of a 16-bit type) each, so its sums are lane sums without LDS.  A thread
// keeps its row's angles in registers over several heads (they are 64 bytes a thread, four
// times its share of a 16-bit row).  The partner of a half-split pair is fetched from its
// lane as raw input, which is half as many lane reads as normalised floats for 16-bit rows.
// dw: each workgroup sums its rows in registers and writes one partial row of D floats;
// a second kernel adds the partials up, always in the same order.
//
// Measured (a large copy reaches 5.16 TB/s).  Forward, 32 sequences of 256-1024 tokens, 16 heads of
// q and k, D = 128, fp16, padding rows written as zeros: 457 MB in 90 us, 5.1 TB/s; packed rows
// with gains per head, 359 MB in 67.  Backward of the latter, 539 MB in 119 to 124 + 5 us (4.4 TB/s), and
// 112 + 5 with shared gains.  64 decoding tokens: 4.4 us, latency.
#include "fmlm_common.h"

#include <algorithm>
#include <type_traits>

namespace fmlm {

constexpr int kNrThreads = 256;
constexpr int kNrHeads = 4;  // heads in flight per thread

typedef fmlm_norm_rope_params NrParams;
typedef fmlm_norm_rope_tensor NrTensor;

// ---- 8 elements of a row, as loaded (raw dwords) and as floats
template <typename T>
struct Oct {
  static constexpr int W = sizeof(T) == 2 ? 4 : 8;  // dwords
  uint32_t w[W];
};
template <typename T>
FMLM_DEV Oct<T> oct_load(const T* p) {
  Oct<T> o;
#pragma unroll
  for (int i = 0; i < Oct<T>::W; i += 4) {
    const u32x4 v = *(const u32x4*)((const char*)p + 4 * i);
#pragma unroll
    for (int j = 0; j < 4; ++j) o.w[i + j] = v[j];
  }
  return o;
}
template <typename T>
FMLM_DEV void oct_floats(const Oct<T>& o, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __builtin_bit_cast(float, o.w[i]);
  } else if constexpr (std::is_same<T, bf16>::value) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __builtin_bit_cast(float, o.w[i] << 16);
      x[2 * i + 1] = __builtin_bit_cast(float, o.w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const auto v = __builtin_bit_cast(typename Pair<f16>::type, o.w[i]);
      x[2 * i] = (float)v[0];
      x[2 * i + 1] = (float)v[1];
    }
  }
}
template <typename T>
FMLM_DEV void oct_store(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    *(f32x4*)p = f32x4{x[0], x[1], x[2], x[3]};
    *((f32x4*)p + 1) = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x[2 * i], x[2 * i + 1]}, typename Pair<T>::type));
    *(u32x4*)p = v;
  }
}

template <int CTRL>
FMLM_DEV float dpp_add(float x) {
  const int y = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true);
  return x + __builtin_bit_cast(float, y);
}
// sum over the LPR lanes of a row (LPR a power of two, rows aligned to it)
template <int LPR>
FMLM_DEV float lane_sum(float x) {
  if constexpr (LPR >= 2) x = dpp_add<0xB1>(x);   // lanes l ^ 1
  if constexpr (LPR >= 4) x = dpp_add<0x4E>(x);   // l ^ 2
  if constexpr (LPR >= 8) x = dpp_add<0x141>(x);  // the other four of eight lanes
  if constexpr (LPR >= 16) x = dpp_add<0x140>(x); // the other eight of sixteen
  if constexpr (LPR >= 32) {
    const int xi = __builtin_bit_cast(int, x);
    const auto a = __builtin_amdgcn_permlane16_swap(xi, xi, false, false);
    x = __builtin_bit_cast(float, (int)a[0]) + __builtin_bit_cast(float, (int)a[1]);
  }
  if constexpr (LPR >= 64) {
    const int xi = __builtin_bit_cast(int, x);
    const auto a = __builtin_amdgcn_permlane32_swap(xi, xi, false, false);
    x = __builtin_bit_cast(float, (int)a[0]) + __builtin_bit_cast(float, (int)a[1]);
  }
  return x;
}

// 8 gains from element d on (1 without gains)
FMLM_DEV void load_gain(const NrParams& p, const NrTensor& t, int h, int d, float (&w)[8]) {
  if (!t.weight) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 1.f;
    return;
  }
  const int64_t at = (int64_t)h * t.w_sh + d;
  if (p.w_dtype == FMLM_DTYPE_BF16) oct_floats(oct_load((const bf16*)t.weight + at), w);
  else if (p.w_dtype == FMLM_DTYPE_F16) oct_floats(oct_load((const f16*)t.weight + at), w);
  else oct_floats(oct_load((const float*)t.weight + at), w);
}

FMLM_DEV int64_t index_at(const void* a, bool i64, int64_t i) {
  return i64 ? ((const int64_t*)a)[i] : (int64_t)((const int32_t*)a)[i];
}

// Row i of the call (padded: b * N + pos; packed: token i): its sequence and position in
// it, the index of its packed or padded token, whether it is a token at all.
struct NrRow {
  int b, pos;
  bool real;
  int64_t angle;  // row of the angle tables
};
FMLM_DEV NrRow nr_row(const NrParams& p, int i) {
  NrRow r;
  uint32_t at = (uint32_t)i;
  if (p.layout == FMLM_LAYOUT_PACKED && p.token_indices) at = (uint32_t)p.token_indices[i];
  const uint32_t b = at / (uint32_t)p.N;
  r.pos = (int)(at - b * (uint32_t)p.N);
  r.b = (int)min(b, (uint32_t)p.B - 1u);
  r.real = true;
  int64_t tok = i;  // index into positions
  if (p.cu_seqlens && p.layout == FMLM_LAYOUT_PADDED) {
    // (a token past the positions is none, whatever the offsets say)
    const int c0 = p.cu_seqlens[r.b], at = c0 + r.pos;
    r.real = r.pos < p.cu_seqlens[r.b + 1] - c0 && (p.n_positions == 0 || (uint32_t)at < (uint32_t)p.n_positions);
    tok = at;
  }
  r.angle = 0;
  if (p.rotary_dim > 0 && r.real) {
    int64_t s = r.pos;
    if (p.positions) s = index_at(p.positions, p.flags & FMLM_NR_POSITIONS_I64, tok);
    else if (p.offsets) s += index_at(p.offsets, p.flags & FMLM_NR_OFFSETS_I64, r.b);
    r.angle = s < 0 ? 0 : s < p.table_rows ? s : p.table_rows - 1;
  }
  return r;
}

// The angles of a thread's 8 elements from element d on: cs / sn of element j, and the lane
// of its row that holds the other halves of its pairs.  Interleaved pairs are the thread's
// own.  The sign of sn is the pair member's: y_j = n_j cs_j + n_partner sn_j.
struct Angles {
  float cs[8], sn[8];
  int from;     // lane of the wave with the partners (half-split)
  bool turned;  // some element is rotated
};
template <int LPR>
FMLM_DEV Angles load_angles(const NrParams& p, int64_t row, int c) {
  Angles a;
  const int half = p.rotary_dim / 2, d = 8 * c;
  a.turned = d < p.rotary_dim;
  const int lane = threadIdx.x & 63;
  a.from = lane;
  if (!a.turned) return a;
  if (p.flags & FMLM_NR_INTERLEAVED) {
    const f32x4 cv = *(const f32x4*)(p.cos + row * half + d / 2);
    const f32x4 sv = *(const f32x4*)(p.sin + row * half + d / 2);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      a.cs[j] = cv[j / 2];
      a.sn[j] = j & 1 ? sv[j / 2] : -sv[j / 2];
    }
  } else {
    const bool hi = d >= half;
    const int64_t at = row * half + (hi ? d - half : d);
    a.from = hi ? lane - half / 8 : lane + half / 8;
#pragma unroll
    for (int j = 0; j < 8; j += 4) {
      const f32x4 cv = *(const f32x4*)(p.cos + at + j);
      const f32x4 sv = *(const f32x4*)(p.sin + at + j);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a.cs[j + i] = cv[i];
        a.sn[j + i] = hi ? sv[i] : -sv[i];
      }
    }
  }
  return a;
}

// the partner lane's raw elements (every lane of the row takes part)
template <typename T>
FMLM_DEV Oct<T> oct_from(const Oct<T>& o, int lane) {
  Oct<T> r;
#pragma unroll
  for (int i = 0; i < Oct<T>::W; ++i) r.w[i] = (uint32_t)__builtin_amdgcn_ds_bpermute(lane * 4, (int)o.w[i]);
  return r;
}

// head chunk blockIdx.y: chunks of hc heads of q, then of k
struct NrChunk {
  const NrTensor* t;
  int h0, h1, tensor;
};
FMLM_DEV NrChunk nr_chunk(const NrParams& p, int hc) {
  NrChunk k;
  const int nq = (p.q.heads + hc - 1) / hc;
  const int y = blockIdx.y;
  k.tensor = y >= nq;
  k.t = k.tensor ? &p.k : &p.q;
  k.h0 = (k.tensor ? y - nq : y) * hc;
  k.h1 = min(k.h0 + hc, (int)k.t->heads);
  return k;
}

FMLM_DEV int64_t nr_offset(const NrParams& p, int i, const NrRow& r, int64_t sb, int64_t sn) {
  return p.layout == FMLM_LAYOUT_PACKED ? (int64_t)i * sn : (int64_t)r.b * sb + (int64_t)r.pos * sn;
}

// PERHEAD: gains for each head, which the workgroup puts into LDS as floats (loaded from memory
// head by head they held up every row: 32 sequences of 256-1024 tokens, 16 heads, D = 128, 88 us
// instead of 71).
constexpr int kNrGains = 4096;  // floats of them
template <typename T, int LPR, bool PERHEAD>
__global__ __launch_bounds__(kNrThreads) void norm_rope_kernel(const NrParams p, int hc) {
  constexpr int RPB = kNrThreads / LPR, D = 8 * LPR;
  constexpr int U = kNrHeads;
  __shared__ __align__(16) float gains[PERHEAD ? kNrGains : 1];
  const int c = threadIdx.x % LPR;
  const int64_t i64 = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR;
  const NrChunk ck = nr_chunk(p, hc);
  const NrTensor& t = *ck.t;
  if constexpr (PERHEAD) {
    for (int at = 8 * threadIdx.x; at < (ck.h1 - ck.h0) * D; at += 8 * kNrThreads) {
      float w[8];
      load_gain(p, t, ck.h0 + at / D, at % D, w);
      oct_store(gains + at, w);
    }
    __syncthreads();
  }
  if (i64 >= p.rows) return;  // whole rows
  const int i = (int)i64;
  const NrRow r = nr_row(p, i);
  const T* src = (const T*)t.x + nr_offset(p, i, r, t.x_sb, t.x_sn) + 8 * c;
  T* dst = (T*)t.y + nr_offset(p, i, r, t.y_sb, t.y_sn) + 8 * c;
  if (!r.real) {
    const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int h = ck.h0; h < ck.h1; ++h) oct_store(dst + h * t.y_sh, z);
    return;
  }
  // the first heads' rows before what the angles and gains wait for
  Oct<T> x[U];
  auto load = [&](int h) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (h + u < ck.h1) x[u] = oct_load(src + (h + u) * t.x_sh);
  };
  load(ck.h0);
  const bool norm = p.flags & FMLM_NR_NORM, inter = p.flags & FMLM_NR_INTERLEAVED;
  const Angles a = load_angles<LPR>(p, r.angle, c);
  const int cp = c + (a.from - ((int)threadIdx.x & 63));  // the partner's chunk
  float w[8], wp[8];
  if constexpr (!PERHEAD) {
    load_gain(p, t, 0, 8 * c, w);
    load_gain(p, t, 0, 8 * cp, wp);
  }
  for (int h = ck.h0; h < ck.h1; h += U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (h + u >= ck.h1) break;
      if constexpr (PERHEAD) {
        const float* g = gains + (h + u - ck.h0) * D;
        oct_floats(oct_load(g + 8 * c), w);
        oct_floats(oct_load(g + 8 * cp), wp);
      }
      float n[8], y[8];
      oct_floats(x[u], n);
      float rs = 1.f;
      if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(n[j], n[j], ss);
        ss = lane_sum<LPR>(ss);
        rs = rsqrtf(ss * (1.f / (8 * LPR)) + p.eps);
      }
      if (p.rotary_dim > 0 && !inter) {
        float q[8];
        oct_floats(oct_from(x[u], a.from), q);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float own = n[j] * rs * w[j];
          y[j] = a.turned ? fmaf(own, a.cs[j], q[j] * rs * wp[j] * a.sn[j]) : own;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) n[j] = n[j] * rs * w[j];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = a.turned ? fmaf(n[j], a.cs[j], n[j ^ 1] * a.sn[j]) : n[j];
      }
      oct_store(dst + (h + u) * t.y_sh, y);
    }
    if (h + U < ck.h1) load(h + U);
  }
}

// Backward.  A workgroup takes row tiles blockIdx.x, + gridDim.x, ... of kNrHeads heads;
// its sums of dw go to row chunk * gridDim.x + blockIdx.x of the tensor's part of the
// workspace, or with PERHEAD (a tensor has gains per head) to head * gridDim.x + blockIdx.x
// for each of its heads.
template <typename T, int LPR, bool PERHEAD>
__global__ __launch_bounds__(kNrThreads, sizeof(T) == 2 ? 4 : 3) void norm_rope_bwd_kernel(const NrParams p, float* part_q, float* part_k) {
  constexpr int RPB = kNrThreads / LPR, D = 8 * LPR;
  constexpr int U = kNrHeads, NA = PERHEAD ? U : 1;
  __shared__ __align__(16) float red[kNrThreads / 64][D];
  const int c = threadIdx.x % LPR;
  const NrChunk ck = nr_chunk(p, U);
  const NrTensor& t = *ck.t;
  float* const part = ck.tensor ? part_k : part_q;
  const bool norm = p.flags & FMLM_NR_NORM, inter = p.flags & FMLM_NR_INTERLEAVED;
  // gains per head in LDS: in 32 registers of a thread the kernel had 3 waves a SIMD and took 7 us more.
  // The sums of dw for each head still cost the 16-bit types 4 to 6 spilled registers at four waves (20
  // to 28 bytes of scratch a lane): 539 MB in 119 to 124 us where shared gains, unspilled, take 112
  __shared__ __align__(16) float gains[PERHEAD ? U * D : 1];
  float w[8];
  if constexpr (PERHEAD) {
    for (int at = 8 * threadIdx.x; at < (ck.h1 - ck.h0) * D; at += 8 * kNrThreads) {
      load_gain(p, t, ck.h0 + at / D, at % D, w);
      oct_store(gains + at, w);
    }
    __syncthreads();
  } else {
    load_gain(p, t, 0, 8 * c, w);
  }
  float dw[NA][8];
#pragma unroll
  for (int u = 0; u < NA; ++u)
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[u][j] = 0.f;

  const int64_t tiles = (p.rows + RPB - 1) / RPB;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t i64 = tile * RPB + threadIdx.x / LPR;
    if (i64 >= p.rows) break;  // whole rows, and no later tile has any
    const int i = (int)i64;
    const NrRow r = nr_row(p, i);
    const T* xs = (const T*)t.x + nr_offset(p, i, r, t.x_sb, t.x_sn) + 8 * c;
    const T* ds = (const T*)t.dy + nr_offset(p, i, r, t.dy_sb, t.dy_sn) + 8 * c;
    T* dst = (T*)t.y + nr_offset(p, i, r, t.y_sb, t.y_sn) + 8 * c;
    if (!r.real) {
      const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int h = ck.h0; h < ck.h1; ++h) oct_store(dst + h * t.y_sh, z);
      continue;
    }
    Oct<T> x[U], dy[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (ck.h0 + u < ck.h1) {
        dy[u] = oct_load(ds + (ck.h0 + u) * t.dy_sh);
        if (norm) x[u] = oct_load(xs + (ck.h0 + u) * t.x_sh);
      }
    const Angles a = load_angles<LPR>(p, r.angle, c);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (ck.h0 + u >= ck.h1) break;
      const int iu = PERHEAD ? u : 0;
      float g[8], gr[8], xv[8];
      if constexpr (PERHEAD) oct_floats(oct_load(gains + u * D + 8 * c), w);
      oct_floats(dy[u], gr);
      if (p.rotary_dim > 0 && !inter) {
        float q[8];
        oct_floats(oct_from(dy[u], a.from), q);
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = a.turned ? fmaf(gr[j], a.cs[j], -q[j] * a.sn[j]) : gr[j];
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = a.turned ? fmaf(gr[j], a.cs[j], -gr[j ^ 1] * a.sn[j]) : gr[j];
      }
      if (norm) {
        oct_floats(x[u], xv);
        float ss = 0.f, ux = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          ss = fmaf(xv[j], xv[j], ss);
          ux = fmaf(g[j] * w[j], xv[j], ux);
        }
        ss = lane_sum<LPR>(ss);
        ux = lane_sum<LPR>(ux);
        const float rs = rsqrtf(ss * (1.f / D) + p.eps);
        const float m = ux * rs * (1.f / D);  // mean(u xh)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float xh = xv[j] * rs;
          dw[iu][j] = fmaf(g[j], xh, dw[iu][j]);
          g[j] = rs * fmaf(-xh, m, g[j] * w[j]);
        }
      }
      oct_store(dst + (ck.h0 + u) * t.y_sh, g);
    }
  }
  if (!t.dweight) return;
  // the workgroup's sums: over a wave's rows by lanes, then over the waves
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int u = 0; u < NA; ++u) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int off = LPR; off < 64; off <<= 1) dw[u][j] += __shfl_xor(dw[u][j], off);
    if (lane < LPR) {
#pragma unroll
      for (int j = 0; j < 8; ++j) red[wave][8 * c + j] = dw[u][j];
    }
    __syncthreads();
    const int64_t row = PERHEAD ? (int64_t)(ck.h0 + u) * gridDim.x + blockIdx.x
                                : (int64_t)(ck.h0 / U) * gridDim.x + blockIdx.x;
    if (!PERHEAD || ck.h0 + u < ck.h1)
      for (int d = threadIdx.x; d < D; d += kNrThreads) {
        float s = 0.f;
#pragma unroll
        for (int v = 0; v < kNrThreads / 64; ++v) s += red[v][d];
        part[row * D + d] = s;
      }
    __syncthreads();
  }
}

// dw row h of a tensor from its n partial rows: 16 columns a workgroup, its 64 slices of rows
// added up in order (5 us, the latency of a launch and of its loads)
constexpr int kNrSumThreads = 1024;
constexpr int kNrSumCols = 16;
__global__ __launch_bounds__(kNrSumThreads) void norm_rope_dw_kernel(const NrParams p, const float* part_q,
                                                                     const float* part_k, int nq, int nk) {
  constexpr int S = kNrSumThreads / kNrSumCols;
  __shared__ float red[S][kNrSumCols + 1];
  const int rows_q = p.q.dweight ? (p.q.w_sh ? p.q.heads : 1) : 0;
  const bool is_k = (int)blockIdx.y >= rows_q;
  const NrTensor& t = is_k ? p.k : p.q;
  const int h = is_k ? blockIdx.y - rows_q : blockIdx.y;
  const int n = is_k ? nk : nq;
  const float* src = (is_k ? part_k : part_q) + (int64_t)h * n * p.D;
  const int col = blockIdx.x * kNrSumCols + threadIdx.x % kNrSumCols, s = threadIdx.x / kNrSumCols;
  float acc = 0.f;
#pragma unroll 8
  for (int i = s; i < n; i += S) acc += src[(int64_t)i * p.D + col];
  red[s][threadIdx.x % kNrSumCols] = acc;
  __syncthreads();
  for (int off = S / 2; off > 0; off >>= 1) {
    if (s < off) red[s][threadIdx.x % kNrSumCols] += red[s + off][threadIdx.x % kNrSumCols];
    __syncthreads();
  }
  if (s == 0) {
    const float v = red[0][threadIdx.x % kNrSumCols];
    const int64_t at = (int64_t)h * p.D + col;
    if (p.w_dtype == FMLM_DTYPE_BF16) ((bf16*)t.dweight)[at] = (bf16)v;
    else if (p.w_dtype == FMLM_DTYPE_F16) ((f16*)t.dweight)[at] = (f16)v;
    else ((float*)t.dweight)[at] = v;
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
static bool nr_aligned(const void* ptr, int64_t sb, int64_t sh, int64_t sn, int es) {
  auto ok = [&](int64_t s) { return (s * es) % 16 == 0; };
  return ((uintptr_t)ptr & 15) == 0 && ok(sb) && ok(sh) && ok(sn);
}

static int nr_check(const NrParams& p, bool bwd) {
  const int es = elem_size(p.dtype);
  if (!es) return FMLM_E_DTYPE;
  if (p.w_dtype != FMLM_DTYPE_BF16 && p.w_dtype != FMLM_DTYPE_F16 && p.w_dtype != FMLM_DTYPE_F32) return FMLM_E_DTYPE;
  switch (p.D) {
    case 16: case 32: case 64: case 128: case 256: case 512: break;
    default: return FMLM_E_HEAD_DIM;
  }
  if (p.B < 0 || p.N < 0 || p.rows < 0 || p.q.heads < 0 || p.k.heads < 0) return FMLM_E_ARG;
  if ((int64_t)p.B * p.N > 0x7fffffff || p.rows > 0x7fffffff) return FMLM_E_ARG;
  if (p.layout != FMLM_LAYOUT_PADDED && p.layout != FMLM_LAYOUT_PACKED) return FMLM_E_ARG;
  if (p.rows > 0 && p.N < 1) return FMLM_E_ARG;
  if (p.layout == FMLM_LAYOUT_PADDED ? p.rows != (int64_t)p.B * p.N : p.rows > (int64_t)p.B * p.N) return FMLM_E_ARG;
  if (p.layout == FMLM_LAYOUT_PACKED && !p.token_indices && p.B != 1) return FMLM_E_ARG;
  if (p.rotary_dim < 0 || p.rotary_dim > p.D || p.rotary_dim % 16) return FMLM_E_ARG;
  if (p.rotary_dim > 0 && (!p.cos || !p.sin || p.table_rows < 1)) return FMLM_E_ARG;
  if (p.rotary_dim > 0 && (((uintptr_t)p.cos | (uintptr_t)p.sin) & 15)) return FMLM_E_ALIGN;
  for (const NrTensor* t : {&p.q, &p.k}) {
    if (t->heads == 0 || p.rows == 0) continue;
    if (!t->x || !t->y || (bwd && !t->dy)) return FMLM_E_ARG;
    if (t->w_sh != 0 && t->w_sh != p.D) return FMLM_E_ARG;
    if (!nr_aligned(t->x, t->x_sb, t->x_sh, t->x_sn, es) || !nr_aligned(t->y, t->y_sb, t->y_sh, t->y_sn, es) ||
        ((uintptr_t)t->weight & 15))
      return FMLM_E_ALIGN;
    if (bwd && !nr_aligned(t->dy, t->dy_sb, t->dy_sh, t->dy_sn, es)) return FMLM_E_ALIGN;
    if (bwd && t->dweight && (!t->weight || !(p.flags & FMLM_NR_NORM))) return FMLM_E_ARG;
  }
  return 0;
}

static int div_up(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

static bool nr_per_head(const NrParams& p) { return p.q.w_sh || p.k.w_sh; }

// Heads a forward thread works through: all of them where that leaves enough workgroups (the
// angles are then loaded once), else fewer.  32 sequences of 64-512 tokens, 12 heads, D = 64, bf16: 18.7
// us with at least 1024 workgroups, 22.3 with 4096, 36 with 8192; 64 decoding tokens, 16 heads of 128:
// 5.1, 5.4, 5.7.  Heads in flight (kNrHeads): 2, 4 and 8 take 36.5, 18.7 and 40.5 us in the former.
constexpr int kNrMinGroups = 1024;
static int nr_heads_per_chunk(const NrParams& p) {
  const int tiles = div_up(p.rows, kNrThreads / (p.D / 8));
  const int most = std::max(p.q.heads, p.k.heads);
  int hc = nr_per_head(p) ? std::min(most, kNrGains / p.D) : most;
  while (hc > 1 && (int64_t)tiles * (div_up(p.q.heads, hc) + div_up(p.k.heads, hc)) < kNrMinGroups) hc = (hc + 1) / 2;
  return hc;
}

// Row tiles side by side in the backward: enough for the GPU, few enough partial rows of dw (512 to
// 4096 workgroups differ by 3% in the sizes above).
constexpr int kNrBwdGroups = 2048;
static int nr_bwd_grid(const NrParams& p) {
  const int tiles = div_up(p.rows, kNrThreads / (p.D / 8));
  const int chunks = std::max(1, div_up(p.q.heads, kNrHeads) + div_up(p.k.heads, kNrHeads));
  return std::max(1, std::min(tiles, std::max(1, kNrBwdGroups / chunks)));
}
// partial rows of a row of dw
static int64_t nr_partials(const NrParams& p, const NrTensor& t, int gx) {
  return (int64_t)gx * (t.w_sh ? 1 : nr_per_head(p) ? t.heads : div_up(t.heads, kNrHeads));
}
static int64_t nr_partial_floats(const NrParams& p, const NrTensor& t, int gx) {
  return t.dweight ? nr_partials(p, t, gx) * (t.w_sh ? t.heads : 1) * p.D : 0;
}

template <typename T, bool PERHEAD>
static int nr_launch(const NrParams& p, hipStream_t s) {
  const int hc = nr_heads_per_chunk(p), lpr = p.D / 8;
  const dim3 grid((unsigned)div_up(p.rows, kNrThreads / lpr), (unsigned)(div_up(p.q.heads, hc) + div_up(p.k.heads, hc)));
#define FMLM_NR(L) case L: hipLaunchKernelGGL((norm_rope_kernel<T, L, PERHEAD>), grid, dim3(kNrThreads), 0, s, p, hc); break;
  switch (lpr) { FMLM_NR(2) FMLM_NR(4) FMLM_NR(8) FMLM_NR(16) FMLM_NR(32) FMLM_NR(64) }
#undef FMLM_NR
  return launch_status();
}

template <typename T, bool PERHEAD>
static int nr_bwd_launch(const NrParams& p, hipStream_t s) {
  const int gx = nr_bwd_grid(p), lpr = p.D / 8;
  float* const part_q = (float*)p.workspace;
  float* const part_k = part_q + nr_partial_floats(p, p.q, gx);
  const dim3 grid((unsigned)gx, (unsigned)(div_up(p.q.heads, kNrHeads) + div_up(p.k.heads, kNrHeads)));
#define FMLM_NR(L) \
  case L: hipLaunchKernelGGL((norm_rope_bwd_kernel<T, L, PERHEAD>), grid, dim3(kNrThreads), 0, s, p, part_q, part_k); break;
  switch (lpr) { FMLM_NR(2) FMLM_NR(4) FMLM_NR(8) FMLM_NR(16) FMLM_NR(32) FMLM_NR(64) }
#undef FMLM_NR
  const int rows_q = p.q.dweight ? (p.q.w_sh ? p.q.heads : 1) : 0, rows_k = p.k.dweight ? (p.k.w_sh ? p.k.heads : 1) : 0;
  if (rows_q + rows_k > 0)
    hipLaunchKernelGGL(norm_rope_dw_kernel, dim3(p.D / kNrSumCols, rows_q + rows_k), dim3(kNrSumThreads), 0, s, p, part_q,
                       part_k, (int)nr_partials(p, p.q, gx), (int)nr_partials(p, p.k, gx));
  return launch_status();
}

}  // namespace fmlm

using namespace fmlm;

extern "C" int fmlm_norm_rope_params_size(void) { return (int)sizeof(fmlm_norm_rope_params); }

extern "C" int fmlm_norm_rope(const fmlm_norm_rope_params* pp, void* stream) {
  if (!pp) return FMLM_E_ARG;
  const int rc = nr_check(*pp, false);
  if (rc) return rc;
  if (pp->rows == 0 || pp->q.heads + pp->k.heads == 0) return 0;
  const bool per_head = nr_per_head(*pp);
  hipStream_t s = (hipStream_t)stream;
  switch (pp->dtype) {
    case FMLM_DTYPE_BF16: return per_head ? nr_launch<bf16, true>(*pp, s) : nr_launch<bf16, false>(*pp, s);
    case FMLM_DTYPE_F16: return per_head ? nr_launch<f16, true>(*pp, s) : nr_launch<f16, false>(*pp, s);
    default: return per_head ? nr_launch<float, true>(*pp, s) : nr_launch<float, false>(*pp, s);
  }
}

extern "C" int64_t fmlm_norm_rope_bwd_workspace_bytes(const fmlm_norm_rope_params* pp) {
  if (!pp) return FMLM_E_ARG;
  const int rc = nr_check(*pp, true);
  if (rc) return rc;
  const int gx = nr_bwd_grid(*pp);
  return 4 * (nr_partial_floats(*pp, pp->q, gx) + nr_partial_floats(*pp, pp->k, gx));
}

extern "C" int fmlm_norm_rope_bwd(const fmlm_norm_rope_params* pp, void* stream) {
  if (!pp) return FMLM_E_ARG;
  const int64_t need = fmlm_norm_rope_bwd_workspace_bytes(pp);
  if (need < 0) return (int)need;
  if (need > 0 && (!pp->workspace || pp->workspace_bytes < need)) return FMLM_E_WORKSPACE;
  // (no rows: the gains' gradients are sums over nothing, and the launch writes zeros)
  if (pp->q.heads + pp->k.heads == 0) return 0;
  const bool per_head = nr_per_head(*pp);
  hipStream_t s = (hipStream_t)stream;
  switch (pp->dtype) {
    case FMLM_DTYPE_BF16: return per_head ? nr_bwd_launch<bf16, true>(*pp, s) : nr_bwd_launch<bf16, false>(*pp, s);
    case FMLM_DTYPE_F16: return per_head ? nr_bwd_launch<f16, true>(*pp, s) : nr_bwd_launch<f16, false>(*pp, s);
    default: return per_head ? nr_bwd_launch<float, true>(*pp, s) : nr_bwd_launch<float, false>(*pp, s);
  }
}
