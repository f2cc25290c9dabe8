// Appends to a paged context with the position rotation on the way, in 16 or in 4 bits, and the
// values of 4-bit rows.
//
// Rotation: of a row at position s, the pairs (a, b) of its first R elements become
// (a c - b s', a s' + b c) with c, s' = cos[s, i], sin[s, i] of pair i.  One rounding to the input
// type (q, and k in 16 bits).
// 4 bits: with A the largest magnitude of 32 neighbouring values, e is the smallest integer with
// A < 7 2^e: everything then rounds within the codes (A to at most 6).  A = f 2^x with f in
// [1, 2) gives e = x - 2 for f < 7/4, else x - 1.  The instruction that makes codes rounds
// x 2^-e to nearest even; 2^-e is exact, so a code depends on its block's values alone.  A rotated key
// is no 16-bit value: rounded to fp32 on the way it could come out on the border of two codes.  It is
// computed in fp64, where the products of 11-bit values and fp32 angles are exact, and goes to
// fp32 with rounding to odd, which keeps it on its side of every border.  (fp64 runs at half the fp32
// rate here: nothing beside the memory.)
//
// Bound by memory: every row is read once and written once.  A row belongs to D / 8 neighbouring
// lanes, 8 elements each, so that a block's maximum is a maximum of four lanes; a thread keeps its
// row's angles over its heads.  The partner of a half-split pair comes from its lane, as read.
// Measured: 589 MB of fp16 prompts 115 us, a large copy's rate; 20 thousand tokens with 12 heads
// of 64 stored in 4 bits 47 us, their values made again 19 us (together at 83% of that rate); 64 tokens with 16
// heads of 128 4.9 us.
#include "fmlm_common.h"

#include <algorithm>
#include <type_traits>

#include "fmlm_fp4.h"

namespace fmlm {

constexpr int kRaThreads = 256;
constexpr int kRaHeads = 4;  // heads of a thread whose loads are in flight

constexpr int kRaHeads4 = 2;  // ... of the 4-bit kernel, whose 64-bit rotation takes registers
constexpr int kRaMany = 16;
constexpr int64_t kRaManyThreads = 256 * 2048 / 3;  // threads of one of q, k, v that fill their share of the GPU

typedef fmlm_append_params RaParams;

template <typename T>
FMLM_DEV void oct_of(u32x4 w, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = w[i];  // (a bit_cast of the vector's element itself takes element 0)
    const auto v = __builtin_bit_cast(typename Pair<T>::type, u);
    x[2 * i] = (float)v[0];
    x[2 * i + 1] = (float)v[1];
  }
}
template <typename T>
FMLM_DEV u32x4 oct_to(const float (&x)[8]) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x[2 * i], x[2 * i + 1]}, typename Pair<T>::type));
  return v;
}

// x to fp32, rounded to odd: cut off, the last bit set when anything was
FMLM_DEV float round_to_odd(double x) {
  const float f = (float)x;
  uint32_t u = __builtin_bit_cast(uint32_t, f);
  const double d = (double)f;
  if (d != x && x == x) {
    if (fabs(d) > fabs(x)) --u;  // (an overflow to infinity becomes the largest value)
    u |= 1u;
  }
  return __builtin_bit_cast(float, u);
}

// the larger of x and x of the lane whose number differs in bit 0 / bit 1 (NaN if either is)
template <int CTRL>
FMLM_DEV float quad_max(float x) {
  const int y = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true);
  return vmax(x, __builtin_bit_cast(float, y));
}
FMLM_DEV float block_max(const float (&x)[8]) {
  float a = fabsf(x[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) a = vmax(a, fabsf(x[i]));
  return quad_max<0x4E>(quad_max<0xB1>(a));
}

// the codes of 8 values, a quarter of their block, whose other quarters the three lanes beside hold
template <typename T>
FMLM_DEV uint32_t fp4_encode(float (&x)[8], uint32_t& scale_byte) {
  constexpr bool BF = std::is_same<T, bf16>::value;
  constexpr float top = BF ? 0x1.fep127f : 65504.f;
  constexpr int lo = BF ? -125 : -23, hi = BF ? 125 : 13;
  float a = block_max(x);
  if (__builtin_amdgcn_ballot_w64(!(a <= top))) {  // an infinity, NaN or a rotated value past the type's
    asm volatile("");  // (a real branch)
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] == x[i] ? fminf(fmaxf(x[i], -top), top) : 0.f;
    a = block_max(x);
  }
  const uint32_t u = __builtin_bit_cast(uint32_t, a);
  int e = (int)(u >> 23) - 127 - ((u & 0x7fffffu) < 0x600000u ? 2 : 1);
  e = min(max(e, lo), hi);
  scale_byte = (uint32_t)(e + 127);
  const float s = fp4_scale(scale_byte);
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], s, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], s, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], s, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], s, 3);
  return c;
}

// blockIdx.y: chunk of `heads` heads, z: q, k, v, and slices of kRaGridX workgroups (a launch has fewer than 2^32
// threads in x).  Rows: padded ones b * N + pos, or packed tokens
constexpr unsigned kRaGridX = 1u << 23;
template <typename T, bool FP4>
__global__ __launch_bounds__(kRaThreads) void rotate_append_kernel(const RaParams p, int lpr_log2, int heads) {
  constexpr int NH = FP4 ? kRaHeads4 : kRaHeads;
  const int which = blockIdx.z % 3;
  const fmlm_append_rows& a = which == 0 ? p.q : which == 1 ? p.k : p.v;
  if (!a.dst) return;
  const bool padded = p.layout == FMLM_LAYOUT_PADDED;
  const int64_t at = ((int64_t)(blockIdx.z / 3) * kRaGridX + blockIdx.x) * kRaThreads + threadIdx.x;
  const int64_t row = at >> lpr_log2;
  if (row >= (padded ? (int64_t)p.B * p.N : p.T)) return;
  const int d = (int)(at - (row << lpr_log2)) * 8;
  int64_t t = row, src = row * a.s_sn, dst = row * a.d_sn;
  bool real = true;
  if (padded) {
    const int b = (int)((uint32_t)row / (uint32_t)p.N), pos = (int)row - b * p.N;
    const int c0 = p.cu_seqlens[b];
    t = (int64_t)c0 + pos;
    real = pos < p.cu_seqlens[b + 1] - c0 && t >= 0 && t < p.T;
    src = (int64_t)b * a.s_sb + (int64_t)pos * a.s_sn;
    dst = (int64_t)b * a.d_sb + (int64_t)pos * a.d_sn;
  }
  int h0 = blockIdx.y * heads;
  const int h1 = min(h0 + heads, p.H);
  T* const out = (T*)a.dst + dst + d;
  if (!real) {
    if (which == 0)
      for (int h = h0; h < h1; ++h) *(u32x4*)(out + h * a.d_sh) = u32x4{0u, 0u, 0u, 0u};
    return;
  }
  int64_t slot = 0;
  if (which > 0) {
    slot = p.slots[t];
    if (slot < 0 || slot >= p.pool_rows) return;
  }
  const bool turn = which < 2 && d < p.rotary_dim, pairs = p.flags & FMLM_AP_INTERLEAVED;
  const int half = p.rotary_dim / 2;
  // half-split: the lane of the row that holds the partners (every lane of a row has come this far)
  const int from = (threadIdx.x & 63) + (!turn ? 0 : d < half ? half / 8 : -half / 8);
  const T* in = (const T*)a.src + src + d;
  u32x4 x[NH];
  auto load = [&](int h) {
#pragma unroll
    for (int u = 0; u < NH; ++u)
      if (h + u < h1) x[u] = *(const u32x4*)(in + (h + u) * a.s_sh);
  };
  load(h0);
  float cs[8], sn[8];  // sn with the pair member's sign: element j becomes x_j cs_j + partner_j sn_j
  if (turn) {
    int64_t s = p.flags & FMLM_AP_POSITIONS_I64 ? ((const int64_t*)p.positions)[t] : ((const int32_t*)p.positions)[t];
    s = s < 0 ? 0 : s < p.table_rows ? s : p.table_rows - 1;
    if (pairs) {
      const f32x4 c4 = *(const f32x4*)(p.cos + s * half + d / 2), s4 = *(const f32x4*)(p.sin + s * half + d / 2);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        cs[j] = c4[j / 2];
        sn[j] = j & 1 ? s4[j / 2] : -s4[j / 2];
      }
    } else {
      const int64_t i = s * half + (d < half ? d : d - half);
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        const f32x4 c4 = *(const f32x4*)(p.cos + i + j), s4 = *(const f32x4*)(p.sin + i + j);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          cs[j + e] = c4[e];
          sn[j + e] = d < half ? -s4[e] : s4[e];
        }
      }
    }
  }
  for (; h0 < h1; h0 += NH) {
  u32x4 cur[NH];
#pragma unroll
  for (int u = 0; u < NH; ++u) cur[u] = x[u];
  if (h0 + NH < h1) load(h0 + NH);
#pragma unroll
  for (int u = 0; u < NH; ++u) {
    if (h0 + u >= h1) break;
    float f[8], g[8];
    oct_of<T>(cur[u], f);
    if (pairs) {
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = f[j ^ 1];
    } else if (which < 2 && p.rotary_dim > 0) {  // (the same in a wave: every lane gives its own)
      u32x4 y;
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * from, (int)cur[u][j]);
      oct_of<T>(y, g);
    }
    if (FP4 && which > 0) {
      if (turn) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = round_to_odd((double)f[j] * (double)cs[j] + (double)g[j] * (double)sn[j]);
      }
      uint32_t sb;
      const uint32_t c = fp4_encode<T>(f, sb);
      const int64_t e = ((int64_t)(h0 + u) * p.pool_rows + slot) * p.D + d;
      *(uint32_t*)((char*)a.dst + e / 2) = c;
      if (d % kFp4Block == 0) a.scales[e / kFp4Block] = (uint8_t)sb;
    } else {
      u32x4 v = cur[u];
      if (turn) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = fmaf(f[j], cs[j], g[j] * sn[j]);
        v = oct_to<T>(f);
      }
      T* const to = which == 0 ? out + (h0 + u) * a.d_sh
                               : (T*)a.dst + ((int64_t)(h0 + u) * p.pool_rows + slot) * p.D + d;
      *(u32x4*)to = v;
    }
  }  }
}

// 8 values a thread and step; blockIdx.y: pool
constexpr int kFvSteps = 4;
struct Fp4Pools {
  fmlm_fp4_rows t[2];
};
template <typename T>
__global__ __launch_bounds__(256) void fp4_values_kernel(const Fp4Pools pools, int64_t n) {
  const fmlm_fp4_rows& p = pools.t[blockIdx.y];
  const uint32_t* const codes = (const uint32_t*)p.codes;
  u32x4* const out = (u32x4*)p.out;
  const int64_t first = (int64_t)blockIdx.x * (256 * kFvSteps) + threadIdx.x;
  uint32_t c[kFvSteps], s[kFvSteps];
#pragma unroll
  for (int i = 0; i < kFvSteps; ++i) {
    const int64_t at = first + i * 256;
    if (at < n) {
      c[i] = codes[at];
      s[i] = p.scales[at / (kFp4Block / 8)];
    }
  }
#pragma unroll
  for (int i = 0; i < kFvSteps; ++i) {
    const int64_t at = first + i * 256;
    if (at < n) out[at] = fp4_oct<T>(c[i], fp4_scale(s[i]));
  }
}

static bool all16(uint64_t x) { return x % 16 == 0; }

static int check_append(const RaParams& p) {
  if (p.dtype != FMLM_DTYPE_BF16 && p.dtype != FMLM_DTYPE_F16) return FMLM_E_DTYPE;
  const bool fp4 = p.flags & FMLM_AP_FP4;
  if (p.D != 16 && p.D != 32 && p.D != 64 && p.D != 128 && p.D != 256) return FMLM_E_HEAD_DIM;
  if (fp4 && p.D < kFp4Block) return FMLM_E_HEAD_DIM;
  if (p.layout != FMLM_LAYOUT_PADDED && p.layout != FMLM_LAYOUT_PACKED) return FMLM_E_ARG;
  if (p.B < 0 || p.N < 0 || p.T < 0 || p.H < 0 || p.H > 65535 * kRaHeads || p.pool_rows < 0) return FMLM_E_ARG;
  if (p.rotary_dim < 0 || p.rotary_dim > p.D || p.rotary_dim % 16) return FMLM_E_ARG;
  if (p.rotary_dim > 0 && p.T > 0 && (!p.cos || !p.sin || !p.positions || p.table_rows < 1)) return FMLM_E_ARG;
  if (p.layout == FMLM_LAYOUT_PADDED && p.B > 0 && !p.cu_seqlens) return FMLM_E_ARG;
  if ((p.k.dst || p.v.dst) && p.T > 0 && !p.slots) return FMLM_E_ARG;
  const fmlm_append_rows* t[3] = {&p.q, &p.k, &p.v};
  for (int i = 0; i < 3; ++i) {
    const fmlm_append_rows& a = *t[i];
    if (!a.dst) continue;
    if (!a.src || (fp4 && i > 0 && !a.scales)) return FMLM_E_ARG;
    if (!all16((uint64_t)a.src | (uint64_t)(a.s_sb * 2) | (uint64_t)(a.s_sh * 2) | (uint64_t)(a.s_sn * 2)))
      return FMLM_E_ALIGN;
    if (i == 0 ? !all16((uint64_t)a.dst | (uint64_t)(a.d_sb * 2) | (uint64_t)(a.d_sh * 2) | (uint64_t)(a.d_sn * 2))
               : (uint64_t)a.dst % (fp4 ? 4 : 16) != 0)
      return FMLM_E_ALIGN;
  }
  if (!all16((uint64_t)p.cos | (uint64_t)p.sin)) return FMLM_E_ALIGN;
  return 0;
}

}  // namespace fmlm

using namespace fmlm;

extern "C" int fmlm_append_params_size(void) { return (int)sizeof(fmlm_append_params); }

extern "C" int fmlm_rotate_append(const fmlm_append_params* pp, void* stream) {
  if (!pp) return FMLM_E_ARG;
  const RaParams& p = *pp;
  const int rc = check_append(p);
  if (rc) return rc;
  const int64_t rows = p.layout == FMLM_LAYOUT_PADDED ? (int64_t)p.B * p.N : p.T;
  if (rows == 0 || p.H == 0) return 0;
  if (rows > 0x7fffffff) return FMLM_E_ARG;
  const int lpr = p.D / 8, lpr_log2 = __builtin_ctz(lpr);
  const int64_t blocks = (rows * lpr + kRaThreads - 1) / kRaThreads;
  if (blocks > 0x7fffffff) return FMLM_E_ARG;
  // Many rows: the angles, the slot and the sequence of a row serve kRaMany heads (fp16, 20 thousand rows of 16
  // heads, D = 128: 130 us with 4 heads a thread, 116 with 16); few: all the threads there are (64
  // rows of 16 heads 5.1 us, with 16 heads a thread 8.5)
  const int heads = rows * lpr >= kRaManyThreads ? kRaMany : kRaHeads;
  const dim3 grid((unsigned)std::min<int64_t>(blocks, kRaGridX), (p.H + heads - 1) / heads,
                  3 * (unsigned)((blocks + kRaGridX - 1) / kRaGridX));
  hipStream_t s = (hipStream_t)stream;
  const bool fp4 = p.flags & FMLM_AP_FP4;
  if (p.dtype == FMLM_DTYPE_BF16) {
    if (fp4) hipLaunchKernelGGL((rotate_append_kernel<bf16, true>), grid, dim3(kRaThreads), 0, s, p, lpr_log2, heads);
    else hipLaunchKernelGGL((rotate_append_kernel<bf16, false>), grid, dim3(kRaThreads), 0, s, p, lpr_log2, heads);
  } else {
    if (fp4) hipLaunchKernelGGL((rotate_append_kernel<f16, true>), grid, dim3(kRaThreads), 0, s, p, lpr_log2, heads);
    else hipLaunchKernelGGL((rotate_append_kernel<f16, false>), grid, dim3(kRaThreads), 0, s, p, lpr_log2, heads);
  }
  return launch_status();
}

extern "C" int fmlm_fp4_values(int32_t dtype, const fmlm_fp4_rows* tensors, int32_t n_tensors, int64_t rows, int32_t D,
                               void* stream) {
  if (dtype != FMLM_DTYPE_BF16 && dtype != FMLM_DTYPE_F16) return FMLM_E_DTYPE;
  if (D < kFp4Block || D % kFp4Block) return FMLM_E_HEAD_DIM;
  if (!tensors || n_tensors < 1 || n_tensors > 2 || rows < 0) return FMLM_E_ARG;
  if (rows == 0) return 0;
  Fp4Pools pools{};
  for (int i = 0; i < n_tensors; ++i) {
    const fmlm_fp4_rows& t = pools.t[i] = tensors[i];
    if (!t.codes || !t.scales || !t.out) return FMLM_E_ARG;
    if ((uint64_t)t.codes % 4 || (uint64_t)t.out % 16) return FMLM_E_ALIGN;
  }
  const int64_t n = rows * (D / 8), blocks = (n + 256 * kFvSteps - 1) / (256 * kFvSteps);
  if (blocks > 0x7fffffff) return FMLM_E_ARG;
  const dim3 grid((unsigned)blocks, n_tensors);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == FMLM_DTYPE_BF16) hipLaunchKernelGGL(fp4_values_kernel<bf16>, grid, dim3(256), 0, s, pools, n);
  else hipLaunchKernelGGL(fp4_values_kernel<f16>, grid, dim3(256), 0, s, pools, n);
  return launch_status();
}
