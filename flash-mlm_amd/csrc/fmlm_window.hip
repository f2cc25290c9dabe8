// Window attention with sinks, over contexts in 16 or 4 bits, and its gradients (bf16 / fp16).
//
// The query at position s sees key j iff j <= s + right and (j >= s - left or j < sinks); keys are
// the context rows, then the main keys.  o = softmax(scale q K^T) V over what a row sees, zero where
// that is nothing.  With P the probabilities, delta = rowsum(do o), dS = scale P (do V^T - delta):
//   dq = dS K,  dK = dS^T q,  dV = P^T do.
//
// Forward: a workgroup of four waves has BQ = 64 QB query rows of one head and walks the 64-key
// tiles that any of them sees: those of the sinks, then those of its band (WinTiles).  Only tiles
// on an edge are masked.  S^T = K Q^T and O^T = V^T P^T, so that a lane keeps one query row.
// 16-bit tiles go straight to LDS (direct loads, rows swizzled, the next tile loading during the
// math); 4-bit ones through registers, converted once a workgroup, and are 16-bit tiles from there on.
// Long key ranges of few rows are cut into parts whose records a second kernel joins.
// Backward: dq by query tiles over the tiles they see, then dK and dV by key tiles over the query
// rows that see them; no atomics.
#include "fmlm_common.h"

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "fmlm_fp4.h"

namespace fmlm {
namespace {

constexpr int kNW = 4;    // waves of a workgroup
constexpr int kBK = 64;   // keys of a tile
constexpr int kMaxParts = 32;
constexpr int kMinPartTiles = 4;  // key tiles of a part at least
constexpr int kNoLimit = 1 << 30;  // a window without a limit; positions stay below
// the running maximum moves only when a new one exceeds it by more than this (log2 units)
constexpr float kSlack = 8.0f;

struct WinArgs {
  int left, right, sinks;
  bool appended;
  int tiles;   // query tiles (dK / dV: key tiles) of a sequence
  int groups;  // (sequence, head) pairs, rounded up to a multiple of the XCDs
  int parts;   // parts of a key range at most
  int rec_rows;  // rows of a part's record
  const uint8_t* k_scales;
  const uint8_t* v_scales;
  float* records;
};

// ---- a sequence of the call: its tokens, its keys, the position of its first token
struct WinSeq {
  int b, h, q0, len;
  int ctx, total;  // context keys, all keys
  int first;       // position of token 0
};
FMLM_DEV WinSeq win_seq(const fmlm_attn_params& p, const WinArgs& a, int b, int h) {
  const SeqInfo si = seq_info(p, b);
  WinSeq s;
  s.b = b;
  s.h = h;
  s.q0 = si.q0;
  s.len = si.q0 >= 0 ? si.len : 0;  // (offsets that no call has)
  s.ctx = si.ctx;
  s.total = si.ctx + (a.appended ? 0 : s.len);
  s.first = a.appended ? si.ctx - s.len : si.ctx;
  return s;
}

// ---- the key tiles that the rows at positions [p0, p1] see: tiles [0, sink) and then [lo, ...),
// n in all; tile t < nt0 is context keys 64 t.., the others main keys 64 (t - nt0)..
struct WinTiles {
  int sink, lo, n, nt0;
  FMLM_DEV int tile(int v) const { return v < sink ? v : lo + (v - sink); }
};
FMLM_DEV WinTiles win_tiles(const WinArgs& a, const WinSeq& s, int p0, int p1) {
  WinTiles w;
  w.nt0 = (s.ctx + kBK - 1) / kBK;
  auto tile_of = [&](int key) { return key < s.ctx ? key / kBK : w.nt0 + (key - s.ctx) / kBK; };
  const int hi = min(s.total, p1 + a.right + 1), lo = max(0, p0 - a.left);
  w.sink = w.lo = w.n = 0;
  if (hi <= 0) return w;
  const int end = tile_of(hi - 1) + 1;  // tiles below are needed at most
  w.sink = a.sinks > 0 ? tile_of(min(a.sinks, hi) - 1) + 1 : 0;
  w.lo = lo < hi ? tile_of(lo) : end;
  if (w.sink >= w.lo) w.sink = w.lo = 0;  // they meet: one run
  w.n = w.sink + (end - w.lo);
  return w;
}
// parts that n tiles are cut into
FMLM_DEV int win_parts(int n, int parts) { return max(1, min(parts, n / kMinPartTiles)); }

// the work of a workgroup: part, (sequence, head) group, tile; groups vary fastest and keep to one
// XCD (workgroup w runs on XCD w % 8), so that neighbouring tiles share its L2
FMLM_DEV void win_unit(const WinArgs& a, int parts, int& g, int& part, int& tile) {
  const uint32_t w = blockIdx.x, r = w / (uint32_t)a.groups;
  g = (int)(w - r * (uint32_t)a.groups);
  tile = (int)(r / (uint32_t)parts);
  part = (int)(r - (uint32_t)tile * (uint32_t)parts);
}

// ---- a 64-row (or 32-row) tile of D 16-bit elements in LDS, 16-byte chunks swizzled by kv_swz
template <typename T, int D>
struct WTile {
  typedef typename Mfma<T>::v8 v8;
  static constexpr int ROWB = D * 2;
  static constexpr int CPR = D / 8;
  static constexpr int RPI = 64 / CPR;  // rows of a wave-wide direct load
  int koff[4], voff[8];
  FMLM_DEV WTile(int l16, int g) {
    const int ksw = kv_swz<D>(l16), vr = 4 * g + (l16 >> 2), vsw = kv_swz<D>(vr), x = (l16 & 3) >> 1;
#pragma unroll
    for (int b = 0; b < 4; ++b) koff[b] = l16 * ROWB + 16 * ((4 * b + g) ^ ksw);
#pragma unroll
    for (int b = 0; b < 8; ++b) voff[b] = vr * ROWB + 16 * ((2 * b + x) ^ vsw) + 8 * (l16 & 1);
  }
  // A operand: rows 16 rb + l16, columns 32 kc + 8 g ..
  FMLM_DEV v8 row(const char* tile, int rb, int kc) const {
    return *(const v8*)(tile + rb * 16 * ROWB + 256 * (kc / 4) + koff[kc % 4]);
  }
  // A operand of the transpose: column 16 db + l16, rows 32 ks + {4 g + e, 16 + 4 g + e}
  FMLM_DEV v8 col(const char* tile, int ks, int db) const {
    const char* a = tile + ks * 32 * ROWB + 256 * (db / 8) + voff[db % 8];
    const s16x4 lo = lds_read_tr16(a), hi = lds_read_tr16(a + 16 * ROWB);
    return __builtin_bit_cast(v8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  // starts the loads of ROWS rows from src at `pitch` bytes; rows past `last` repeat it
  template <int ROWS>
  static FMLM_DEV void load(const char* src, uint32_t pitch, int last, uint32_t lds, int wave, int lane) {
    src = uniform_ptr(src);
    pitch = __builtin_amdgcn_readfirstlane(pitch);
#pragma unroll
    for (int j = 0; j < ROWS / (RPI * kNW); ++j) {
      const int i = wave + j * kNW, row = i * RPI + lane / CPR;
      dma16_sbase(src, (uint32_t)min(row, last) * pitch + 16u * (uint32_t)((lane % CPR) ^ kv_swz<D>(row)),
                  __builtin_amdgcn_readfirstlane(lds + i * 1024));
    }
  }
};

FMLM_DEV int64_t row_at(int layout, int b, int h, int q0, int pos, int64_t sb, int64_t sh, int64_t sn) {
  return layout == FMLM_LAYOUT_PACKED ? (int64_t)h * sh + (int64_t)(q0 + pos) * sn
                                      : (int64_t)b * sb + (int64_t)h * sh + (int64_t)pos * sn;
}

// 8 elements of a row of 16-bit values, zeros where it is none
template <typename T>
FMLM_DEV typename Mfma<T>::v8 ld_frag(const void* base, int64_t elem, bool ok) {
  u32x4 r = u32x4{0u, 0u, 0u, 0u};
  if (ok) r = *(const u32x4*)((const char*)base + elem * 2);
  return __builtin_bit_cast(typename Mfma<T>::v8, r);
}

template <typename T>
FMLM_DEV uint32_t pack2(float x, float y) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x, y}, typename Pair<T>::type));
}

template <int D>
struct FwdCfg {
  static constexpr int TILEB = kBK * D * 2;
  static constexpr int LDS = 4 * TILEB;  // two K and two V tiles
  static constexpr int WPS = D <= 128 ? 2 : 1;
  static constexpr int KC = D / 32, NDB = D / 16;
};

// ---------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------
template <typename T, int D, int QB, bool FP4>
__global__ __launch_bounds__(kNW * 64, FwdCfg<D>::WPS) void window_fwd_kernel(const fmlm_attn_params p, const WinArgs a) {
  typedef FwdCfg<D> C;
  typedef typename Mfma<T>::v8 v8;
  constexpr int BQ = kNW * QB * 16;
  extern __shared__ __align__(16) char smem[];
  auto kbuf = [&](int i) { return smem + i * C::TILEB; };
  auto vbuf = [&](int i) { return smem + (2 + i) * C::TILEB; };

  int g, part, tile;
  win_unit(a, a.parts, g, part, tile);
  if (g >= p.B * p.H) return;
  tile = a.tiles - 1 - tile;  // the last rows see the most
  const WinSeq s = win_seq(p, a, g / p.H, g % p.H);
  const int row0 = tile * BQ, rows = min(BQ, s.len - row0);
  if (rows <= 0) return;
  const WinTiles wt = win_tiles(a, s, s.first + row0, s.first + row0 + rows - 1);
  const int parts = win_parts(wt.n, a.parts);
  if (part >= parts) return;
  const int vb = (int)((int64_t)wt.n * part / parts), ve = (int)((int64_t)wt.n * (part + 1) / parts);

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, gq = lane >> 4;
  const WTile<T, D> tr(l16, gq);
  const bool active = wave * QB * 16 < rows;
  // scores in log2 units are c times the products; a negative scale goes into q's sign
  const uint32_t qsign = p.scale < 0.f ? 0x80008000u : 0u;
  const float c = fmaxf(fabsf(p.scale) * kLog2e, 1e-30f);

  v8 qf[QB][C::KC];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int row = (wave * QB + qb) * 16 + l16;
    const int64_t off = row_at(p.q_layout, s.b, s.h, s.q0, row0 + row, p.q_sb, p.q_sh, p.q_sn);
#pragma unroll
    for (int kc = 0; kc < C::KC; ++kc) {
      const u32x4 r = __builtin_bit_cast(u32x4, ld_frag<T>(p.q, off + kc * 32 + gq * 8, row < rows));
      qf[qb][kc] = __builtin_bit_cast(v8, r ^ qsign);
    }
  }

  // ---- loads
  const int cb = ctx_batch_of(p, s.b);
  int ctx0 = 0, ctx1;
  ctx_range(p, cb, ctx0, ctx1);
  const int32_t* const pages = p.ctx_block_table ? p.ctx_block_table + (int64_t)cb * p.ctx_pages_per_batch : nullptr;
  auto keys_in = [&](int t) { return min(kBK, t < wt.nt0 ? s.ctx - t * kBK : s.total - s.ctx - (t - wt.nt0) * kBK); };
  // context tile t's first row, in elements of a pool or a packed context
  auto ctx_elem = [&](int t) {
    if (!pages) return (int64_t)s.h * p.c_sh + (int64_t)(ctx0 + t * kBK) * p.c_sn;
    const int pg = min(max(ldc(pages, t), 0), max(p.ctx_rows - 1, 0));
    return (int64_t)s.h * p.c_sh + (int64_t)pg * p.ctx_page_stride;
  };
  // a 4-bit tile: a quarter of a row each of 256 threads, D / 8 bytes
  constexpr int CW = FP4 ? D / 32 : 1;  // dwords of codes
  constexpr int CS = FP4 && D == 256 ? 2 : 1;  // scales
  uint32_t kcode[CW], vcode[CW], ksc[CS], vsc[CS];
  auto load_codes = [&](const void* codes, const uint8_t* scales, int64_t e, uint32_t (&w)[CW], uint32_t (&sc)[CS]) {
    const char* src = (const char*)codes + e / 2;
    if constexpr (CW == 1) w[0] = *(const uint32_t*)src;
    else if constexpr (CW == 2) { const u32x2 x = *(const u32x2*)src; w[0] = x[0]; w[1] = x[1]; }
    else
#pragma unroll
      for (int i = 0; i < CW; i += 4) {
        const u32x4 x = *(const u32x4*)(src + 4 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[i + j] = x[j];
      }
#pragma unroll
    for (int i = 0; i < CS; ++i) sc[i] = scales[e / kFp4Block + i];
  };
  auto issue = [&](int v) {
    const int t = wt.tile(v), buf = (v - vb) & 1, last = keys_in(t) - 1;
    if (t < wt.nt0) {
      const int64_t e = ctx_elem(t);
      if constexpr (FP4) {
        const int64_t at = e + (int64_t)min(tid >> 2, last) * D + (tid & 3) * (D / 4);
        load_codes(p.k_ctx, a.k_scales, at, kcode, ksc);
        load_codes(p.v_ctx, a.v_scales, at, vcode, vsc);
      } else {
        WTile<T, D>::template load<kBK>((const char*)p.k_ctx + e * 2, (uint32_t)p.c_sn * 2u, last, lds_addr(kbuf(buf)), wave, lane);
        WTile<T, D>::template load<kBK>((const char*)p.v_ctx + e * 2, (uint32_t)p.c_sn * 2u, last, lds_addr(vbuf(buf)), wave, lane);
      }
    } else {
      const int j = (t - wt.nt0) * kBK;
      WTile<T, D>::template load<kBK>((const char*)p.k + row_at(p.kv_layout, s.b, s.h, s.q0, j, p.k_sb, p.k_sh, p.k_sn) * 2,
                                      (uint32_t)p.k_sn * 2u, last, lds_addr(kbuf(buf)), wave, lane);
      WTile<T, D>::template load<kBK>((const char*)p.v + row_at(p.kv_layout, s.b, s.h, s.q0, j, p.v_sb, p.v_sh, p.v_sn) * 2,
                                      (uint32_t)p.v_sn * 2u, last, lds_addr(vbuf(buf)), wave, lane);
    }
  };
  // the loaded codes as a 16-bit tile
  auto put_codes = [&](char* tile, const uint32_t (&w)[CW], const uint32_t (&sc)[CS]) {
    const int row = tid >> 2;
#pragma unroll
    for (int i = 0; i < CW; ++i) {
      const int chunk = (tid & 3) * CW + i;
      *(u32x4*)(tile + row * (D * 2) + 16 * (chunk ^ kv_swz<D>(row))) = fp4_oct<T>(w[i], fp4_scale(sc[i / 4 % CS]));
    }
  };

  f32x4 o[C::NDB][QB], lsum[QB];
  float m[QB];
  v8 ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) ones[e] = (T)1.0f;

  // Values that are not finite in keys that a row does not see would reach it as 0 inf.  That is
  // looked for in the result; if it is there, the tiles on an edge are added key by key in a
  // second pass.
  for (bool careful = false;; careful = true) {
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      m[qb] = -INFINITY;
      lsum[qb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int db = 0; db < C::NDB; ++db) o[db][qb] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (vb < ve) issue(vb);
    for (int v = vb; v < ve; ++v) {
      const int t = wt.tile(v), buf = (v - vb) & 1, nk = keys_in(t);
      if (FP4 && t < wt.nt0) {  // (its buffer was last read two tiles ago)
        put_codes(kbuf(buf), kcode, ksc);
        put_codes(vbuf(buf), vcode, vsc);
      }
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
      if (v + 1 < ve) issue(v + 1);
      if (!active) continue;
      const char *kt = kbuf(buf), *vt = vbuf(buf);
      f32x4 sc[4][QB];
#pragma unroll
      for (int kc = 0; kc < C::KC; ++kc)
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
          const v8 x = tr.row(kt, kb, kc);
#pragma unroll
          for (int qb = 0; qb < QB; ++qb)
            sc[kb][qb] = Mfma<T>::run(x, qf[qb][kc], kc == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sc[kb][qb]);
        }
      // the tile's keys are at positions from kp on; the wave's rows at [w0, w1]
      const int kp = t < wt.nt0 ? t * kBK : s.ctx + (t - wt.nt0) * kBK;
      const int w0 = s.first + row0 + wave * QB * 16, w1 = min(w0 + QB * 16, s.first + row0 + rows) - 1;
      const bool edge = nk < kBK || kp + kBK - 1 > w0 + a.right || (kp < w1 - a.left && kp + kBK > a.sinks);
      if (edge) {
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          const int pos = w0 + qb * 16 + l16, k0 = kp + 4 * gq;  // element (kb, r) is key k0 + 16 kb + r
          const int top = min(pos + a.right - k0, nk - 1 - 4 * gq), low = pos - a.left - k0, snk = a.sinks - k0;
#pragma unroll
          for (int kb = 0; kb < 4; ++kb)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int j = kb * 16 + r;
              if (!(j <= top && (j >= low || j < snk))) sc[kb][qb][r] = -INFINITY;
            }
        }
      }
      float mx[QB];
      bool grow = false;
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        float x = vmax(vmax(sc[0][qb][0], sc[0][qb][1]), vmax(sc[0][qb][2], sc[0][qb][3]));
#pragma unroll
        for (int kb = 1; kb < 4; ++kb)
          x = vmax(vmax(x, vmax(sc[kb][qb][0], sc[kb][qb][1])), vmax(sc[kb][qb][2], sc[kb][qb][3]));
        mx[qb] = lane_max_xor16_32(x) * c;
        grow = grow || mx[qb] > m[qb] + kSlack;
      }
      if (__builtin_amdgcn_ballot_w64(grow)) {
        asm volatile("");  // (a real branch)
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          const float mn = mx[qb] > m[qb] + kSlack ? mx[qb] : m[qb];
          const float alpha = mn == -INFINITY ? 1.f : fast_exp2(m[qb] - mn);
          m[qb] = mn;
          lsum[qb] *= alpha;
#pragma unroll
          for (int db = 0; db < C::NDB; ++db) o[db][qb] *= alpha;
        }
      }
      u32x4 pf[2][QB];
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        const float ref = m[qb] == -INFINITY ? 0.f : m[qb];  // (no key yet: every score is -inf)
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
#pragma unroll
          for (int r = 0; r < 4; r += 2)
            pf[kb >> 1][qb][(kb & 1) * 2 + r / 2] = pack2<T>(fast_exp2(fmaf(sc[kb][qb][r], c, -ref)),
                                                             fast_exp2(fmaf(sc[kb][qb][r + 1], c, -ref)));
      }
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) lsum[qb] = Mfma<T>::run(ones, __builtin_bit_cast(v8, pf[ks][qb]), lsum[qb]);
      if (careful && edge) {
        // key j = 16 kb + 4 x + r of the tile: its weight is in lane l16 + 16 x
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int kb = 0; kb < 4; ++kb)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int j = kb * 16 + 4 * x + r;
#pragma unroll
              for (int qb = 0; qb < QB; ++qb) {
                const uint32_t pw = (uint32_t)__shfl((int)pf[kb >> 1][qb][(kb & 1) * 2 + r / 2], l16 + 16 * x);
                const float wgt = (float)__builtin_bit_cast(T, (uint16_t)(r & 1 ? pw >> 16 : pw));
                if (wgt != 0.f) {
#pragma unroll
                  for (int db = 0; db < C::NDB; ++db) {
                    const int chunk = 2 * db + (gq >> 1);
                    const T* val = (const T*)(vt + j * (D * 2) + 16 * (chunk ^ kv_swz<D>(j)) + 8 * (gq & 1));
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[db][qb][e] = fmaf(wgt, (float)val[e], o[db][qb][e]);
                  }
                }
              }
            }
      } else {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int db = 0; db < C::NDB; ++db) {
            const v8 x = tr.col(vt, ks, db);
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) o[db][qb] = Mfma<T>::run(x, __builtin_bit_cast(v8, pf[ks][qb]), o[db][qb]);
          }
      }
    }
    if (careful) break;
    float bad = 0.f;
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
#pragma unroll
      for (int db = 0; db < C::NDB; ++db)
#pragma unroll
        for (int r = 0; r < 4; ++r) bad = fmaf(o[db][qb][r], 0.f, bad);
    if (!__syncthreads_or(bad != bad)) break;  // (and every wave is done with the tiles)
  }

  if (!active) return;
  if (parts > 1) {  // this part's record: O, then m and l of each row
    const int64_t unit = ((int64_t)(a.tiles - 1 - tile) * a.groups + g) * a.parts + part;
    float* const rec = a.records + unit * a.rec_rows * (D + 4);
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const int row = (wave * QB + qb) * 16 + l16;
      if (row >= rows) continue;
#pragma unroll
      for (int db = 0; db < C::NDB; ++db) *(f32x4*)(rec + (int64_t)row * D + db * 16 + gq * 4) = o[db][qb];
      if (gq == 0) {
        rec[(int64_t)a.rec_rows * D + 2 * row] = m[qb];
        rec[(int64_t)a.rec_rows * D + 2 * row + 1] = lsum[qb][0];
      }
    }
    return;
  }
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int row = (wave * QB + qb) * 16 + l16;
    if (row >= rows) continue;
    const float l = lsum[qb][0], inv = l > 0.f || l != l ? 1.f / l : 0.f;
    if (p.lse && gq == 0)
      p.lse[(int64_t)s.h * p.total_q + s.q0 + row0 + row] = l > 0.f ? m[qb] + __log2f(l) : l != l ? l : INFINITY;
    const int64_t off = row_at(p.o_layout, s.b, s.h, s.q0, row0 + row, p.o_sb, p.o_sh, p.o_sn);
#pragma unroll
    for (int db = 0; db < C::NDB; ++db) {
      const f32x4 x = o[db][qb] * inv;
      *(u32x2*)((char*)p.o + (off + db * 16 + gq * 4) * 2) = u32x2{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
    }
  }
}

// ---------------------------------------------------------------------------
// The parts' records joined: 8 columns of a row a thread
// ---------------------------------------------------------------------------
template <typename T, int D>
__global__ __launch_bounds__(256) void window_merge_kernel(const fmlm_attn_params p, const WinArgs a, int bq) {
  constexpr int CPR = D / 8;
  int g, part, tile;
  win_unit(a, 1, g, part, tile);
  if (g >= p.B * p.H) return;
  tile = a.tiles - 1 - tile;
  const WinSeq s = win_seq(p, a, g / p.H, g % p.H);
  const int row0 = tile * bq, rows = min(bq, s.len - row0);
  if (rows <= 0) return;
  const int parts = win_parts(win_tiles(a, s, s.first + row0, s.first + row0 + rows - 1).n, a.parts);
  if (parts <= 1) return;
  const int64_t unit = ((int64_t)(a.tiles - 1 - tile) * a.groups + g) * a.parts, pitch = (int64_t)a.rec_rows * (D + 4);
  const float* const rec = a.records + unit * pitch;
  for (int i = threadIdx.x; i < rows * CPR; i += 256) {
    const int row = i / CPR, d = (i % CPR) * 8;
    const float* const st = rec + (int64_t)a.rec_rows * D + 2 * row;
    float top = -INFINITY;
    for (int k = 0; k < parts; ++k) top = vmax(top, st[k * pitch]);
    const float ref = top == -INFINITY ? 0.f : top;
    float l = 0.f;
    f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f}, y = x;
#pragma unroll 4
    for (int k = 0; k < parts; ++k) {
      const float w = fast_exp2(st[k * pitch] - ref);
      const f32x4* src = (const f32x4*)(rec + k * pitch + (int64_t)row * D + d);
      l = fmaf(w, st[k * pitch + 1], l);
      x += src[0] * w;
      y += src[1] * w;
    }
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    x *= inv;
    y *= inv;
    const int64_t off = row_at(p.o_layout, s.b, s.h, s.q0, row0 + row, p.o_sb, p.o_sh, p.o_sn);
    *(u32x4*)((char*)p.o + (off + d) * 2) =
        u32x4{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3])};
  }
}

// ---------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------
template <int D>
struct BwdCfg {
  static constexpr int QB = D == 128 ? 2 : 1;   // dq: 16-row blocks of a wave
  static constexpr int BQ = kNW * QB * 16;
  static constexpr int QS = D == 256 ? 32 : 64;  // dK / dV: query rows of a step
  static constexpr int TILEB = kBK * D * 2;
  static constexpr int DQ_LDS = 4 * TILEB;
  static constexpr int STEPB = QS * D * 2;
  static constexpr int SB = 2 * STEPB + 2 * QS * 4;  // a step: q rows, do rows, lse, delta
  static constexpr int DKV_LDS = 2 * SB;
  static constexpr int WPS = D <= 128 ? 2 : 1;
  static constexpr int KC = D / 32, NDB = D / 16;
};

template <typename T>
FMLM_DEV void zero_row4(void* base, int64_t elem) {
  *(u32x2*)((char*)base + elem * 2) = u32x2{0u, 0u};
}

template <typename T, int D>
__global__ __launch_bounds__(kNW * 64, BwdCfg<D>::WPS) void window_dq_kernel(const fmlm_attn_params p, const WinArgs a,
                                                                             const fmlm_attn_grads gr) {
  typedef BwdCfg<D> C;
  typedef typename Mfma<T>::v8 v8;
  constexpr int QB = C::QB;
  extern __shared__ __align__(16) char smem[];
  auto kbuf = [&](int i) { return smem + i * C::TILEB; };
  auto vbuf = [&](int i) { return smem + (2 + i) * C::TILEB; };
  int g, part, tile;
  win_unit(a, 1, g, part, tile);
  if (g >= p.B * p.H) return;
  tile = a.tiles - 1 - tile;
  const WinSeq s = win_seq(p, a, g / p.H, g % p.H);
  const int row0 = tile * C::BQ, rows = min(C::BQ, s.len - row0);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, gq = lane >> 4;
  if (p.q_layout == FMLM_LAYOUT_PADDED) {  // padding rows of dq
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const int row = row0 + (wave * QB + qb) * 16 + l16;
      if (row < s.len || row >= p.N) continue;
      const int64_t off = row_at(p.q_layout, s.b, s.h, s.q0, row, gr.dq_sb, gr.dq_sh, gr.dq_sn);
#pragma unroll
      for (int db = 0; db < C::NDB; ++db) zero_row4<T>(gr.dq, off + db * 16 + gq * 4);
    }
  }
  if (rows <= 0) return;
  const WinTiles wt = win_tiles(a, s, row0, row0 + rows - 1);
  const WTile<T, D> tr(l16, gq);
  const bool active = wave * QB * 16 < rows;
  const float c = p.scale * kLog2e;

  v8 qf[QB][C::KC], df[QB][C::KC];
  float delta[QB], lse[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int row = (wave * QB + qb) * 16 + l16;
    const bool ok = row < rows;
    const int64_t qo = row_at(p.q_layout, s.b, s.h, s.q0, row0 + row, p.q_sb, p.q_sh, p.q_sn);
    const int64_t oo = row_at(p.o_layout, s.b, s.h, s.q0, row0 + row, p.o_sb, p.o_sh, p.o_sn);
    const int64_t po = row_at(p.o_layout, s.b, s.h, s.q0, row0 + row, gr.do_sb, gr.do_sh, gr.do_sn);
    float sum = 0.f;
#pragma unroll
    for (int kc = 0; kc < C::KC; ++kc) {
      const int col = kc * 32 + gq * 8;
      qf[qb][kc] = ld_frag<T>(p.q, qo + col, ok);
      df[qb][kc] = ld_frag<T>(gr.dout, po + col, ok);
      const v8 ov = ld_frag<T>(p.o, oo + col, ok);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf((float)df[qb][kc][e], (float)ov[e], sum);
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    delta[qb] = sum;
    const int64_t at = (int64_t)s.h * p.total_q + s.q0 + row0 + row;
    lse[qb] = ok ? p.lse[at] : INFINITY;
    if (ok && gq == 0) ((float*)gr.workspace)[at] = sum;  // for the dK / dV kernel
  }
  auto keys_in = [&](int t) { return min(kBK, s.total - t * kBK); };
  auto issue = [&](int v) {
    const int t = wt.tile(v), buf = v & 1, last = keys_in(t) - 1;
    WTile<T, D>::template load<kBK>((const char*)p.k + row_at(p.kv_layout, s.b, s.h, s.q0, t * kBK, p.k_sb, p.k_sh, p.k_sn) * 2,
                                    (uint32_t)p.k_sn * 2u, last, lds_addr(kbuf(buf)), wave, lane);
    WTile<T, D>::template load<kBK>((const char*)p.v + row_at(p.kv_layout, s.b, s.h, s.q0, t * kBK, p.v_sb, p.v_sh, p.v_sn) * 2,
                                    (uint32_t)p.v_sn * 2u, last, lds_addr(vbuf(buf)), wave, lane);
  };
  f32x4 dq[C::NDB][QB];
#pragma unroll
  for (int db = 0; db < C::NDB; ++db)
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) dq[db][qb] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (wt.n > 0) issue(0);
  for (int v = 0; v < wt.n; ++v) {
    const int t = wt.tile(v), buf = v & 1, nk = keys_in(t);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (v + 1 < wt.n) issue(v + 1);
    if (!active) continue;
    const char *kt = kbuf(buf), *vt = vbuf(buf);
    f32x4 sc[4][QB], dp[4][QB];
#pragma unroll
    for (int kc = 0; kc < C::KC; ++kc)
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) {
        const v8 x = tr.row(kt, kb, kc), y = tr.row(vt, kb, kc);
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          sc[kb][qb] = Mfma<T>::run(x, qf[qb][kc], kc == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sc[kb][qb]);
          dp[kb][qb] = Mfma<T>::run(y, df[qb][kc],
                                    kc == 0 ? f32x4{-delta[qb], -delta[qb], -delta[qb], -delta[qb]} : dp[kb][qb]);
        }
      }
    const int kp = t * kBK, w0 = row0 + wave * QB * 16, w1 = min(w0 + QB * 16, row0 + rows) - 1;
    const bool edge = nk < kBK || kp + kBK - 1 > w0 + a.right || (kp < w1 - a.left && kp + kBK > a.sinks);
    u32x4 ds[2][QB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) dp[kb][qb][r] *= fast_exp2(fmaf(sc[kb][qb][r], c, -lse[qb]));
      if (edge) {
        const int pos = w0 + qb * 16 + l16, k0 = kp + 4 * gq;
        const int top = min(pos + a.right - k0, nk - 1 - 4 * gq), low = pos - a.left - k0, snk = a.sinks - k0;
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = kb * 16 + r;
            if (!(j <= top && (j >= low || j < snk))) dp[kb][qb][r] = 0.f;
          }
      }
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int r = 0; r < 4; r += 2)
          ds[kb >> 1][qb][(kb & 1) * 2 + r / 2] = pack2<T>(dp[kb][qb][r], dp[kb][qb][r + 1]);
    }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int db = 0; db < C::NDB; ++db) {
        const v8 x = tr.col(kt, ks, db);
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) dq[db][qb] = Mfma<T>::run(x, __builtin_bit_cast(v8, ds[ks][qb]), dq[db][qb]);
      }
  }
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int row = (wave * QB + qb) * 16 + l16;
    if (row >= rows) continue;
    const int64_t off = row_at(p.q_layout, s.b, s.h, s.q0, row0 + row, gr.dq_sb, gr.dq_sh, gr.dq_sn);
#pragma unroll
    for (int db = 0; db < C::NDB; ++db) {
      const f32x4 x = dq[db][qb] * p.scale;
      *(u32x2*)((char*)gr.dq + (off + db * 16 + gq * 4) * 2) = u32x2{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
    }
  }
}

template <typename T, int D>
__global__ __launch_bounds__(kNW * 64, BwdCfg<D>::WPS) void window_dkv_kernel(const fmlm_attn_params p, const WinArgs a,
                                                                              const fmlm_attn_grads gr) {
  typedef BwdCfg<D> C;
  typedef typename Mfma<T>::v8 v8;
  constexpr int QS = C::QS, NRB = QS / 16;
  extern __shared__ __align__(16) char smem[];
  auto qbuf = [&](int i) { return smem + i * C::SB; };
  auto obuf = [&](int i) { return smem + i * C::SB + C::STEPB; };
  auto stat = [&](int i) { return (float*)(smem + i * C::SB + 2 * C::STEPB); };
  int g, part, tile;
  win_unit(a, 1, g, part, tile);
  if (g >= p.B * p.H) return;
  const WinSeq s = win_seq(p, a, g / p.H, g % p.H);
  const int j0 = tile * kBK;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, gq = lane >> 4;
  const int key = j0 + wave * 16 + l16;
  const bool kok = key < s.len;
  const int64_t dko = row_at(p.kv_layout, s.b, s.h, s.q0, key, gr.dk_sb, gr.dk_sh, gr.dk_sn) + gq * 4;
  const int64_t dvo = row_at(p.kv_layout, s.b, s.h, s.q0, key, gr.dv_sb, gr.dv_sh, gr.dv_sn) + gq * 4;
  if (p.kv_layout == FMLM_LAYOUT_PADDED && !kok && key < p.N) {  // padding rows of dk and dv
#pragma unroll
    for (int db = 0; db < C::NDB; ++db) {
      zero_row4<T>(gr.dk, dko + db * 16);
      zero_row4<T>(gr.dv, dvo + db * 16);
    }
  }
  if (j0 >= s.len) return;
  const WTile<T, D> tr(l16, gq);
  const float c = p.scale * kLog2e;
  v8 kf[C::KC], vf[C::KC];
  {
    const int64_t ko = row_at(p.kv_layout, s.b, s.h, s.q0, key, p.k_sb, p.k_sh, p.k_sn);
    const int64_t vo = row_at(p.kv_layout, s.b, s.h, s.q0, key, p.v_sb, p.v_sh, p.v_sn);
#pragma unroll
    for (int kc = 0; kc < C::KC; ++kc) {
      kf[kc] = ld_frag<T>(p.k, ko + kc * 32 + gq * 8, kok);
      vf[kc] = ld_frag<T>(p.v, vo + kc * 32 + gq * 8, kok);
    }
  }
  // the rows that see any of these keys
  const int last_key = min(j0 + kBK, s.len) - 1;
  const int r_lo = max(0, j0 - a.right), r_hi = j0 < a.sinks ? s.len - 1 : min(s.len - 1, last_key + a.left);
  const int steps = r_hi >= r_lo ? (r_hi - r_lo) / QS + 1 : 0;
  const float* const st_delta = (const float*)gr.workspace;
  float lreg = 0.f, dreg = 0.f;
  auto issue = [&](int i) {
    const int p0 = r_lo + i * QS, last = min(QS, r_hi + 1 - p0) - 1;
    if (tid < QS) {  // rows past the last: lse inf, so P = 0
      const int64_t at = (int64_t)s.h * p.total_q + s.q0 + p0 + tid;
      lreg = tid <= last ? p.lse[at] : INFINITY;
      dreg = tid <= last ? st_delta[at] : 0.f;
    }
    WTile<T, D>::template load<QS>((const char*)p.q + row_at(p.q_layout, s.b, s.h, s.q0, p0, p.q_sb, p.q_sh, p.q_sn) * 2,
                                   (uint32_t)p.q_sn * 2u, last, lds_addr(qbuf(i & 1)), wave, lane);
    WTile<T, D>::template load<QS>((const char*)gr.dout + row_at(p.o_layout, s.b, s.h, s.q0, p0, gr.do_sb, gr.do_sh, gr.do_sn) * 2,
                                   (uint32_t)gr.do_sn * 2u, last, lds_addr(obuf(i & 1)), wave, lane);
  };
  f32x4 dk[C::NDB], dv[C::NDB];
#pragma unroll
  for (int db = 0; db < C::NDB; ++db) dk[db] = dv[db] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (steps > 0) issue(0);
  for (int i = 0; i < steps; ++i) {
    const int p0 = r_lo + i * QS;
    const char *qt = qbuf(i & 1), *ot = obuf(i & 1);
    float* const ls = stat(i & 1);
    if (tid < QS) {
      ls[tid] = lreg;
      ls[QS + tid] = dreg;
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (i + 1 < steps) issue(i + 1);
    const int k0 = j0 + wave * 16, k1 = k0 + 15;
    const bool edge = k1 >= s.len || k1 > p0 + a.right || (k0 < p0 + QS - 1 - a.left && k1 >= a.sinks);
    // rows pos with lo <= pos <= hi see the lane's key
    const int lo = key - a.right - p0, hi = !kok ? -1 : key < a.sinks ? QS : key + a.left - p0;
    u32x4 pw[NRB / 2], dw[NRB / 2];
#pragma unroll
    for (int rb = 0; rb < NRB; ++rb) {
      f32x4 sc, dp;
#pragma unroll
      for (int kc = 0; kc < C::KC; ++kc) {
        sc = Mfma<T>::run(tr.row(qt, rb, kc), kf[kc], kc == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sc);
        dp = Mfma<T>::run(tr.row(ot, rb, kc), vf[kc], kc == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : dp);
      }
      const f32x4 L = *(const f32x4*)(ls + rb * 16 + gq * 4), Dl = *(const f32x4*)(ls + QS + rb * 16 + gq * 4);
      f32x4 pv, dsv;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        pv[r] = fast_exp2(fmaf(sc[r], c, -L[r]));
        dsv[r] = pv[r] * (dp[r] - Dl[r]);
      }
      if (edge) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int pos = rb * 16 + gq * 4 + r;
          if (!(pos >= lo && pos <= hi)) pv[r] = dsv[r] = 0.f;
        }
      }
      pw[rb >> 1][(rb & 1) * 2] = pack2<T>(pv[0], pv[1]);
      pw[rb >> 1][(rb & 1) * 2 + 1] = pack2<T>(pv[2], pv[3]);
      dw[rb >> 1][(rb & 1) * 2] = pack2<T>(dsv[0], dsv[1]);
      dw[rb >> 1][(rb & 1) * 2 + 1] = pack2<T>(dsv[2], dsv[3]);
    }
#pragma unroll
    for (int ks = 0; ks < NRB / 2; ++ks)
#pragma unroll
      for (int db = 0; db < C::NDB; ++db) {
        dv[db] = Mfma<T>::run(tr.col(ot, ks, db), __builtin_bit_cast(v8, pw[ks]), dv[db]);
        dk[db] = Mfma<T>::run(tr.col(qt, ks, db), __builtin_bit_cast(v8, dw[ks]), dk[db]);
      }
  }
  if (!kok) return;
#pragma unroll
  for (int db = 0; db < C::NDB; ++db) {
    const f32x4 x = dk[db] * p.scale, y = dv[db];
    *(u32x2*)((char*)gr.dk + (dko + db * 16) * 2) = u32x2{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
    *(u32x2*)((char*)gr.dv + (dvo + db * 16) * 2) = u32x2{pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3])};
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
// a kernel's LDS beyond 64 KB has to be allowed once a device
int allow_lds(const void* fn, int bytes) {
  if (bytes <= 65536) return 0;
  hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  return e == hipSuccess ? 0 : (int)e;
}

struct FwdLaunch {
  const void* fn;
  const void* merge;
  int bq, lds;
};
template <typename T, int D, int QB>
FwdLaunch fwd_of(bool fp4) {
  FwdLaunch f;
  f.fn = fp4 ? (const void*)window_fwd_kernel<T, D, QB, true> : (const void*)window_fwd_kernel<T, D, QB, false>;
  f.merge = (const void*)window_merge_kernel<T, D>;
  f.bq = kNW * QB * 16;
  f.lds = FwdCfg<D>::LDS;
  return f;
}
template <typename T>
FwdLaunch pick_fwd(const fmlm_attn_params& p, bool fp4) {
  const bool wide = p.N == 0 || p.N > 64;  // 128 rows share a tile's loads
  switch (p.D) {
    case 32: return wide ? fwd_of<T, 32, 2>(fp4) : fwd_of<T, 32, 1>(fp4);
    case 64: return wide ? fwd_of<T, 64, 2>(fp4) : fwd_of<T, 64, 1>(fp4);
    case 128: return wide ? fwd_of<T, 128, 2>(fp4) : fwd_of<T, 128, 1>(fp4);
    default: return fwd_of<T, 256, 1>(fp4);  // (two blocks of 16 rows spill)
  }
}
FwdLaunch pick_fwd(const fmlm_attn_params& p, bool fp4) {
  return p.dtype == FMLM_DTYPE_BF16 ? pick_fwd<bf16>(p, fp4) : pick_fwd<f16>(p, fp4);
}

bool row_ok(const void* base, int64_t sb, int64_t sh, int64_t sn) {
  return base && (uint64_t)base % 16 == 0 && sb % 8 == 0 && sh % 8 == 0 && sn % 8 == 0 && sn >= 0 && sn < (1 << 22);
}

int longest(const fmlm_attn_params& p) { return p.N > 0 && p.N < p.total_q ? p.N : p.total_q; }

int check_window(const fmlm_attn_params& p, const fmlm_window& w) {
  if (p.dtype != FMLM_DTYPE_BF16 && p.dtype != FMLM_DTYPE_F16) return FMLM_E_DTYPE;
  if (p.D != 32 && p.D != 64 && p.D != 128 && p.D != 256) return FMLM_E_HEAD_DIM;
  if (p.flags & ~FMLM_FLAG_NOSPLIT) return FMLM_E_ARG;
  if (w.flags & ~(FMLM_WINDOW_APPENDED | FMLM_WINDOW_FP4)) return FMLM_E_ARG;
  if (p.B < 0 || p.H < 0 || p.N < 0 || p.total_q < 0 || p.total_q >= kNoLimit) return FMLM_E_ARG;
  if (p.B == 0 || p.H == 0 || p.total_q == 0) return 0;
  if (!p.cu_seqlens_q || (int64_t)p.B * p.H > 0x7fffff00) return FMLM_E_ARG;
  const bool appended = w.flags & FMLM_WINDOW_APPENDED, fp4 = w.flags & FMLM_WINDOW_FP4;
  const bool ctx = p.cu_seqlens_kv || p.ctx_block_table || p.ctx_len > 0;
  if (!ctx && (appended || fp4)) return FMLM_E_ARG;
  if (ctx) {
    if (!p.cu_seqlens_kv || p.ctx_rows < 0 || p.ctx_batch < 1) return FMLM_E_ARG;
    if (!p.ctx_index && p.ctx_batch > 1 && p.ctx_batch < p.B) return FMLM_E_ARG;
    const int64_t rows = p.ctx_block_table ? (int64_t)p.ctx_pages_per_batch * FMLM_PAGE_ROWS : (int64_t)p.ctx_rows;
    if (rows + p.total_q >= kNoLimit || p.ctx_pages_per_batch < 0) return FMLM_E_ARG;
    if (rows > 0 && p.ctx_rows > 0) {
      if (!row_ok(p.k_ctx, 0, p.c_sh, p.c_sn) || !row_ok(p.v_ctx, 0, p.c_sh, p.c_sn)) return FMLM_E_ALIGN;
      if (p.ctx_block_table && p.ctx_page_stride % 8) return FMLM_E_ALIGN;
      if (fp4 && (!p.ctx_block_table || !w.k_scales || !w.v_scales || p.c_sn != p.D || p.c_sh % (16 * kFp4Block) ||
                  p.ctx_page_stride % (16 * kFp4Block)))
        return FMLM_E_ARG;
    } else if (p.ctx_block_table && rows > 0) {
      return FMLM_E_ARG;  // pages of an empty pool
    }
  }
  if (!row_ok(p.q, p.q_sb, p.q_sh, p.q_sn) || !row_ok(p.o, p.o_sb, p.o_sh, p.o_sn)) return FMLM_E_ALIGN;
  if (!appended && (!row_ok(p.k, p.k_sb, p.k_sh, p.k_sn) || !row_ok(p.v, p.v_sb, p.v_sh, p.v_sn))) return FMLM_E_ALIGN;
  return 0;
}

int limit(int x) { return x < 0 || x >= kNoLimit ? kNoLimit - 2 : x; }

WinArgs win_args(const fmlm_attn_params& p, const fmlm_window& w, int rows) {
  WinArgs a{};
  a.left = limit(w.left);
  a.right = limit(w.right);
  a.sinks = std::min(std::max(w.sinks, 0), kNoLimit - 2);
  a.appended = w.flags & FMLM_WINDOW_APPENDED;
  a.tiles = (longest(p) + rows - 1) / rows;
  a.groups = (p.B * p.H + 7) / 8 * 8;
  a.parts = 1;
  a.k_scales = w.k_scales;
  a.v_scales = w.v_scales;
  return a;
}

// parts that key ranges are cut into at most, and a record's rows
void plan_parts(const fmlm_attn_params& p, const fmlm_window& w, const FwdLaunch& f, WinArgs& a) {
  a.rec_rows = std::min(f.bq, longest(p));
  const int64_t units = (int64_t)p.B * p.H * a.tiles;
  if (p.lse || (p.flags & FMLM_FLAG_NOSPLIT) || units >= 1024) return;
  int64_t keys = longest(p);
  if (p.cu_seqlens_kv)
    keys += p.ctx_block_table ? (int64_t)p.ctx_pages_per_batch * FMLM_PAGE_ROWS
                              : std::min((int64_t)p.ctx_rows, 2 * (int64_t)p.ctx_rows / std::max(p.ctx_batch, 1));
  keys = std::min(keys, (int64_t)a.left + a.right + a.sinks + f.bq);
  const int64_t tiles = keys / kBK + 2, want = (2048 + units - 1) / units;
  a.parts = (int)std::max<int64_t>(1, std::min<int64_t>({want, tiles / kMinPartTiles, kMaxParts}));
}

int64_t record_bytes(const fmlm_attn_params& p, const WinArgs& a) {
  return a.parts > 1 ? (int64_t)a.tiles * a.groups * a.parts * a.rec_rows * (p.D + 4) * 4 : 0;
}

template <typename T, int D>
int launch_bwd(const fmlm_attn_params& p, const fmlm_window& w, const fmlm_attn_grads& g, hipStream_t s) {
  typedef BwdCfg<D> C;
  // padded gradients are written whole: tiles up to N
  WinArgs a = win_args(p, w, C::BQ), b = win_args(p, w, kBK);
  if (p.N > 0 && p.q_layout == FMLM_LAYOUT_PADDED) a.tiles = (p.N + C::BQ - 1) / C::BQ;
  if (p.N > 0 && p.kv_layout == FMLM_LAYOUT_PADDED) b.tiles = (p.N + kBK - 1) / kBK;
  if ((int64_t)a.tiles * a.groups > 0x7fffffff || (int64_t)b.tiles * b.groups > 0x7fffffff) return FMLM_E_ARG;
  const void *dq = (const void*)window_dq_kernel<T, D>, *dkv = (const void*)window_dkv_kernel<T, D>;
  int rc = allow_lds(dq, C::DQ_LDS);
  if (!rc) rc = allow_lds(dkv, C::DKV_LDS);
  if (rc) return rc;
  hipLaunchKernelGGL((window_dq_kernel<T, D>), dim3((unsigned)(a.tiles * a.groups)), dim3(kNW * 64), C::DQ_LDS, s, p, a, g);
  hipLaunchKernelGGL((window_dkv_kernel<T, D>), dim3((unsigned)(b.tiles * b.groups)), dim3(kNW * 64), C::DKV_LDS, s, p, b, g);
  return launch_status();
}
template <typename T>
int launch_bwd(const fmlm_attn_params& p, const fmlm_window& w, const fmlm_attn_grads& g, hipStream_t s) {
  switch (p.D) {
    case 32: return launch_bwd<T, 32>(p, w, g, s);
    case 64: return launch_bwd<T, 64>(p, w, g, s);
    case 128: return launch_bwd<T, 128>(p, w, g, s);
    default: return launch_bwd<T, 256>(p, w, g, s);
  }
}

}  // namespace
}  // namespace fmlm

using namespace fmlm;

extern "C" int fmlm_window_size(void) { return (int)sizeof(fmlm_window); }

extern "C" int64_t fmlm_window_workspace_bytes(const fmlm_attn_params* pp, const fmlm_window* ww) {
  if (!pp || !ww) return FMLM_E_ARG;
  const int rc = check_window(*pp, *ww);
  if (rc) return rc;
  if (pp->B == 0 || pp->H == 0 || pp->total_q == 0) return 0;
  const FwdLaunch f = pick_fwd(*pp, ww->flags & FMLM_WINDOW_FP4);
  WinArgs a = win_args(*pp, *ww, f.bq);
  plan_parts(*pp, *ww, f, a);
  return record_bytes(*pp, a);
}

extern "C" int fmlm_window_fwd(const fmlm_attn_params* pp, const fmlm_window* ww, void* stream) {
  if (!pp || !ww) return FMLM_E_ARG;
  fmlm_attn_params p = *pp;
  int rc = check_window(p, *ww);
  if (rc) return rc;
  if (p.B == 0 || p.H == 0 || p.total_q == 0) return 0;
  const FwdLaunch f = pick_fwd(p, ww->flags & FMLM_WINDOW_FP4);
  WinArgs a = win_args(p, *ww, f.bq);
  plan_parts(p, *ww, f, a);
  const int64_t need = record_bytes(p, a), blocks = (int64_t)a.tiles * a.groups * a.parts;
  if (need > 0 && (!p.workspace || p.workspace_bytes < need)) return FMLM_E_WORKSPACE;
  if (need > 0 && (uint64_t)p.workspace % 16) return FMLM_E_ALIGN;
  if (blocks > 0x7fffffff) return FMLM_E_ARG;
  a.records = (float*)p.workspace;
  p.flags = p.cu_seqlens_kv ? 0 : FMLM_FLAG_PREFILL;  // (without a context)
  rc = allow_lds(f.fn, f.lds);
  if (rc) return rc;
  hipStream_t s = (hipStream_t)stream;
  void* args[2] = {&p, &a};
  hipError_t e = hipLaunchKernel(f.fn, dim3((unsigned)blocks), dim3(kNW * 64), args, f.lds, s);
  if (e != hipSuccess) return (int)e;
  if (a.parts > 1) {
    int bq = f.bq;
    void* margs[3] = {&p, &a, &bq};
    e = hipLaunchKernel(f.merge, dim3((unsigned)(a.tiles * a.groups)), dim3(256), margs, 0, s);
    if (e != hipSuccess) return (int)e;
  }
  return launch_status();
}

extern "C" int fmlm_window_bwd(const fmlm_attn_params* pp, const fmlm_window* ww, const fmlm_attn_grads* gg,
                               void* stream) {
  if (!pp || !ww || !gg) return FMLM_E_ARG;
  fmlm_attn_params p = *pp;
  const fmlm_attn_grads& g = *gg;
  const int rc = check_window(p, *ww);
  if (rc) return rc;
  if (ww->flags || p.cu_seqlens_kv || g.dk_ctx || g.dv_ctx) return FMLM_E_ARG;
  if (p.B == 0 || p.H == 0 || p.total_q == 0) return 0;
  if (!p.lse) return FMLM_E_ARG;
  if (!row_ok(g.dout, g.do_sb, g.do_sh, g.do_sn) || !row_ok(g.dq, g.dq_sb, g.dq_sh, g.dq_sn) ||
      !row_ok(g.dk, g.dk_sb, g.dk_sh, g.dk_sn) || !row_ok(g.dv, g.dv_sb, g.dv_sh, g.dv_sn))
    return FMLM_E_ALIGN;
  if (!g.workspace || g.workspace_bytes < (int64_t)p.H * p.total_q * 4) return FMLM_E_WORKSPACE;
  p.flags = FMLM_FLAG_PREFILL;
  return p.dtype == FMLM_DTYPE_BF16 ? launch_bwd<bf16>(p, *ww, g, (hipStream_t)stream)
                                    : launch_bwd<f16>(p, *ww, g, (hipStream_t)stream);
}
