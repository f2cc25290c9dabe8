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
#include <atomic>
#include <cmath>
#include <type_traits>

#include "fmlm_fp4.h"

namespace fmlm {
namespace {

constexpr int kNW = 4;    // waves of a workgroup
constexpr int kBK = 64;   // keys of a tile; 32 at D = 256, where two workgroups of them fit a CU
constexpr int tile_keys(int D) { return D == 256 ? 32 : kBK; }
constexpr int kMaxParts = 32;
constexpr int kMinPartTiles = 4;  // key tiles of a part at least
constexpr int kFewTiles = 8;      // ... where its waves walk apart
constexpr int kFill = 512;        // workgroups: two a CU
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
  int lg;        // log2 of the keys of a tile of the records' walk
  const uint8_t* k_scales;
  const uint8_t* v_scales;
  float* records;
  void* o_low;  // what the rounding of o took away, for the backward
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
// n in all; of tiles of 2^lg keys, t < nt0 is context keys 2^lg t.., the others main keys
struct WinTiles {
  int sink, lo, n, nt0;
  FMLM_DEV int tile(int v) const { return v < sink ? v : lo + (v - sink); }
};
FMLM_DEV WinTiles win_tiles(const WinArgs& a, const WinSeq& s, int p0, int p1, int lg) {
  WinTiles w;
  w.nt0 = (s.ctx + (1 << lg) - 1) >> lg;
  auto tile_of = [&](int key) { return key < s.ctx ? key >> lg : w.nt0 + ((key - s.ctx) >> lg); };
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
// XCD (workgroup w runs on XCD w % 8), so that neighbouring tiles share its L2.  Returns whether there is any.
// (A launch has fewer than 2^32 threads in x: kGridX workgroups there, and z of them.)
constexpr uint32_t kGridX = 1u << 23;
FMLM_DEV bool win_unit(const fmlm_attn_params& p, const WinArgs& a, int parts, int& g, int& part, int& tile) {
  const uint32_t w = blockIdx.x + blockIdx.z * kGridX, r = w / (uint32_t)a.groups;
  g = (int)(w - r * (uint32_t)a.groups);
  tile = (int)(r / (uint32_t)parts);
  part = (int)(r - (uint32_t)tile * (uint32_t)parts);
  return g < p.B * p.H && tile < a.tiles;
}

// ---- which of a lane's elements are in view, as bits: element (block b, r) is bit 16 b + r, b < 4, r < 4.
// A conditional per element becomes a branch each (three compares, two saves of exec); a bit spread
// over a word and one bitwise select are two instructions and serve both edges and the sinks alike.
struct InView {
  int w[2];
  InView() = default;
  // elements [low, top], and [0, sinks) up to top
  FMLM_DEV InView(int low, int top, int sinks) {
    const uint64_t x = ~from(top + 1) & (from(low) | ~from(sinks));
    w[0] = (int)x;
    w[1] = (int)(x >> 32);
  }
  FMLM_DEV static uint64_t from(int n) { return ~0ull << min(max(n, 0), 63); }  // (bit 63 is no element)
  FMLM_DEV float pick(int b, int r, float x, float none) const {
    int keep = __builtin_amdgcn_sbfe(w[b >> 1], (b & 1) * 16 + r, 1);
    asm("" : "+v"(keep));  // (else a compare and two selects)
    return __int_as_float((__float_as_int(x) & keep) | (__float_as_int(none) & ~keep));
  }
};

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
  // the lane's offsets of a whole tile of ROWS rows at `pitch` bytes, and its loads with them
  template <int ROWS>
  static FMLM_DEV void offsets(uint32_t pitch, int wave, int lane, uint32_t (&off)[ROWS / (RPI * kNW)]) {
#pragma unroll
    for (int j = 0; j < ROWS / (RPI * kNW); ++j) {
      const int row = (wave + j * kNW) * RPI + lane / CPR;
      off[j] = (uint32_t)row * pitch + 16u * (uint32_t)((lane % CPR) ^ kv_swz<D>(row));
    }
  }
  template <int ROWS>
  static FMLM_DEV void load_at(const char* src, const uint32_t (&off)[ROWS / (RPI * kNW)], uint32_t lds, int wave) {
#pragma unroll
    for (int j = 0; j < ROWS / (RPI * kNW); ++j)
      dma16_sbase(src, off[j], __builtin_amdgcn_readfirstlane(lds + (wave + j * kNW) * 1024));
  }
  // starts the loads of ROWS rows from src at `pitch` bytes; rows past `last` repeat it
  template <int ROWS>
  static FMLM_DEV void load(const char* src, uint32_t pitch, int last, uint32_t lds, int wave, int lane) {
    src = uniform_ptr(src);
    pitch = __builtin_amdgcn_readfirstlane(pitch);
    asm volatile("" : "+v"(lane));  // (offsets of a rare tile: computed here, not kept)
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

// K tiles are double-buffered, V tiles have a third buffer where it fits beside a second workgroup
// on the CU (80 KB each): their loads then have two steps to land.
template <int D, bool FP4>
struct FwdCfg {
  static constexpr int BK = tile_keys(D), TILEB = BK * D * 2;
  static constexpr int NV = FP4 ? 2 : 3;
  static constexpr int TPR = kNW * 64 / BK;    // threads that share a 4-bit row
  static constexpr int CW = D / TPR / 8;       // dwords of codes of each
  static constexpr bool STAGE = FP4 && CW == 4;  // codes wait in LDS (else in registers)
  static constexpr int LDS = (2 + NV) * TILEB + (STAGE ? 2 * kNW * 1024 : 0);
  static constexpr int KC = D / 32, NDB = D / 16, NKB = BK / 16, NKS = BK / 32;
  static constexpr int LEAD = D <= 64 ? 2 : 3;  // LDS fragment reads in flight ahead of use
  static constexpr int NKF = KC * NKB, NVF = NKS * NDB;  // K and V fragments of a tile
};

// ---------------------------------------------------------------------------
// Forward.  Step v of the walk computes S(v + 1) beside the exponentials of P(v), then O += V(v)^T P(v)
// beside the row maxima of S(v + 1): fenced slots, each the MFMAs of one LDS fragment and a share of
// the other work, the fragment of LEAD slots later being read.  In the same step the tiles of later
// ones load: K(v + 2) into K(v)'s buffer and V(v + NV - 1) into V(v - 1)'s.  4-bit tiles are a step
// ahead of that: their codes arrive in step v and are converted, by the wave that loaded them, at
// the start of step v + 1.
//
// P goes to the input type as an operand of the matrix cores, off by half a step; l adds up the same
// rounded values (a product with ones), so that what all of a row's probabilities share cancels.  Scores, maxima,
// l and O stay in 32 bits.  The statistics for a backward (LSE) are of the sum as it is: with the rounded one
// all of a row's probabilities would be off alike there by the mean rounding of its keys, which counts where they are
// few (dv over 4 keys with a sink 1.52 times the error of its own rounding, so 1.44).
//
// Bound (times of a warm card, after 0.4 s of the same calls): fp16, 4 x 16 causal sequences of 4096 rows of 128:
// a window of 64 takes 73 us (268 MB, 73% of a large copy's rate), all keys 283 us (970 TFLOP/s, 73% of a
// large matrix product's rate).  Between them the two add up (1024 keys: 169 us; for a backward 30% of the matrix
// cores, 39% of the VALU), as workgroups read their first tiles and rows while few others compute; another order of
// the tiles, staggered starts or more fragments in flight changed nothing.  Single rows over 1024 keys of a paged
// context (64 users) are at a copy's rate.
// 4 bits: 87 us for the 44 GFLOP of four chunks of 300 to 512 rows over 2000 to 4000 keys, 21% of the matrix
// cores and 26% of the VALU (the conversions among it) at 1.2 waves a SIMD: 512 workgroups, of unequal length.
// (Pairs of figures below are of both forms side by side, some on a card that was not warm: up to 20% longer.)
// ---------------------------------------------------------------------------
template <typename T, int D, int QB, bool FP4, bool LSE>
__global__ __launch_bounds__(kNW * 64, 2) void window_fwd_kernel(const fmlm_attn_params p, const WinArgs a) {
  typedef FwdCfg<D, FP4> C;
  typedef typename Mfma<T>::v8 v8;
  constexpr int BQ = kNW * QB * 16, CW = C::CW, BK = C::BK, NKB = C::NKB, NKS = C::NKS;
  extern __shared__ __align__(16) char smem[];
  // buffers of tile v; a step takes them from its place among NU unrolled ones, as constants
  constexpr int NU = C::NV == 2 ? 2 : 6;
  auto kbuf = [&](int v) { return smem + (v & 1) * C::TILEB; };
  auto vbuf = [&](int v) { return smem + (2 + v % C::NV) * C::TILEB; };

  int g, part, tile;
  if (!win_unit(p, a, a.parts, g, part, tile)) return;
  tile = a.tiles - 1 - tile;  // the last rows see the most
  const WinSeq s = win_seq(p, a, g / p.H, g % p.H);
  const int row0 = tile * BQ, rows = min(BQ, s.len - row0);
  if (rows <= 0) return;
  const WinTiles wt = win_tiles(a, s, s.first + row0, s.first + row0 + rows - 1, BK == 64 ? 6 : 5);
  const int parts = win_parts(wt.n, a.parts);
  if (part >= parts) return;
  const int vb = (int)((int64_t)wt.n * part / parts), n = (int)((int64_t)wt.n * (part + 1) / parts) - vb;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, gq = lane >> 4;
  const WTile<T, D> tr(l16, gq);
  const bool active = wave * QB * 16 < rows;
  // scores in log2 units are c times the products; a negative scale goes into q's sign
  const uint32_t qsign = p.scale < 0.f ? 0x80008000u : 0u;
  const float c = fmaxf(fabsf(p.scale) * kLog2e, 1e-30f);

  // ---- loads of tile v of this part: t(v) of the walk
  auto tile_at = [&](int v) { return __builtin_amdgcn_readfirstlane(wt.tile(vb + v)); };
  const int cb = ctx_batch_of(p, s.b);
  int ctx0 = 0, ctx1;
  ctx_range(p, cb, ctx0, ctx1);
  const int32_t* const pages = p.ctx_block_table ? p.ctx_block_table + (int64_t)cb * p.ctx_pages_per_batch : nullptr;
  auto keys_in = [&](int t) { return min(BK, t < wt.nt0 ? s.ctx - t * BK : s.total - s.ctx - (t - wt.nt0) * BK); };
  // Ids of 64 consecutive pages, one a lane: a tile then costs a lane read.  (One load a tile
  // would wait, with everything in flight, a round trip each.)
  int win_ids = 0, win_first = -(1 << 30);
  auto page_of = [&](int t) {
    if ((unsigned)(t - win_first) >= 64u) {
      win_first = t;
      win_ids = pages[min(t + lane, max(p.ctx_pages_per_batch - 1, 0))];
      asm volatile("" ::"v"(win_ids));  // (the wait for it stays here)
    }
    return min(max(__builtin_amdgcn_readlane(win_ids, t - win_first), 0), max(p.ctx_rows - 1, 0));
  };
  // context tile t's first row, in elements of a pool or a packed context
  auto ctx_elem = [&](int t) {
    constexpr int PT = FMLM_PAGE_ROWS / BK;  // tiles of a page
    return (int64_t)s.h * p.c_sh + (pages ? (int64_t)page_of(t / PT) * p.ctx_page_stride + (t % PT) * BK * p.c_sn
                                          : (int64_t)(ctx0 + t * BK) * p.c_sn);
  };
  // a 16-bit tile's loads
  auto fetch = [&](int t, bool is_v, char* to) {
    const int last = keys_in(t) - 1;
    if (t < wt.nt0) {
      WTile<T, D>::template load<BK>((const char*)(is_v ? p.v_ctx : p.k_ctx) + ctx_elem(t) * 2, (uint32_t)p.c_sn * 2u, last,
                                      lds_addr(to), wave, lane);
    } else {
      const int64_t sb = is_v ? p.v_sb : p.k_sb, sh = is_v ? p.v_sh : p.k_sh, sn = is_v ? p.v_sn : p.k_sn;
      WTile<T, D>::template load<BK>((const char*)(is_v ? p.v : p.k) + row_at(p.kv_layout, s.b, s.h, s.q0, (t - wt.nt0) * BK, sb, sh, sn) * 2,
                                      (uint32_t)sn * 2u, last, lds_addr(to), wave, lane);
    }
  };
  // The walk of the 16-bit tiles: the next tile's first rows of K and V, moved on by their pitch, a page or
  // (the first tile of the band, and of the new tokens) from the segment's start.
  struct Walk {
    const char *k, *v;
    uint32_t rk, rv;
    int at, t;
  } wk{nullptr, nullptr, 0, 0, 0, 0};
  auto seek = [&](int v) {  // to tile v of this part
    wk.at = v;
    wk.t = tile_at(v);
    if (wk.t < wt.nt0) {
      const int64_t e = ctx_elem(wk.t) * 2;
      wk.rk = wk.rv = __builtin_amdgcn_readfirstlane((uint32_t)p.c_sn * 2u);
      wk.k = uniform_ptr((const char*)p.k_ctx + e);
      wk.v = uniform_ptr((const char*)p.v_ctx + e);
    } else {
      const int j = (wk.t - wt.nt0) * BK;
      wk.rk = __builtin_amdgcn_readfirstlane((uint32_t)p.k_sn * 2u);
      wk.rv = __builtin_amdgcn_readfirstlane((uint32_t)p.v_sn * 2u);
      wk.k = uniform_ptr((const char*)p.k + row_at(p.kv_layout, s.b, s.h, s.q0, j, p.k_sb, p.k_sh, p.k_sn) * 2);
      wk.v = uniform_ptr((const char*)p.v + row_at(p.kv_layout, s.b, s.h, s.q0, j, p.v_sb, p.v_sh, p.v_sn) * 2);
    }
  };
  const int jump = wt.sink - vb;  // the first tile of the band, in this part's count
  auto move = [&]() {
    const int v = wk.at + 1;
    if (v >= n) return;
    if (v == jump || wk.t + 1 == wt.nt0 || (pages && wk.t < wt.nt0)) {
      seek(v);
      return;
    }
    wk.at = v;
    wk.t += 1;
    wk.k += (size_t)wk.rk * BK;
    wk.v += (size_t)wk.rv * BK;
  };
  // lane offsets of a whole tile at the pitch of most of them
  typedef WTile<T, D> Tile;
  constexpr int NL = BK / (Tile::RPI * kNW);
  uint32_t off0[FP4 ? 1 : NL];
  uint32_t pitch0 = 0;
  auto load_rows = [&](const char* src, uint32_t pitch, int last, char* to) {
    if constexpr (!FP4) {
      if (last == BK - 1 && pitch == pitch0) {
        Tile::template load_at<BK>(src, off0, lds_addr(to), wave);
        return;
      }
    }
    Tile::template load<BK>(src, pitch, last, lds_addr(to), wave, lane);
  };
  // a 4-bit tile: thread i has part i % TPR of row i / TPR, CW dwords
  uint32_t code[2][C::STAGE ? 1 : CW], csc[2];
  auto fetch_codes = [&](int t, bool is_v) {
    const int row = min(tid / C::TPR, keys_in(t) - 1), x = is_v ? 1 : 0;
    const int64_t e0 = ctx_elem(t);
    const uint32_t at = (uint32_t)row * D + (tid % C::TPR) * (D / C::TPR);
    const char* const src = uniform_ptr((const char*)(is_v ? p.v_ctx : p.k_ctx) + e0 / 2);
    const char* const ssc = uniform_ptr((const char*)(is_v ? a.v_scales : a.k_scales) + e0 / kFp4Block);
    if constexpr (C::STAGE) {
      dma16_sbase(src, at / 2, __builtin_amdgcn_readfirstlane(lds_addr(smem) + (2 + C::NV) * C::TILEB + (2 * wave + x) * 1024));
    } else if constexpr (CW == 1) {
      code[x][0] = *(const uint32_t*)(src + at / 2);
    } else if constexpr (CW == 2) {
      const u32x2 w = *(const u32x2*)(src + at / 2);
      code[x][0] = w[0];
      code[x][1] = w[1];
    }
    csc[x] = (uint8_t)ssc[at / kFp4Block];
  };
  // the loaded codes as a 16-bit tile (STAGE: this wave's load has landed)
  auto put_codes = [&](bool is_v, char* to) {
    const int row = tid / C::TPR, x = is_v ? 1 : 0;
    uint32_t w[CW];
    if constexpr (C::STAGE) {
      const u32x4 r = *(const u32x4*)(smem + (2 + C::NV) * C::TILEB + (2 * wave + x) * 1024 + 16 * lane);
#pragma unroll
      for (int i = 0; i < CW; ++i) w[i] = r[i];
    } else {
#pragma unroll
      for (int i = 0; i < CW; ++i) w[i] = code[x][i];
    }
#pragma unroll
    for (int i = 0; i < CW; ++i)
      *(u32x4*)(to + row * (D * 2) + 16 * (((tid % C::TPR) * CW + i) ^ kv_swz<D>(row))) = fp4_oct<T>(w[i], fp4_scale(csc[x]));
  };
  auto is_code = [&](int t) { return FP4 && t < wt.nt0; };

  v8 qf[QB][C::KC];
  f32x4 o[C::NDB][QB], lsum[QB];
  float m[QB], mx[QB], lx[QB];  // lx (LSE): the lane's part of the sum of the probabilities as they are
  f32x4 sa[NKB][QB], sb[NKB][QB];
  v8 ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) ones[e] = (T)1.0f;
  pin(ones);

  // raw row maxima of a score tile
  auto row_max = [&](const f32x4 (&x)[NKB][QB]) {
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      float y = vmax(vmax(x[0][qb][0], x[0][qb][1]), vmax(x[0][qb][2], x[0][qb][3]));
#pragma unroll
      for (int kb = 1; kb < NKB; ++kb)
        y = vmax(vmax(y, vmax(x[kb][qb][0], x[kb][qb][1])), vmax(x[kb][qb][2], x[kb][qb][3]));
      mx[qb] = lane_max_xor16_32(y);
    }
  };
  const int w0 = s.first + row0 + wave * QB * 16, w1 = min(w0 + QB * 16, s.first + row0 + rows) - 1;
  // position of a tile's first key; whether any of the wave's rows sees a key of it
  auto key_at = [&](int t) { return t < wt.nt0 ? t * BK : s.ctx + (t - wt.nt0) * BK; };
  auto seen = [&](int t) {
    const int kp = key_at(t);
    return kp <= w1 + a.right && (kp + BK > w0 - a.left || kp < a.sinks);
  };
  // scores of keys that a row does not see to -inf; returns whether there can be any
  auto mask = [&](int t, f32x4 (&x)[NKB][QB]) {
    const int nk = keys_in(t), kp = key_at(t);
    if (!(nk < BK || kp + BK - 1 > w0 + a.right || (kp < w1 - a.left && kp + BK > a.sinks))) return false;
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const int pos = w0 + qb * 16 + l16, k0 = kp + 4 * gq;  // element (kb, r) is key k0 + 16 kb + r
      const InView view(pos - a.left - k0, min(pos + a.right - k0, nk - 1 - 4 * gq), a.sinks - k0);
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[kb][qb][r] = view.pick(kb, r, x[kb][qb][r], -INFINITY);
    }
    return true;
  };

  // ---- the slots.  Slot s runs the MFMAs of fragment s: [0, NKF) of K(v + 1) (sn += K Q^T, beside a
  // share of P(v)'s exponentials), [NKF, NF) of V(v) (O += V^T P, beside a share of sn's maxima).
  constexpr int NF = C::NKF + C::NVF, NP = NKB * QB * 2, NMS = NKB * QB + QB;
  u32x4 pf[NKS][QB];
  auto slots = [&](f32x4 (&sc)[NKB][QB], f32x4 (&sn)[NKB][QB], const char* kn, const char* vt) {
    float ref[QB], mpart[QB], mhold[QB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) ref[qb] = m[qb] == -INFINITY ? 0.f : -m[qb];  // (no key yet: every score is -inf)
    v8 fr[C::LEAD + 1];
    auto issue = [&](int r) {
      if (r < C::NKF) fr[r % (C::LEAD + 1)] = tr.row(kn, r % NKB, r / NKB);
      else fr[r % (C::LEAD + 1)] = tr.col(vt, (r - C::NKF) / C::NDB, (r - C::NKF) % C::NDB);
    };
    auto exp_pair = [&](int pi) {
      const int qb = pi / (2 * NKB), kb = (pi >> 1) % NKB, r = (pi & 1) * 2;
      if (r == 0) pin(sc[kb][qb]);
      const float e0 = fast_exp2(fmaf(sc[kb][qb][r], c, ref[qb])), e1 = fast_exp2(fmaf(sc[kb][qb][r + 1], c, ref[qb]));
      uint32_t w = pack2<T>(e0, e1);
      pin(w);
      if constexpr (LSE) lx[qb] += e0 + e1;
      pf[kb >> 1][qb][(kb & 1) * 2 + (pi & 1)] = w;
    };
    auto max_step = [&](int k) {
      if (k < NKB * QB) {
        const int qb = k / NKB, kb = k % NKB;
        pin(sn[kb][qb]);
        const f32x4 x = sn[kb][qb];
        if (kb == 0) {
          mpart[qb] = vmax(vmax(x[0], x[1]), x[2]);
        } else {
          mpart[qb] = vmax(vmax(mpart[qb], mhold[qb]), x[0]);
          mpart[qb] = vmax(vmax(mpart[qb], x[1]), x[2]);
        }
        mhold[qb] = x[3];
        if (kb == NKB - 1) mpart[qb] = vmax(mpart[qb], mhold[qb]);
        pin(mpart[qb]);
      } else {
        const int qb = k - NKB * QB;
        mx[qb] = lane_max_xor16_32(mpart[qb]);
        pin(mx[qb]);
      }
    };
#pragma unroll
    for (int r = 0; r < C::LEAD; ++r) issue(r);
    __builtin_amdgcn_s_setprio(1);  // ahead of a wave that waits or loads, the second half highest
#pragma unroll
    for (int sl = 0; sl < NF; ++sl) {
      if (sl + C::LEAD < NF) issue(sl + C::LEAD);
      if (sl == C::NKF) __builtin_amdgcn_s_setprio(2);
      const v8 x = fr[sl % (C::LEAD + 1)];
      if (sl < C::NKF) {
        const int kb = sl % NKB, kc = sl / NKB;
#pragma unroll
        for (int qb = 0; qb < QB; ++qb)
          sn[kb][qb] = Mfma<T>::run(x, qf[qb][kc], kc == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sn[kb][qb]);
#pragma unroll
        for (int pi = sl * NP / C::NKF; pi < (sl + 1) * NP / C::NKF; ++pi) exp_pair(pi);
      } else {
        const int j = sl - C::NKF, ks = j / C::NDB, db = j % C::NDB;
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) o[db][qb] = Mfma<T>::run(x, __builtin_bit_cast(v8, pf[ks][qb]), o[db][qb]);
        if (db == C::NDB - 1)
#pragma unroll
          for (int qb = 0; qb < QB; ++qb) lsum[qb] = Mfma<T>::run(ones, __builtin_bit_cast(v8, pf[ks][qb]), lsum[qb]);
#pragma unroll
        for (int k = j * NMS / C::NVF; k < (j + 1) * NMS / C::NVF; ++k) max_step(k);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
  };
  auto step = [&](int v, int u, f32x4 (&sc)[NKB][QB], f32x4 (&sn)[NKB][QB]) {
    if constexpr (FP4) {
      const int tk = v + 2 < n ? tile_at(v + 2) : -1, tv = v + 1 < n ? tile_at(v + 1) : -1;
      if (tk >= 0 && is_code(tk)) put_codes(false, kbuf(u));
      if (tv >= 0 && is_code(tv)) put_codes(true, vbuf(u + 1));
      if constexpr (C::STAGE) wait_reads();  // the loads below overwrite what the wave has just read
      if (tk >= 0 && !is_code(tk)) fetch(tk, false, kbuf(u));
      if (tv >= 0 && !is_code(tv)) fetch(tv, true, vbuf(u + 1));
      const int nk = v + 3 < n ? tile_at(v + 3) : -1;
      if (nk >= 0 && is_code(nk)) fetch_codes(nk, false);
      if (tk >= 0 && is_code(tk)) fetch_codes(tk, true);
    } else {
      if (v + 2 < n) {  // the walk stands at tile v + 2
        const int last = keys_in(wk.t) - 1;
        load_rows(wk.k, wk.rk, last, kbuf(u));
        load_rows(wk.v, wk.rv, last, vbuf(u + 2));
        move();
      }
    }
    // A wave that sees neither tile leaves the matrix cores and LDS to the others; the scores that it has
    // then not made are all masked when one of the two tiles is in view.  With 128-row tiles a window of
    // 1024 keys takes 176 us with this and 180 without; with 64-row ones, whose waves differ by less
    // than a tile, 72 without and 74 with it, with 4 bits (no window) 93 and 95.
    bool look = active;
    if constexpr (QB == 2 && !FP4) look = active && (seen(tile_at(v)) || (v + 1 < n && seen(tile_at(v + 1))));
    if (look) {
      if (mask(tile_at(v), sc)) row_max(sc);
      bool grow = false;
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        mx[qb] *= c;
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
          if constexpr (LSE) lx[qb] *= alpha;
#pragma unroll
          for (int db = 0; db < C::NDB; ++db) o[db][qb] *= alpha;
        }
      }
      slots(sc, sn, kbuf(u + 1), vbuf(u));
    }
    // the loads of the next step's tiles have landed: all but V(v + 2)'s, the last ones issued
    constexpr int VPW = BK / (WTile<T, D>::RPI * kNW);
    if (C::NV == 3 && v + 2 < n) __builtin_amdgcn_s_waitcnt((VPW & 15) | (7 << 4) | (0 << 8) | ((VPW >> 4) << 14));
    else __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
  };

  // fragment kc of the lane's row of block qb
  auto q_frag = [&](int qb, int kc) {
    const int row = (wave * QB + qb) * 16 + l16;
    const int64_t off = row_at(p.q_layout, s.b, s.h, s.q0, row0 + row, p.q_sb, p.q_sh, p.q_sn);
    return __builtin_bit_cast(v8, __builtin_bit_cast(u32x4, ld_frag<T>(p.q, off + kc * 32 + gq * 8, row < rows)) ^ qsign);
  };
  // tile v, with the wait for it
  auto bring = [&](int v, bool is_v, char* to) {
    const int t = tile_at(v);
    if constexpr (FP4) {
      if (is_code(t)) {
        fetch_codes(t, is_v);
        __builtin_amdgcn_s_waitcnt(0);
        put_codes(is_v, to);
        if constexpr (C::STAGE) wait_reads();
        return;
      }
    }
    fetch(t, is_v, to);
  };
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    m[qb] = -INFINITY;
    lx[qb] = 0.f;
    lsum[qb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int db = 0; db < C::NDB; ++db) o[db][qb] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if (n > 0) {
    // Tiles 0 and 1 (V(1) only with a third buffer), and of 4-bit ones the codes of the next.  Workgroups that
    // start together all wait for memory here: what S(0) needs comes first, q by LDS too, where V(1) and
    // V(2) follow it, and S(0) does not wait for the others.
    constexpr int VPW = BK / (Tile::RPI * kNW);
    if constexpr (FP4) {
      bring(0, false, kbuf(0));
      bring(0, true, vbuf(0));
      if (n > 1) bring(1, false, kbuf(1));
      if (n > 2 && is_code(tile_at(2))) fetch_codes(tile_at(2), false);
      if (n > 1 && is_code(tile_at(1))) fetch_codes(tile_at(1), true);
    } else {
      static_assert(C::NV == 3 && QB * 16 * kNW <= 2 * BK, "q's rows in V(1) and V(2)");
      Tile::template load<QB * 16 * kNW>((const char*)p.q + row_at(p.q_layout, s.b, s.h, s.q0, row0, p.q_sb, p.q_sh, p.q_sn) * 2,
                                         (uint32_t)p.q_sn * 2u, rows - 1, lds_addr(vbuf(1)), wave, lane);
      seek(0);
      pitch0 = wk.rk;
      Tile::template offsets<BK>(pitch0, wave, lane, off0);
      load_rows(wk.k, wk.rk, keys_in(wk.t) - 1, kbuf(0));
      load_rows(wk.v, wk.rv, keys_in(wk.t) - 1, vbuf(0));
      move();
      if (n > 1) load_rows(wk.k, wk.rk, keys_in(wk.t) - 1, kbuf(1));
    }
    if constexpr (FP4) {
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int kc = 0; kc < C::KC; ++kc) qf[qb][kc] = q_frag(qb, kc);
      __builtin_amdgcn_s_waitcnt(0);
    } else {  // q and K(0) have landed
      if (n > 1) __builtin_amdgcn_s_waitcnt(((2 * VPW) & 15) | (7 << 4) | (0 << 8) | (((2 * VPW) >> 4) << 14));
      else __builtin_amdgcn_s_waitcnt((VPW & 15) | (7 << 4) | (0 << 8) | ((VPW >> 4) << 14));
    }
    __syncthreads();
    if constexpr (!FP4) {
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int kc = 0; kc < C::KC; ++kc)
          qf[qb][kc] = __builtin_bit_cast(v8, __builtin_bit_cast(u32x4, tr.row(vbuf(1), wave * QB + qb, kc)) ^ qsign);
    }
    if (active) {
#pragma unroll
      for (int kc = 0; kc < C::KC; ++kc)
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) {
          const v8 x = tr.row(kbuf(0), kb, kc);
#pragma unroll
          for (int qb = 0; qb < QB; ++qb)
            sa[kb][qb] = Mfma<T>::run(x, qf[qb][kc], kc == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sa[kb][qb]);
        }
      row_max(sa);
    }
    if constexpr (!FP4) __builtin_amdgcn_s_waitcnt(0);  // V(0) and K(1)
    __syncthreads();  // every wave is done with K(0) and q: their buffers may be refilled
    if constexpr (!FP4) {
      if (n > 1) {
        load_rows(wk.v, wk.rv, keys_in(wk.t) - 1, vbuf(1));
        move();
      }
    }
  }
  for (int v = 0; v < n;) {
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      if (v >= n) break;
      if (u & 1) step(v, u, sb, sa);
      else step(v, u, sa, sb);
      ++v;
    }
  }

  // a row's result: a part's record (O, m, l), or the output
  float* const rec = a.records + (((int64_t)(a.tiles - 1 - tile) * a.groups + g) * a.parts + part) * a.rec_rows * (D + 4);
  auto put = [&](int qb, const f32x4 (&x)[C::NDB], float mrow, float l, float lrow) {
    const int row = (wave * QB + qb) * 16 + l16;
    if (row >= rows) return;
    if (parts > 1) {
#pragma unroll
      for (int db = 0; db < C::NDB; ++db) *(f32x4*)(rec + (int64_t)row * D + db * 16 + gq * 4) = x[db];
      if (gq == 0) {
        rec[(int64_t)a.rec_rows * D + 2 * row] = mrow;
        rec[(int64_t)a.rec_rows * D + 2 * row + 1] = l;
      }
      return;
    }
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    if (p.lse && gq == 0)
      p.lse[(int64_t)s.h * p.total_q + s.q0 + row0 + row] = lrow > 0.f ? mrow + __log2f(lrow) : lrow != lrow ? lrow : INFINITY;
    const int64_t off = row_at(p.o_layout, s.b, s.h, s.q0, row0 + row, p.o_sb, p.o_sh, p.o_sn);
#pragma unroll
    for (int db = 0; db < C::NDB; ++db) {
      const f32x4 y = x[db] * inv;
      const u32x2 hi = u32x2{pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3])};
      *(u32x2*)((char*)p.o + (off + db * 16 + gq * 4) * 2) = hi;
      if (a.o_low) {
        f32x4 z;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t w = hi[r / 2];
          z[r] = y[r] - (float)__builtin_bit_cast(T, (uint16_t)(r & 1 ? w >> 16 : w));
        }
        *(u32x2*)((char*)a.o_low + (off + db * 16 + gq * 4) * 2) = u32x2{pack2<T>(z[0], z[1]), pack2<T>(z[2], z[3])};
      }
    }
  };
  float bad = 0.f;
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    f32x4 x[C::NDB];
#pragma unroll
    for (int db = 0; db < C::NDB; ++db) {
      x[db] = o[db][qb];
#pragma unroll
      for (int r = 0; r < 4; ++r) bad = fmaf(x[db][r], 0.f, bad);
    }
    if constexpr (LSE) {
      lx[qb] += __shfl_xor(lx[qb], 16);
      lx[qb] += __shfl_xor(lx[qb], 32);
    }
    put(qb, x, m[qb], lsum[qb][0], LSE ? lx[qb] : lsum[qb][0]);
  }
  // Values that are not finite in keys that a row does not see have reached it as 0 inf.  If there may
  // be any, the rows are computed again, a tile and a block of rows at a time, key by key.
  // (The tiles' LDS is free: every wave has passed the last step's barrier.)
  if (lane == 0) ((int*)smem)[wave] = __builtin_amdgcn_ballot_w64(bad != bad) != 0;
  __syncthreads();
  const int any = ((const int*)smem)[0] | ((const int*)smem)[1] | ((const int*)smem)[2] | ((const int*)smem)[3];
  __syncthreads();
  if (!any) return;
  T* const pw = (T*)(kbuf(1) + wave * 2048);  // the wave's weights [16][64], behind K(0): kbuf(1), V(0) follows 8 KB on
  char* const vt = smem + C::LDS - (C::STAGE ? 2 * kNW * 1024 : 0) - C::TILEB;  // the last V buffer
  for (int qb = 0; qb < QB; ++qb) {
    float mr = -INFINITY, l = 0.f;
    f32x4 x[C::NDB];
#pragma unroll
    for (int db = 0; db < C::NDB; ++db) x[db] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int v = 0; v < n; ++v) {
      bring(v, false, kbuf(0));
      bring(v, true, vt);
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
      const int t = tile_at(v), nk = keys_in(t), kp = t < wt.nt0 ? t * BK : s.ctx + (t - wt.nt0) * BK;
      f32x4 sc[NKB];
#pragma unroll
      for (int kc = 0; kc < C::KC; ++kc) {
        const v8 f = q_frag(qb, kc);
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
          sc[kb] = Mfma<T>::run(tr.row(kbuf(0), kb, kc), f, kc == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sc[kb]);
      }
      const int pos = w0 + qb * 16 + l16, k0 = kp + 4 * gq;
      const int top = min(pos + a.right - k0, nk - 1 - 4 * gq), low = pos - a.left - k0, snk = a.sinks - k0;
      float y = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = kb * 16 + r;
          if (!(j <= top && (j >= low || j < snk))) sc[kb][r] = -INFINITY;
          y = vmax(y, sc[kb][r]);
        }
      const float mn = vmax(mr, lane_max_xor16_32(y) * c), ref = mn == -INFINITY ? 0.f : mn;
      const float alpha = fast_exp2((mr == -INFINITY ? ref : mr) - ref);
      mr = mn;
      l *= alpha;
#pragma unroll
      for (int db = 0; db < C::NDB; ++db) x[db] *= alpha;
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) pw[l16 * 64 + kb * 16 + 4 * gq + r] = (T)fast_exp2(fmaf(sc[kb][r], c, -ref));
      asm volatile("" ::: "memory");
#pragma clang loop unroll(disable)
      for (int j = 0; j < BK; ++j) {
        const float w = (float)pw[l16 * 64 + j];
        l += w;
        if (w != 0.f) {
#pragma unroll
          for (int db = 0; db < C::NDB; ++db) {
            const T* val = (const T*)(vt + j * (D * 2) + 16 * ((2 * db + (gq >> 1)) ^ kv_swz<D>(j)) + 8 * (gq & 1));
#pragma unroll
            for (int e = 0; e < 4; ++e) x[db][e] = fmaf(w, (float)val[e], x[db][e]);
          }
        }
      }
      __syncthreads();
    }
    put(qb, x, mr, l, l);
  }
}

// ---------------------------------------------------------------------------
// Forward of few rows (at most 16 a sequence) over a 4-bit context: a wave has all rows and walks
// tiles of its own, without a barrier.  Lane l16 + 16 g loads quarter g of the rows 16 kb + l16 of a
// tile, D / 8 bytes, which are whole lines for the wave, and a dword of it is a fragment of
// S^T = K Q^T: the contraction takes the elements in the order (quarter, fragment), and q comes in
// that order too.  V is converted the same way into a wave's own 32 rows of LDS and read back
// transposed.  A tile's registers are loaded again as soon as they have been converted.  The four
// waves' sums meet in LDS at the end.  Bound by memory: 64 users over 500 to 8192 keys of 16 heads, D = 128, 633 MB of
// codes and scales in 127 us, 97% of a large copy's rate; the same through window_fwd_kernel's
// shared tiles 226 us with 4096 keys each, here 114 (16 rows a sequence: 73 and 35).
// A wave whose rows come out not finite walks its tiles once more, key by key (see there).
// ---------------------------------------------------------------------------
constexpr int kFewRows = 16;

template <int D>
struct FewCfg {
  static constexpr int KC = D / 32, NDB = D / 16;
  static constexpr int CS = D == 256 ? 2 : 1;             // scales of a quarter row
  static constexpr int WAVEB = 32 * D * 2;                // V rows; at the end 16 rows of fp32
  static constexpr int LDS = kNW * (WAVEB + 2 * kFewRows * 4);  // ... and m and l of each
  static constexpr int WPS = D <= 128 ? 3 : 2;
};

template <typename T, int D>
__global__ __launch_bounds__(kNW * 64, FewCfg<D>::WPS) void window_fp4_few_kernel(const fmlm_attn_params p, const WinArgs a) {
  typedef FewCfg<D> C;
  typedef typename Mfma<T>::v8 v8;
  extern __shared__ __align__(16) char smem[];
  int g, part, tile;
  if (!win_unit(p, a, a.parts, g, part, tile)) return;
  const WinSeq s = win_seq(p, a, g / p.H, g % p.H);
  const int rows = min(kFewRows, s.len);
  if (rows <= 0) return;
  const WinTiles wt = win_tiles(a, s, s.first, s.first + rows - 1, 6);
  const int parts = win_parts(wt.n, a.parts);
  if (part >= parts) return;
  const int vb = (int)((int64_t)wt.n * part / parts), ve = (int)((int64_t)wt.n * (part + 1) / parts);

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, gq = lane >> 4;
  const WTile<T, D> tr(l16, gq);
  char* const vt = smem + wave * C::WAVEB;
  const uint32_t qsign = p.scale < 0.f ? 0x80008000u : 0u;
  const float c = fmaxf(fabsf(p.scale) * kLog2e, 1e-30f);
  v8 qf[C::KC];
  {
    const int64_t off = row_at(p.q_layout, s.b, s.h, s.q0, l16, p.q_sb, p.q_sh, p.q_sn) + gq * (D / 4);
#pragma unroll
    for (int kc = 0; kc < C::KC; ++kc)
      qf[kc] = __builtin_bit_cast(v8, __builtin_bit_cast(u32x4, ld_frag<T>(p.q, off + kc * 8, l16 < rows)) ^ qsign);
  }
  const int cb = ctx_batch_of(p, s.b);
  const int32_t* const pages = p.ctx_block_table + (int64_t)cb * p.ctx_pages_per_batch;
  auto page_of = [&](int v) {  // of context tile v of the walk (any, past its end)
    const int t = min(wt.tile(v), max(wt.nt0 - 1, 0));
    return wt.nt0 > 0 ? min(max(ldc(pages, t), 0), max(p.ctx_rows - 1, 0)) : 0;
  };
  uint32_t kw[4][C::KC], vw[4][C::KC], ks[4][C::CS], vs[4][C::CS];
  auto load = [&](const void* codes, const uint8_t* scales, int page, int last, uint32_t (&w)[4][C::KC],
                  uint32_t (&sc)[4][C::CS]) {
    const int64_t e0 = (int64_t)s.h * p.c_sh + (int64_t)page * p.ctx_page_stride;
    const char* const src = uniform_ptr((const char*)codes + e0 / 2);
    const char* const ssc = uniform_ptr((const char*)scales + e0 / kFp4Block);
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      const uint32_t row = (uint32_t)min(kb * 16 + l16, last), at = row * (D / 2) + gq * (D / 8);
      if constexpr (C::KC == 1) w[kb][0] = *(const uint32_t*)(src + at);
      else if constexpr (C::KC == 2) {
        const u32x2 x = *(const u32x2*)(src + at);
        w[kb][0] = x[0];
        w[kb][1] = x[1];
      } else {
#pragma unroll
        for (int i = 0; i < C::KC; i += 4) {
          const u32x4 x = *(const u32x4*)(src + at + 4 * i);
#pragma unroll
          for (int j = 0; j < 4; ++j) w[kb][i + j] = x[j];
        }
      }
      const uint32_t sat = row * (D / kFp4Block) + gq * (D / 4) / kFp4Block;
#pragma unroll
      for (int i = 0; i < C::CS; ++i) sc[kb][i] = (uint8_t)ssc[sat + i];
    }
  };
  auto keys_in = [&](int t) { return min(kBK, t < wt.nt0 ? s.ctx - t * kBK : s.total - s.ctx - (t - wt.nt0) * kBK); };

  f32x4 o[C::NDB], lsum = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY;
#pragma unroll
  for (int db = 0; db < C::NDB; ++db) o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
  v8 ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) ones[e] = (T)1.0f;

  // scores of a tile of nk keys from position kp on: masked, the running maximum and P
  u32x4 pf[2];
  bool edge;
  auto softmax = [&](f32x4 (&sc)[4], int kp, int nk) {
    edge = nk < kBK || kp + kBK - 1 > s.first + a.right || (kp < s.first + rows - 1 - a.left && kp + kBK > a.sinks);
    if (edge) {
      const int pos = s.first + l16, k0 = kp + 4 * gq;
      const InView view(pos - a.left - k0, min(pos + a.right - k0, nk - 1 - 4 * gq), a.sinks - k0);
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[kb][r] = view.pick(kb, r, sc[kb][r], -INFINITY);
    }
    float mx = vmax(vmax(sc[0][0], sc[0][1]), vmax(sc[0][2], sc[0][3]));
#pragma unroll
    for (int kb = 1; kb < 4; ++kb) mx = vmax(vmax(mx, vmax(sc[kb][0], sc[kb][1])), vmax(sc[kb][2], sc[kb][3]));
    mx = lane_max_xor16_32(mx) * c;
    if (__builtin_amdgcn_ballot_w64(mx > m + kSlack)) {
      const float mn = mx > m + kSlack ? mx : m;
      const float alpha = mn == -INFINITY ? 1.f : fast_exp2(m - mn);
      m = mn;
      lsum *= alpha;
#pragma unroll
      for (int db = 0; db < C::NDB; ++db) o[db] *= alpha;
    }
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int r = 0; r < 4; r += 2)
        pf[kb >> 1][(kb & 1) * 2 + r / 2] =
            pack2<T>(fast_exp2(fmaf(sc[kb][r], c, -ref)), fast_exp2(fmaf(sc[kb][r + 1], c, -ref)));
#pragma unroll
    for (int h = 0; h < 2; ++h) lsum = Mfma<T>::run(ones, __builtin_bit_cast(v8, pf[h]), lsum);
  };
  // O += P V of the 32 keys in LDS
  auto values = [&](int h) {
    asm volatile("" ::: "memory");
#pragma unroll
    for (int db = 0; db < C::NDB; ++db) o[db] = Mfma<T>::run(tr.col(vt, 0, db), __builtin_bit_cast(v8, pf[h]), o[db]);
    asm volatile("" ::: "memory");
  };

  // of the loaded codes: scores, and the values of keys 32 h.. as 16-bit rows in LDS
  auto scores = [&](f32x4 (&sc)[4]) {
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      sc[kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kc = 0; kc < C::KC; ++kc)
        sc[kb] = Mfma<T>::run(__builtin_bit_cast(v8, fp4_oct<T>(kw[kb][kc], fp4_scale(ks[kb][kc / 4 % C::CS]))), qf[kc], sc[kb]);
    }
  };
  auto put_row = [&](int i, int kc, u32x4 x) {  // chunk kc of the lane's quarter of row 16 i + l16
    *(u32x4*)(vt + (i * 16 + l16) * (D * 2) + 16 * ((gq * C::KC + kc) ^ kv_swz<D>(l16))) = x;
  };
  auto put_values = [&](int h) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int kc = 0; kc < C::KC; ++kc)
        put_row(i, kc, fp4_oct<T>(vw[2 * h + i][kc], fp4_scale(vs[2 * h + i][kc / 4 % C::CS])));
  };
  // scores of the new tokens' own keys, nk of them, and their values in LDS
  auto own_tile = [&](f32x4 (&sc)[4], int nk) {
    const int64_t ko = row_at(p.kv_layout, s.b, s.h, s.q0, min(l16, nk - 1), p.k_sb, p.k_sh, p.k_sn) + gq * (D / 4);
    const int64_t vo = row_at(p.kv_layout, s.b, s.h, s.q0, min(l16, nk - 1), p.v_sb, p.v_sh, p.v_sn) + gq * (D / 4);
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) sc[kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kc = 0; kc < C::KC; ++kc) {
      sc[0] = Mfma<T>::run(ld_frag<T>(p.k, ko + kc * 8, true), qf[kc], sc[0]);
      put_row(0, kc, *(const u32x4*)((const char*)p.v + (vo + kc * 8) * 2));
      put_row(1, kc, u32x4{0u, 0u, 0u, 0u});
    }
  };

  int page = page_of(vb + wave), next = page_of(vb + wave + kNW);
  if (vb + wave < ve && wt.tile(vb + wave) < wt.nt0) {
    const int last = keys_in(wt.tile(vb + wave)) - 1;
    load(p.k_ctx, a.k_scales, page, last, kw, ks);
    load(p.v_ctx, a.v_scales, page, last, vw, vs);
  }
  for (int v = vb + wave; v < ve; v += kNW) {
    const int t = wt.tile(v), nk = keys_in(t);
    if (t >= wt.nt0) break;  // the new tokens, at most 16: one tile, the last
    f32x4 sc[4];
    scores(sc);
    const bool more = v + kNW < ve && wt.tile(v + kNW) < wt.nt0;
    const int nlast = more ? keys_in(wt.tile(v + kNW)) - 1 : 0;
    page = next;
    if (more) load(p.k_ctx, a.k_scales, page, nlast, kw, ks);
    next = page_of(v + 2 * kNW);
    softmax(sc, t * kBK, nk);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      put_values(h);
      values(h);
    }
    if (more) load(p.v_ctx, a.v_scales, page, nlast, vw, vs);
  }
  // the new tokens' own keys, by the wave whose turn it is
  if (ve > vb && wt.tile(ve - 1) >= wt.nt0 && (ve - 1 - vb) % kNW == wave) {
    const int nk = keys_in(wt.tile(ve - 1));
    f32x4 sc[4];
    own_tile(sc, nk);
    softmax(sc, s.ctx, nk);
    values(0);
  }

  // Values that are not finite in keys that a row does not see have reached it as 0 inf.  If there may be
  // any, the wave walks its tiles once more and adds what a row sees key by key.
  float bad = 0.f;
#pragma unroll
  for (int db = 0; db < C::NDB; ++db)
#pragma unroll
    for (int r = 0; r < 4; ++r) bad = fmaf(o[db][r], 0.f, bad);
  if (__builtin_amdgcn_ballot_w64(bad != bad)) {
    m = -INFINITY;
    lsum = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int db = 0; db < C::NDB; ++db) o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma clang loop unroll(disable)
    for (int v = vb + wave; v < ve; v += kNW) {
      const int t = wt.tile(v), nk = keys_in(t);
      const bool own = t >= wt.nt0;
      f32x4 sc[4];
      if (own) {
        own_tile(sc, nk);
      } else {
        page = page_of(v);
        load(p.k_ctx, a.k_scales, page, nk - 1, kw, ks);
        load(p.v_ctx, a.v_scales, page, nk - 1, vw, vs);
        scores(sc);
      }
      softmax(sc, own ? s.ctx : t * kBK, nk);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (own && h > 0) break;
        if (!own) put_values(h);
        asm volatile("" ::: "memory");
#pragma clang loop unroll(disable)
        for (int x = 0; x < 8; ++x) {  // keys 4 x.. of these 32: their weights are in lane l16 + 16 (x % 4)
          const uint32_t w0 = x < 4 ? pf[h][0] : pf[h][2], w1 = x < 4 ? pf[h][1] : pf[h][3];
          const uint32_t w[2] = {(uint32_t)__shfl((int)w0, l16 + 16 * (x & 3)), (uint32_t)__shfl((int)w1, l16 + 16 * (x & 3))};
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float wgt = (float)__builtin_bit_cast(T, (uint16_t)(r & 1 ? w[r / 2] >> 16 : w[r / 2]));
            const int j = 4 * x + r;
            if (wgt != 0.f) {
#pragma unroll
              for (int db = 0; db < C::NDB; ++db) {
                const T* const val = (const T*)(vt + j * (D * 2) + 16 * ((2 * db + (gq >> 1)) ^ kv_swz<D>(j & 15)) + 8 * (gq & 1));
#pragma unroll
                for (int e = 0; e < 4; ++e) o[db][e] = fmaf(wgt, (float)val[e], o[db][e]);
              }
            }
          }
        }
        asm volatile("" ::: "memory");
      }
    }
  }

  // ---- the four waves' parts: O to LDS (over V), m and l behind
  float* const stat = (float*)(smem + kNW * C::WAVEB);
  asm volatile("" ::: "memory");
  if (l16 < rows) {
#pragma unroll
    for (int db = 0; db < C::NDB; ++db) *(f32x4*)(vt + (l16 * D + db * 16 + gq * 4) * 4) = o[db];
    if (gq == 0) {
      stat[(wave * kFewRows + l16) * 2] = m;
      stat[(wave * kFewRows + l16) * 2 + 1] = lsum[0];
    }
  }
  __syncthreads();
  const int64_t unit = (int64_t)g * a.parts + part;
  float* const rec = a.records + unit * a.rec_rows * (D + 4);
  for (int i = tid; i < rows * (D / 8); i += kNW * 64) {
    const int row = i / (D / 8), d = (i % (D / 8)) * 8;
    float top = -INFINITY, l = 0.f;
#pragma unroll
    for (int k = 0; k < kNW; ++k) top = vmax(top, stat[(k * kFewRows + row) * 2]);
    const float ref = top == -INFINITY ? 0.f : top;
    f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f}, y = x;
#pragma unroll
    for (int k = 0; k < kNW; ++k) {
      const float w = fast_exp2(stat[(k * kFewRows + row) * 2] - ref);
      const f32x4* src = (const f32x4*)(smem + k * C::WAVEB + (row * D + d) * 4);
      l = fmaf(w, stat[(k * kFewRows + row) * 2 + 1], l);
      x += src[0] * w;
      y += src[1] * w;
    }
    if (parts > 1) {
      *(f32x4*)(rec + row * D + d) = x;
      *(f32x4*)(rec + row * D + d + 4) = y;
      if (d == 0) {
        rec[(int64_t)a.rec_rows * D + 2 * row] = top;
        rec[(int64_t)a.rec_rows * D + 2 * row + 1] = l;
      }
      continue;
    }
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    x *= inv;
    y *= inv;
    const int64_t off = row_at(p.o_layout, s.b, s.h, s.q0, row, p.o_sb, p.o_sh, p.o_sn);
    *(u32x4*)((char*)p.o + (off + d) * 2) =
        u32x4{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3])};
  }
}

// ---------------------------------------------------------------------------
// The parts' records joined.  A workgroup takes RR rows of a query tile (blockIdx.y), 8 columns of a
// row a thread; with RR < 256 / (D / 8) the other threads share a row's parts, and meet in LDS.  A
// thread has kMergeLoads records in flight (one after the other: 9 us for 32 parts of one row, of
// 19 in all).
// ---------------------------------------------------------------------------
constexpr int kMergeLoads = 4;
template <typename T, int D, int RR>
__global__ __launch_bounds__(256) void window_merge_kernel(const fmlm_attn_params p, const WinArgs a, int bq) {
  constexpr int CPR = D / 8, GG = 256 / (CPR * RR);  // columns and part groups
  __shared__ __align__(16) float sums[GG][RR][D];
  __shared__ float stat[GG][RR][2];
  int g, part, tile;
  if (!win_unit(p, a, 1, g, part, tile)) return;
  tile = a.tiles - 1 - tile;
  const WinSeq s = win_seq(p, a, g / p.H, g % p.H);
  const int row0 = tile * bq, rows = min(bq, s.len - row0);
  const int tid = threadIdx.x, c8 = tid % CPR, rr = (tid / CPR) % RR, gg = tid / (CPR * RR);
  const int row = blockIdx.y * RR + rr;
  if ((int)blockIdx.y * RR >= rows) return;
  const int parts = win_parts(win_tiles(a, s, s.first + row0, s.first + row0 + rows - 1, a.lg).n, a.parts);
  if (parts <= 1) return;
  const int64_t unit = ((int64_t)(a.tiles - 1 - tile) * a.groups + g) * a.parts, pitch = (int64_t)a.rec_rows * (D + 4);
  const float* const rec = a.records + unit * pitch + (int64_t)row * D + c8 * 8;
  const float* const st = a.records + unit * pitch + (int64_t)a.rec_rows * D + 2 * row;
  float top = -INFINITY, l = 0.f;
  f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f}, y = x;
  if (row < rows)
    for (int k0 = gg; k0 < parts; k0 += GG * kMergeLoads) {
      float mk[kMergeLoads], lk[kMergeLoads];
      f32x4 xk[kMergeLoads], yk[kMergeLoads];
#pragma unroll
      for (int i = 0; i < kMergeLoads; ++i) {
        const int64_t at = min(k0 + i * GG, parts - 1) * pitch;
        mk[i] = st[at];
        lk[i] = st[at + 1];
        xk[i] = *(const f32x4*)(rec + at);
        yk[i] = *(const f32x4*)(rec + at + 4);
      }
      float mt = top;
#pragma unroll
      for (int i = 0; i < kMergeLoads; ++i) {
        if (k0 + i * GG >= parts) mk[i] = -INFINITY;
        mt = vmax(mt, mk[i]);
      }
      const float ref = mt == -INFINITY ? 0.f : mt, w0 = fast_exp2((top == -INFINITY ? ref : top) - ref);
      top = mt;
      l *= w0;
      x *= w0;
      y *= w0;
#pragma unroll
      for (int i = 0; i < kMergeLoads; ++i) {
        if (k0 + i * GG >= parts) continue;
        const float w = fast_exp2(mk[i] - ref);
        l = fmaf(w, lk[i], l);
        x += xk[i] * w;
        y += yk[i] * w;
      }
    }
  if constexpr (GG > 1) {
    *(f32x4*)&sums[gg][rr][c8 * 8] = x;
    *(f32x4*)&sums[gg][rr][c8 * 8 + 4] = y;
    if (c8 == 0) {
      stat[gg][rr][0] = top;
      stat[gg][rr][1] = l;
    }
    __syncthreads();
    if (gg > 0) return;
    float all = -INFINITY;
#pragma unroll
    for (int i = 0; i < GG; ++i) all = vmax(all, stat[i][rr][0]);
    const float ref = all == -INFINITY ? 0.f : all;
    l = 0.f;
    x = y = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = 0; i < GG; ++i) {
      const float w = fast_exp2(stat[i][rr][0] - ref);
      l = fmaf(w, stat[i][rr][1], l);
      x += *(const f32x4*)&sums[i][rr][c8 * 8] * w;
      y += *(const f32x4*)&sums[i][rr][c8 * 8 + 4] * w;
    }
  }
  if (row >= rows) return;
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  x *= inv;
  y *= inv;
  const int64_t off = row_at(p.o_layout, s.b, s.h, s.q0, row0 + row, p.o_sb, p.o_sh, p.o_sn);
  *(u32x4*)((char*)p.o + (off + c8 * 8) * 2) =
      u32x4{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3])};
}

// ---------------------------------------------------------------------------
// Backward, with the forward's row statistics: P = 2^(c s - lse) again, no running maximum.  P and dS go to
// the input type as operands, off by half a step each; delta comes from o and o_low in 32 bits, or
// o's rounding, the same for all of a row's keys, would be the largest error of dq and dk (1.55 times
// the plain form's in fp16, with o_low 1.4).  What is left in it of the rounding of the forward's P goes
// for dK: the dq kernel adds up what each row's dS, unrounded, lacks to a sum of 0.  dq itself has the delta that is
// not yet so exact; where that counts (TWO: rows of few keys) its dS goes in two terms.  dS is held without its
// scale: in fp16 P (do V^T - delta) ends at 65504, beyond which gradients are not finite, as beyond a loss scale's
// range.  dq by query tiles, then dK and dV by key tiles, which repeats S and dP (2 of 7 products) and needs no
// atomics: the same bits every time.
//
// Bound (fp16, 4 x 16 sequences of 2000 to 4096 rows of 128, windows of 1024, a warm card): dq 184 us, 37% of the
// matrix cores and 43% of the VALU; dK / dV 259 us, 33% and 39%, with 37% of LDS: its 16 keys a wave take a fragment
// from LDS for each product.  32 keys a wave halve that and leave one wave a SIMD (404 us for 318 side by side).
// At D = 256 dK / dV spill 12 registers with two waves a SIMD, 100 us for 8 x 8 x 300 to 1024 rows with windows of
// 511 (one wave a SIMD and no spills: 5% more).
// ---------------------------------------------------------------------------
template <int D>
struct BwdCfg {
  static constexpr int QB = D == 128 ? 2 : 1;   // dq: 16-row blocks of a wave
  static constexpr int BQ = kNW * QB * 16;
  static constexpr int QS = D == 256 ? 32 : 64;  // dK / dV: query rows of a step
  static constexpr int BK = tile_keys(D), NKB = BK / 16, NKS = BK / 32;  // dq: keys of a tile
  static constexpr int TILEB = BK * D * 2;
  static constexpr int DQ_LDS = 4 * TILEB;
  static constexpr int STEPB = QS * D * 2;
  static constexpr int SB = 2 * STEPB + 2 * QS * 4;  // a step: q rows, do rows, lse, delta
  static constexpr int DKV_LDS = 2 * SB;
  static constexpr int KC = D / 32, NDB = D / 16;
};

template <typename T>
FMLM_DEV void zero_row4(void* base, int64_t elem) {
  *(u32x2*)((char*)base + elem * 2) = u32x2{0u, 0u};
}

// dS in two terms of the type for the rows of a workgroup of which one sees few keys.  Three roundings are dq's error:
// its own, dS's, and that of the forward's P in delta, which grows with the weight of single keys (sum P^2 of dS's square).
// With one term the error is 1.44 times that of dq's own rounding over hundreds of keys, 1.48 over 64 and 1.50 to
// 1.53 below 16; two leave 1.04 to 1.14.  They cost a third of the products: the whole backward of 4 x 16 x 4096 rows of
// 128 takes 223 us for 220 with windows of 9 keys, 247 : 241 with 128, and would take 299 : 289 with 257, 609 : 576 with
// 1025; 8 x 8 x 1024 rows of 256 169 : 167 with 201, and 218 : 211 with 511.
constexpr int kTwoTermKeys = 256;
// keys that the row at position r sees, of a call without a context
FMLM_DEV int row_keys(const WinArgs& a, const WinSeq& s, int r) {
  const int lo = max(0, r - a.left);
  return min(s.len, r + a.right + 1) - lo + min(a.sinks, lo);
}

template <typename T, int D>
__global__ __launch_bounds__(kNW * 64, 2) void window_dq_kernel(const fmlm_attn_params p, const WinArgs a,
                                                                             const fmlm_attn_grads gr) {
  typedef BwdCfg<D> C;
  typedef typename Mfma<T>::v8 v8;
  constexpr int QB = C::QB, BK = C::BK, NKB = C::NKB, NKS = C::NKS;
  extern __shared__ __align__(16) char smem[];
  auto kbuf = [&](int i) { return smem + i * C::TILEB; };
  auto vbuf = [&](int i) { return smem + (2 + i) * C::TILEB; };
  int g, part, tile;
  if (!win_unit(p, a, 1, g, part, tile)) return;
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
  const WinTiles wt = win_tiles(a, s, row0, row0 + rows - 1, BK == 64 ? 6 : 5);
  const WTile<T, D> tr(l16, gq);
  const bool active = wave * QB * 16 < rows;
  // (a scale of 0 would lose the masked scores' infinity; this one leaves every other 2^(c s) at 1)
  const float c = p.scale != 0.f ? p.scale * kLog2e : 1e-30f;

  auto keys_in = [&](int t) { return min(BK, s.total - t * BK); };
  auto issue = [&](int v) {
    const int t = wt.tile(v), buf = v & 1, last = keys_in(t) - 1;
    WTile<T, D>::template load<BK>((const char*)p.k + row_at(p.kv_layout, s.b, s.h, s.q0, t * BK, p.k_sb, p.k_sh, p.k_sn) * 2,
                                    (uint32_t)p.k_sn * 2u, last, lds_addr(kbuf(buf)), wave, lane);
    WTile<T, D>::template load<BK>((const char*)p.v + row_at(p.kv_layout, s.b, s.h, s.q0, t * BK, p.v_sb, p.v_sh, p.v_sn) * 2,
                                    (uint32_t)p.v_sn * 2u, last, lds_addr(vbuf(buf)), wave, lane);
  };
  if (wt.n > 0) issue(0);
  v8 qf[QB][C::KC], df[QB][C::KC];
  float delta[QB], lse[QB], rest[QB];
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
      const v8 ov = ld_frag<T>(p.o, oo + col, ok), lv = ld_frag<T>(a.o_low, oo + col, ok && a.o_low);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf((float)df[qb][kc][e], (float)ov[e] + (float)lv[e], sum);
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    delta[qb] = sum;
    lse[qb] = ok ? p.lse[(int64_t)s.h * p.total_q + s.q0 + row0 + row] : INFINITY;
    rest[qb] = 0.f;
  }
  f32x4 dq[C::NDB][QB];
#pragma unroll
  for (int db = 0; db < C::NDB; ++db)
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) dq[db][qb] = f32x4{0.f, 0.f, 0.f, 0.f};
  // (a workgroup's own loop for each, not a branch in it)
  auto walk = [&](auto two) {
  constexpr bool TWO = decltype(two)::value;
  for (int v = 0; v < wt.n; ++v) {
    const int t = wt.tile(v), buf = v & 1, nk = keys_in(t);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (v + 1 < wt.n) issue(v + 1);
    const int kp = t * BK, w0 = row0 + wave * QB * 16, w1 = min(w0 + QB * 16, row0 + rows) - 1;
    if (!active || kp > w1 + a.right || (kp + BK <= w0 - a.left && kp >= a.sinks)) continue;  // none in view
    const char *kt = kbuf(buf), *vt = vbuf(buf);
    // ---- fenced slots, each the MFMAs of one LDS fragment: NSS of S^T (step kc, key block kb), NSS of
    // dP^T (block by block), 2 NDB of dq^T; the fragment of slot s + LEAD is read at slot s.  Block
    // kb's P and dS are made beside block kb + 1's dP, the last one's beside the first dq slots.
    constexpr int NSS = NKB * C::KC, NR = 2 * NSS, NS = NR + NKS * C::NDB, LEAD = 3;
    f32x4 sc[NKB][QB], dp[NKB][QB];
    u32x4 ds[NKS][QB], ds2[TWO ? NKS : 1][TWO ? QB : 1];
    v8 fr[LEAD + 1];
    auto read = [&](int r) {
      if (r < NSS) fr[r % (LEAD + 1)] = tr.row(kt, r % NKB, r / NKB);
      else if (r < NR) fr[r % (LEAD + 1)] = tr.row(vt, (r - NSS) / C::KC, (r - NSS) % C::KC);
      else fr[r % (LEAD + 1)] = tr.col(kt, (r - NR) / C::NDB, (r - NR) % C::NDB);
    };
    // elements r, r + 1 of block kb, rows qb (e = 2 qb + r / 2)
    auto soft = [&](int kb, int e) {
      const int qb = e >> 1, r = (e & 1) * 2;
      if (r == 0) pin(dp[kb][qb]);
      const float x = fast_exp2(fmaf(sc[kb][qb][r], c, -lse[qb])) * dp[kb][qb][r];
      const float y = fast_exp2(fmaf(sc[kb][qb][r + 1], c, -lse[qb])) * dp[kb][qb][r + 1];
      rest[qb] += x + y;
      uint32_t w = pack2<T>(x, y);
      pin(w);
      ds[kb >> 1][qb][(kb & 1) * 2 + (r >> 1)] = w;
      if constexpr (TWO) {
        uint32_t w2 = pack2<T>(x - (float)__builtin_bit_cast(T, (uint16_t)w), y - (float)__builtin_bit_cast(T, (uint16_t)(w >> 16)));
        pin(w2);
        ds2[kb >> 1][qb][(kb & 1) * 2 + (r >> 1)] = w2;
      }
    };
#pragma unroll
    for (int r = 0; r < LEAD; ++r) read(r);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int sl = 0; sl < NSS; ++sl) {
      read(sl + LEAD);
      const v8 x = fr[sl % (LEAD + 1)];
      const int kb = sl % NKB, kc = sl / NKB;
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
        sc[kb][qb] = Mfma<T>::run(x, qf[qb][kc], kc == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sc[kb][qb]);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (nk < BK || kp + BK - 1 > w0 + a.right || (kp < w1 - a.left && kp + BK > a.sinks)) {
      asm volatile("");  // (a real branch.)  What a row does not see: P = 0
      const float none = c < 0.f ? INFINITY : -INFINITY;
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        const int pos = w0 + qb * 16 + l16, k0 = kp + 4 * gq;
        const InView view(pos - a.left - k0, min(pos + a.right - k0, nk - 1 - 4 * gq), a.sinks - k0);
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[kb][qb][r] = view.pick(kb, r, sc[kb][qb][r], none);
      }
    }
#pragma unroll
    for (int sl = NSS; sl < NR; ++sl) {
      read(sl + LEAD);
      const v8 x = fr[sl % (LEAD + 1)];
      const int j = sl - NSS, kb = j / C::KC, kc = j % C::KC;
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
        dp[kb][qb] = Mfma<T>::run(x, df[qb][kc], kc == 0 ? f32x4{-delta[qb], -delta[qb], -delta[qb], -delta[qb]} : dp[kb][qb]);
      if (kb > 0) {
#pragma unroll
        for (int e = kc * 2 * QB / C::KC; e < (kc + 1) * 2 * QB / C::KC; ++e) soft(kb - 1, e);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(2);
#pragma unroll
    for (int sl = NR; sl < NS; ++sl) {
      if (sl + LEAD < NS) read(sl + LEAD);
      const v8 x = fr[sl % (LEAD + 1)];
      const int j = sl - NR, ks = j / C::NDB, db = j % C::NDB;
      if (NKS == 1 ? j == 0 : ks == 0) {  // the last block's (with one key step, before its products)
#pragma unroll
        for (int e = NKS == 1 ? 0 : j * 2 * QB / C::NDB; e < (NKS == 1 ? 2 * QB : (j + 1) * 2 * QB / C::NDB); ++e) soft(NKB - 1, e);
      }
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        dq[db][qb] = Mfma<T>::run(x, __builtin_bit_cast(v8, ds[ks][qb]), dq[db][qb]);
        if constexpr (TWO) dq[db][qb] = Mfma<T>::run(x, __builtin_bit_cast(v8, ds2[ks][qb]), dq[db][qb]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
  }
  };
  if (min(row_keys(a, s, row0), row_keys(a, s, row0 + rows - 1)) <= kTwoTermKeys) walk(std::true_type{});
  else walk(std::false_type{});
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int row = (wave * QB + qb) * 16 + l16;
    rest[qb] += __shfl_xor(rest[qb], 16);
    rest[qb] += __shfl_xor(rest[qb], 32);
    if (row >= rows) continue;
    // dS' = P (dP - delta') sums to delta - delta' over a row's keys: delta without the rounding of the forward's P
    if (gq == 0) ((float*)gr.workspace)[(int64_t)s.h * p.total_q + s.q0 + row0 + row] = delta[qb] + rest[qb];
    const int64_t off = row_at(p.q_layout, s.b, s.h, s.q0, row0 + row, gr.dq_sb, gr.dq_sh, gr.dq_sn);
#pragma unroll
    for (int db = 0; db < C::NDB; ++db) {
      const f32x4 x = dq[db][qb] * p.scale;
      *(u32x2*)((char*)gr.dq + (off + db * 16 + gq * 4) * 2) = u32x2{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
    }
  }
}

template <typename T, int D>
__global__ __launch_bounds__(kNW * 64, 2) void window_dkv_kernel(const fmlm_attn_params p, const WinArgs a,
                                                                              const fmlm_attn_grads gr) {
  typedef BwdCfg<D> C;
  typedef typename Mfma<T>::v8 v8;
  constexpr int QS = C::QS, NRB = QS / 16;
  extern __shared__ __align__(16) char smem[];
  auto qbuf = [&](int i) { return smem + i * C::SB; };
  auto obuf = [&](int i) { return smem + i * C::SB + C::STEPB; };
  auto stat = [&](int i) { return (float*)(smem + i * C::SB + 2 * C::STEPB); };
  int g, part, tile;
  if (!win_unit(p, a, 1, g, part, tile)) return;
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
  const float c = p.scale != 0.f ? p.scale * kLog2e : 1e-30f, none = c < 0.f ? INFINITY : -INFINITY;
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
    if (k0 >= s.len || k0 >= p0 + QS + a.right || (k1 < p0 - a.left && k0 >= a.sinks)) continue;  // none in view
    const bool edge = k1 >= s.len || k1 > p0 + a.right || (k0 < p0 + QS - 1 - a.left && k1 >= a.sinks);
    InView view;  // of the lane's key: rows key - right to key + left
    if (edge) {
      asm volatile("");  // (a real branch)
      view = InView(key - a.right - p0 - 4 * gq, (!kok ? -1 : key < a.sinks ? QS : key + a.left - p0) - 4 * gq, 0);
    }
    // ---- fenced slots as in the dq kernel: per block of 16 rows its S and dP (fragments of q and do in turn),
    // the block before's P and dS beside them; then per 32 rows dV^T and dK^T
    constexpr int RBS = 2 * C::KC, NR = NRB * RBS, NCS = 2 * C::NDB, NS = NR + NRB / 2 * NCS, LEAD = 3;
    f32x4 sc[NRB], dp[NRB], L4[NRB], D4[NRB];
    u32x4 pw[NRB / 2], dw[NRB / 2];
    v8 fr[LEAD + 1];
    auto read = [&](int r) {
      if (r < NR) fr[r % (LEAD + 1)] = tr.row((r & 1) ? ot : qt, r / RBS, (r % RBS) >> 1);
      else fr[r % (LEAD + 1)] = tr.col(((r - NR) & 1) ? qt : ot, (r - NR) / NCS, ((r - NR) % NCS) >> 1);
    };
    // a block whose scores are done: its statistics, and what does not see the key
    auto ready = [&](int rb) {
      L4[rb] = *(const f32x4*)(ls + rb * 16 + gq * 4);
      D4[rb] = *(const f32x4*)(ls + QS + rb * 16 + gq * 4);
      if (edge) {
        asm volatile("");  // (a real branch)
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[rb][r] = view.pick(rb, r, sc[rb][r], none);
      }
    };
    // elements 2 e, 2 e + 1 of block rb
    auto soft = [&](int rb, int e) {
      if (e == 0) {
        pin(sc[rb]);
        pin(dp[rb]);
      }
      float pv[2], dv2[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        pv[i] = fast_exp2(fmaf(sc[rb][2 * e + i], c, -L4[rb][2 * e + i]));
        dv2[i] = pv[i] * (dp[rb][2 * e + i] - D4[rb][2 * e + i]);
      }
      uint32_t x = pack2<T>(pv[0], pv[1]), y = pack2<T>(dv2[0], dv2[1]);
      pin(x);
      pin(y);
      pw[rb >> 1][(rb & 1) * 2 + e] = x;
      dw[rb >> 1][(rb & 1) * 2 + e] = y;
    };
#pragma unroll
    for (int r = 0; r < LEAD; ++r) read(r);
#pragma unroll
    for (int sl = 0; sl < NR; ++sl) {
      read(sl + LEAD);
      const v8 x = fr[sl % (LEAD + 1)];
      const int rb = sl / RBS, kc = (sl % RBS) >> 1, loc = sl % RBS;
      if (rb > 0 && loc == 0) ready(rb - 1);
      if ((sl & 1) == 0) sc[rb] = Mfma<T>::run(x, kf[kc], kc == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sc[rb]);
      else dp[rb] = Mfma<T>::run(x, vf[kc], kc == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : dp[rb]);
      if (rb > 0) {
#pragma unroll
        for (int e = loc * 2 / RBS; e < (loc + 1) * 2 / RBS; ++e) soft(rb - 1, e);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int sl = NR; sl < NS; ++sl) {
      if (sl + LEAD < NS) read(sl + LEAD);
      const v8 x = fr[sl % (LEAD + 1)];
      const int j = sl - NR, grp = j / NCS, db = (j % NCS) >> 1;
      if (j == 0) ready(NRB - 1);
      if (NRB == 2 ? j == 0 : grp == 0) {  // the last block's (with one group, before its products)
#pragma unroll
        for (int e = NRB == 2 ? 0 : j * 2 / NCS; e < (NRB == 2 ? 2 : (j + 1) * 2 / NCS); ++e) soft(NRB - 1, e);
      }
      if ((j & 1) == 0) dv[db] = Mfma<T>::run(x, __builtin_bit_cast(v8, pw[grp]), dv[db]);
      else dk[db] = Mfma<T>::run(x, __builtin_bit_cast(v8, dw[grp]), dk[db]);
      __builtin_amdgcn_sched_barrier(0);
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
// A kernel's LDS beyond 64 KB has to be allowed, once a device (2 us a call); `done`: the devices where it is
int allow_lds(const void* fn, int bytes, std::atomic<uint64_t>& done) {
  if (bytes <= 65536) return 0;
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return (int)e;
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return 0;
  e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) return (int)e;
  if (dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
  return 0;
}

dim3 grid_of(int64_t blocks, unsigned y = 1) {  // win_unit's
  return dim3((unsigned)std::min<int64_t>(blocks, kGridX), y, (unsigned)((blocks + kGridX - 1) / kGridX));
}

int longest(const fmlm_attn_params& p) { return p.N > 0 && p.N < p.total_q ? p.N : p.total_q; }

int limit(int x) { return x < 0 || x >= kNoLimit ? kNoLimit - 2 : x; }

// keys that `rows` neighbouring rows walk over, about (a packed context's batches are taken to have
// up to twice their average)
int64_t max_keys(const fmlm_attn_params& p, const fmlm_window& w, int rows) {
  int64_t keys = w.flags & FMLM_WINDOW_APPENDED ? 0 : longest(p);
  if (p.cu_seqlens_kv)
    keys += p.ctx_block_table ? (int64_t)p.ctx_pages_per_batch * FMLM_PAGE_ROWS
                              : std::min((int64_t)p.ctx_rows, 2 * (int64_t)p.ctx_rows / std::max(p.ctx_batch, 1));
  return std::min(keys, (int64_t)limit(w.left) + limit(w.right) + std::max(w.sinks, 0) + rows);
}

constexpr int kWideTiles = 9;
// calls whose key ranges stay whole: the backward reads a row's statistics from one workgroup
bool unsplit(const fmlm_attn_params& p, const fmlm_window& w) { return p.lse || w.o_low || (p.flags & FMLM_FLAG_NOSPLIT); }

struct FwdLaunch {
  const void* fn;
  const void* merge[2];  // by one row a workgroup, by as many as it has threads for
  int merge_rows;        // ... that many
  std::atomic<uint64_t>* allowed;
  int bq, lds, lg;  // rows of a workgroup, its LDS, log2 of a tile's keys
};
template <typename T, int D>
void merge_of(FwdLaunch& f) {
  f.merge_rows = 256 / (D / 8);
  f.merge[0] = (const void*)window_merge_kernel<T, D, 1>;
  f.merge[1] = (const void*)window_merge_kernel<T, D, 256 / (D / 8)>;
}
template <typename T, int D, int QB, bool FP4, bool LSE = false>
FwdLaunch fwd_of() {
  static std::atomic<uint64_t> allowed;
  FwdLaunch f;
  f.allowed = &allowed;
  f.fn = (const void*)window_fwd_kernel<T, D, QB, FP4, LSE>;
  merge_of<T, D>(f);
  f.bq = kNW * QB * 16;
  f.lds = FwdCfg<D, FP4>::LDS;
  f.lg = tile_keys(D) == 64 ? 6 : 5;
  return f;
}
template <typename T, int D, int QB>
FwdLaunch fwd_of(bool fp4, bool lse) {
  return fp4 ? fwd_of<T, D, QB, true>() : lse ? fwd_of<T, D, QB, false, true>() : fwd_of<T, D, QB, false>();
}
template <typename T, int D>
FwdLaunch few_of() {
  static std::atomic<uint64_t> allowed;
  FwdLaunch f;
  f.allowed = &allowed;
  f.fn = (const void*)window_fp4_few_kernel<T, D>;
  merge_of<T, D>(f);
  f.bq = kFewRows;
  f.lds = FewCfg<D>::LDS;
  f.lg = 6;
  return f;
}
template <typename T>
FwdLaunch pick_fwd(const fmlm_attn_params& p, const fmlm_window& w) {
  const bool fp4 = w.flags & FMLM_WINDOW_FP4;
  if (fp4 && p.N > 0 && p.N <= kFewRows && !p.lse && !w.o_low) {
    switch (p.D) {
      case 32: return few_of<T, 32>();
      case 64: return few_of<T, 64>();
      case 128: return few_of<T, 128>();
      default: return few_of<T, 256>();
    }
  }
  const int64_t tiles = max_keys(p, w, 128) / kBK, units = (int64_t)p.B * p.H * ((longest(p) + 127) / 128);
  const bool tall = longest(p) > 64;
  // 128 rows that share a tile.  In 16 bits where its fragments are longest beside the rest (D = 128) and
  // such workgroups are two a CU, parts counted (us with 64 against 128 rows: 8 x 16 x 2048 rows, windows
  // of 100, 450 and 1200, 85 : 79, 135 : 115, 188 : 153, at D = 64 38 : 51, 63 : 74, 95 : 101; 2 x 16 x 512
  // rows 12 : 17; 256 rows over 511 of 8192 keys 14 : 18, over 16384 keys 75 : 54).
  const bool wide = !fp4 && tall && units * (unsplit(p, w) ? 1 : std::max<int64_t>(tiles / kMinPartTiles, 1)) >= kFill;
  // In 4 bits they share its conversion too: at every D, but for short walks, whose workgroups are all start
  // and end.  (us with 64 : 128 rows; 4 x 16 x 512 rows over 128, 512, 1024 and 4096 context keys: D = 128 26 : 34,
  // 37 : 40, 50 : 49, 134 : 99; D = 64 19 : 23, 26 : 28, 37 : 35, 100 : 72; D = 32 17 : 21, 24 : 25, 33 : 30, 87 : 61.  2 x 16 x
  // 2048 rows gain at all of them, D = 128 119 : 82 to 337 : 207, a few workgroups at none: 8 x 100 rows 13 : 16 to
  // 21 : 24.  So the border of 10 tiles, a call's own keys counted, is about right for 512 rows between 500 and
  // 1000 keys.)
  const bool wide4 = fp4 && tall && tiles > kWideTiles;
  const bool lse = p.lse;
  switch (p.D) {
    case 32: return wide4 ? fwd_of<T, 32, 2, true>() : fwd_of<T, 32, 1>(fp4, lse);
    case 64: return wide4 ? fwd_of<T, 64, 2, true>() : fwd_of<T, 64, 1>(fp4, lse);
    case 128: return wide || wide4 ? fwd_of<T, 128, 2>(fp4, lse) : fwd_of<T, 128, 1>(fp4, lse);
    default: return fwd_of<T, 256, 1>(fp4, lse);  // (two blocks of 16 rows spill)
  }
}
FwdLaunch pick_fwd(const fmlm_attn_params& p, const fmlm_window& w) {
  return p.dtype == FMLM_DTYPE_BF16 ? pick_fwd<bf16>(p, w) : pick_fwd<f16>(p, w);
}

bool row_ok(const void* base, int64_t sb, int64_t sh, int64_t sn) {
  return base && (uint64_t)base % 16 == 0 && sb % 8 == 0 && sh % 8 == 0 && sn % 8 == 0 && sn >= 0 && sn < (1 << 22);
}

int check_window(const fmlm_attn_params& p, const fmlm_window& w) {
  if (p.dtype != FMLM_DTYPE_BF16 && p.dtype != FMLM_DTYPE_F16) return FMLM_E_DTYPE;
  if (p.D != 32 && p.D != 64 && p.D != 128 && p.D != 256) return FMLM_E_HEAD_DIM;
  if (p.flags & ~FMLM_FLAG_NOSPLIT) return FMLM_E_ARG;
  if (w.flags & ~(FMLM_WINDOW_APPENDED | FMLM_WINDOW_FP4)) return FMLM_E_ARG;
  if (p.B < 0 || p.H < 0 || p.N < 0 || p.total_q < 0 || p.total_q >= kNoLimit) return FMLM_E_ARG;
  if (p.B == 0 || p.H == 0 || p.total_q == 0) return 0;
  if (!p.cu_seqlens_q || (int64_t)p.B * p.H > 0x7fffff00) return FMLM_E_ARG;
  if (!std::isfinite(p.scale)) return FMLM_E_ARG;  // (a mask is a score of -inf times it)
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
  if (w.o_low && (uint64_t)w.o_low % 16) return FMLM_E_ALIGN;
  if (!appended && (!row_ok(p.k, p.k_sb, p.k_sh, p.k_sn) || !row_ok(p.v, p.v_sb, p.v_sh, p.v_sn))) return FMLM_E_ALIGN;
  return 0;
}

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
  a.o_low = w.o_low;
  return a;
}

// Parts that key ranges are cut into at most, and a record's rows.  Parts until there are kFill workgroups,
// two a CU (us a call in 16 bits, with 256 / 512 / 1024: 2 x 64 rows, 8192 keys, D = 128, 34 / 36 / 47; 8
// single rows, D = 64, 66 / 52 / 53; 256 rows, D = 256, 88 / 68 / 97; the 512 against 256 and 1024 of
// 128-row tiles: 85 : 116 : 111), each with kMinPartTiles tiles; of few rows in 4 bits, where the four waves
// walk apart, with kFewTiles (16 rows, 8192 keys: 16.4 with 4, 13.8 with 8, 15.8 with 16).  Between 512 and 2048
// units of those, parts of 32 tiles even out sequences of different lengths and cost where all are as long, which
// is not known here (single rows of 16 heads of 128, whole : as planned; 512 to 8192 keys: 32 users 81 : 70, 48 103 :
// 99, 64 133 : 125, 96 178 : 178, 127 233 : 235; 8192 keys each 107 : 115, 157 : 161, 213 : 211, 295 : 306, 394 : 405; 4096
// each 53 : 62, 84 : 89, 113 : 113, 156 : 162, 210 : 221); smaller parts cost more (1024 keys, 32 users: 19 whole, 26 in two).
void plan_parts(const fmlm_attn_params& p, const fmlm_window& w, const FwdLaunch& f, WinArgs& a) {
  a.rec_rows = std::min(f.bq, longest(p));
  a.lg = f.lg;
  if (unsplit(p, w)) return;
  const int64_t units = (int64_t)p.B * p.H * a.tiles, tiles = (max_keys(p, w, f.bq) >> f.lg) + 2;
  int64_t want = (kFill + units - 1) / units;
  if (f.bq == kFewRows) {
    if (units >= kFill && units < 4 * kFill) want = std::min<int64_t>(4, tiles / (4 * kFewTiles));
    want = std::min(want, tiles / kFewTiles);
  }
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
  static std::atomic<uint64_t> allowed[2];
  int rc = allow_lds(dq, C::DQ_LDS, allowed[0]);
  if (!rc) rc = allow_lds(dkv, C::DKV_LDS, allowed[1]);
  if (rc) return rc;
  hipLaunchKernelGGL((window_dq_kernel<T, D>), grid_of((int64_t)a.tiles * a.groups), dim3(kNW * 64), C::DQ_LDS, s, p, a, g);
  hipLaunchKernelGGL((window_dkv_kernel<T, D>), grid_of((int64_t)b.tiles * b.groups), dim3(kNW * 64), C::DKV_LDS, s, p, b, g);
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
  const FwdLaunch f = pick_fwd(*pp, *ww);
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
  const FwdLaunch f = pick_fwd(p, *ww);
  WinArgs a = win_args(p, *ww, f.bq);
  plan_parts(p, *ww, f, a);
  const int64_t need = record_bytes(p, a), blocks = (int64_t)a.tiles * a.groups * a.parts;
  if (need > 0 && (!p.workspace || p.workspace_bytes < need)) return FMLM_E_WORKSPACE;
  if (need > 0 && (uint64_t)p.workspace % 16) return FMLM_E_ALIGN;
  if (blocks > 0x7fffffff) return FMLM_E_ARG;
  a.records = (float*)p.workspace;
  p.flags = p.cu_seqlens_kv ? 0 : FMLM_FLAG_PREFILL;  // (without a context)
  rc = allow_lds(f.fn, f.lds, *f.allowed);
  if (rc) return rc;
  hipStream_t s = (hipStream_t)stream;
  void* args[2] = {&p, &a};
  hipError_t e = hipLaunchKernel(f.fn, grid_of(blocks), dim3(kNW * 64), args, f.lds, s);
  if (e != hipSuccess) return (int)e;
  if (a.parts > 1) {
    int bq = f.bq;
    void* margs[3] = {&p, &a, &bq};
    // few rows: a workgroup each, its threads share the parts
    const bool wide = a.rec_rows > 4;
    const int per = wide ? f.merge_rows : 1;
    e = hipLaunchKernel(f.merge[wide], grid_of((int64_t)a.tiles * a.groups, (a.rec_rows + per - 1) / per), dim3(256), margs, 0,
                        s);
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
