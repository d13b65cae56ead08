// How a call of the linear cross-entropy (linear_xent.hip) divides: its tiles,
// its scratch, the parts of the classes and the shares of dX's K.  Plain
// arithmetic of the sizes, so that it can be checked without a device.
#pragma once

#include <algorithm>
#include <cstdint>

namespace aicf::hip {

inline int64_t lx_up_to(int64_t n, int64_t step) { return (n + step - 1) / step * step; }

// K of a share: whole K-steps of every type.
constexpr int lx_share_k(int k, int shares) { return ((k + shares - 1) / shares + 63) / 64 * 64; }
// Shares that k classes fill, and so slabs that they leave.
constexpr int lx_slabs(int k, int share_k) { return (k + share_k - 1) / share_k; }

// Rows of a product's tiles.  16-bit: 256 (256 x 256) where those fill three
// quarters of the CUs, else 128, for few rows 64 or 32.  f32 is bound by its
// MFMAs, so by the CU with most tiles: 64 x 64 unless 128 x 128 give it no more.
inline int lx_tile_rows(int64_t rows, int64_t cols, bool f32) {
  if (rows <= 32) return 32;
  auto tiles = [&](int64_t n) { return ((rows + n - 1) / n) * ((cols + n - 1) / n); };
  if (f32) return (tiles(64) + 255) / 256 < 4 * ((tiles(128) + 255) / 256) ? 64 : 128;
  if (rows <= 64) return 64;
  return rows <= 128 || tiles(256) < 192 ? 128 : 256;
}
// Their columns, and how many of them run on the chip at once (by LDS).
inline int lx_tile_cols(int bm, bool f32) { return bm == 256 ? 256 : bm == 64 && f32 ? 64 : 128; }
inline int lx_slots(int bm, bool f32) { return 256 * (f32 ? (bm == 128 ? 2 : 4) : bm == 128 || bm == 32 ? 2 : 1); }

struct LxPlan {
  int64_t Rp, Dp, Vp, es;
  int bm, bn;               // tiles of the logits
  bool direct;              // W is read in place
  int64_t piece;            // classes of a piece (a multiple of 256)
  int64_t held;             // classes whose G is held in dW first (a multiple of 256)
  int bm_dx;                // tiles of dX
  int64_t slab_rows;        // of all its slabs together
  int64_t stats_off, xc_off, slab_off, wpad_off, g_off, bytes;
};

constexpr int kRowArrays = 8;  // arrays of Rp 4-byte values behind the head

// Work-items of a launch lie below 2^32, and all but the logits' 256 x 256 tiles
// of eight waves, which loop over their tiles, have a workgroup of 256 for each.
constexpr int64_t kRowsEnd = (int64_t)1 << 26;  // a wave copies a row (of X, and of W)
inline bool lx_tiles_loop(int bm, bool f32, int64_t K) { return bm == 256 && !f32 && K < 2048; }
inline int64_t lx_most_tiles(bool loop) { return loop ? INT32_MAX - 1024 : ((int64_t)1 << 24) - 1; }

// The plan of a call, with the largest piece of at most `piece` classes that
// `bytes` of scratch hold (bytes < 0: any).  False: none fits.
inline bool lx_plan(int64_t R, int64_t V, int64_t D, int64_t ldw, bool direct, bool f32, bool grad, int64_t piece,
                    int64_t bytes, LxPlan* pl) {
  LxPlan p{};
  p.es = f32 ? 4 : 2;
  p.Rp = R > 0 ? lx_up_to(R, 256) : 256;
  p.Dp = lx_up_to(D, 64);
  p.Vp = lx_up_to(V, 256);
  p.direct = direct;
  p.bm = lx_tile_rows(R, V, f32);
  p.bn = lx_tile_cols(p.bm, f32);
  const int64_t lim = INT32_MAX;  // 32-bit offsets into an operand
  const int64_t ldk = direct ? ldw : p.Dp;
  if (p.Rp > lim / 2 || p.Dp * p.es * 256 >= lim || ldk * p.es * 256 >= lim || p.Vp > (int64_t)1 << 28) return false;
  // classes of a launch of the logits: all where W is read in place, else a piece
  const int64_t tile_rows = (std::max<int64_t>(R, 1) + p.bm - 1) / p.bm;
  const int64_t in_launch = lx_most_tiles(lx_tiles_loop(p.bm, f32, direct ? D : p.Dp)) / tile_rows * p.bn;
  if (p.Rp >= kRowsEnd || (direct && p.Vp > in_launch)) return false;
  int64_t at = 256 + kRowArrays * p.Rp * 4;
  p.stats_off = at;
  at = lx_up_to(at + p.Vp / p.bn * p.Rp * 8, 256);
  p.xc_off = at;
  at = lx_up_to(at + p.Rp * p.Dp * p.es, 256);
  p.slab_off = at;
  p.bm_dx = lx_tile_rows(R, D, f32);
  p.slab_rows = p.Rp + 4096;
  if (grad) {
    if (p.Rp * p.Dp * p.es >= lim) return false;
    at = lx_up_to(at + p.slab_rows * p.Dp * 4, 256);
  }
  p.wpad_off = at;
  // a piece: its G (with gradients) and its rows of W (where they are copied)
  const int64_t each = (grad ? p.Rp * p.es : 0) + (direct ? 0 : p.Dp * p.es);
  int64_t most = piece > 0 && piece < p.Vp ? lx_up_to(piece, 256) : p.Vp;
  if (grad) {
    most = std::min(most, (lim - 1) / (p.Rp * p.es) / 256 * 256);
    most = std::min(most, (lim - 1) / (ldk * p.es) / 256 * 256);
  }
  if (!direct) most = std::min({most, in_launch / 256 * 256, kRowsEnd - 256});
  if (bytes >= 0 && each > 0) most = std::min(most, (bytes - at - 256) / each / 256 * 256);
  if (most < 256) return false;
  p.piece = most;
  p.g_off = lx_up_to(at + (direct ? 0 : most * p.Dp * p.es), 256);
  p.bytes = p.g_off + (grad ? p.Rp * most * p.es : 0) + 256;  // (the start is rounded up to 256 bytes)
  if (bytes >= 0 && p.bytes > bytes) return false;
  if (grad && bytes > p.bytes) {  // what is left: more slabs, behind everything else
    const int64_t room = (bytes - p.g_off - p.Rp * most * p.es - 256) / (p.Dp * 4);
    if (room > p.slab_rows) {
      p.slab_rows = std::min<int64_t>(room, 8 * p.Rp + 4096);
      p.slab_off = p.g_off + p.Rp * most * p.es;
    }
  }
  if (pl) *pl = p;
  return true;
}

// Classes [0, held) whose G fits in the rows [held, V) of a contiguous dW of
// elements of ob bytes, where scratch does not hold all.
inline int64_t lx_held(const LxPlan& pl, int64_t V, int64_t D, int64_t ldw, int64_t ob) {
  if (pl.piece >= pl.Vp) return 0;
  const int64_t lim = INT32_MAX - 1;
  int64_t n = std::min(pl.Vp - pl.piece, (V * D * ob - 256) / (pl.Rp * pl.es + D * ob));
  n = std::min({n, lim / (pl.Rp * pl.es), lim / ((pl.direct ? ldw : pl.Dp) * pl.es)});
  if (!pl.direct) n = std::min(n, pl.piece);  // (room for the copy of W's rows)
  return n > 0 ? n / 256 * 256 : 0;
}

// The parts of the classes in the order in which their G is used: [0, held),
// which dW's rows hold until then; the last classes, whose G waits in scratch;
// the others, whose logits are computed again and whose G takes its place.
struct LxPart {
  int64_t v0, cols;
};
struct LxParts {
  int64_t V, held, last;  // the part in scratch is [last, V)
  int kept;               // parts whose G is kept from the first logits
  int64_t step, count;

  LxPart at(int64_t k) const {
    if (k == kept - 1) return {last, V - last};
    if (k < kept) return {0, held};
    const int64_t v0 = held + (k - kept) * step;
    return {v0, std::min(step, last - v0)};
  }
  // Classes of the longest part: what dX's shares divide, so that some part
  // writes each of their slabs.  (The part in scratch has fewer than a piece
  // where 256 does not divide V, and the others may have fewer still.)
  int64_t longest() const {
    int64_t n = 0;
    for (int64_t k = 0; k < std::min<int64_t>(count, kept + 1); ++k) n = std::max(n, at(k).cols);
    return n;
  }
};
inline LxParts lx_parts(const LxPlan& pl, int64_t V, bool grad) {
  LxParts q{};
  q.V = V;
  q.held = pl.held;
  q.last = grad ? std::max<int64_t>(pl.Vp - pl.piece, 0) : V;
  q.kept = grad ? (pl.held > 0 ? 2 : 1) : 0;
  q.step = std::min(pl.piece, V);
  q.count = q.kept + (q.last - q.held + q.step - 1) / q.step;
  return q;
}

}  // namespace aicf::hip
