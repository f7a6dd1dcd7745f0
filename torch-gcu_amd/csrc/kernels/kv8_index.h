// Index arithmetic of the 8-bit key/value cache: which tokens, pages and parts
// a call touches.  Plain C++ that runs on the host as well, where the tests
// feed it lengths, starts and tables that no caller should pass: whatever the
// device tensors hold, every index that comes out of here is in bounds.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define MI_HD __host__ __device__ __forceinline__
#else
#define MI_HD inline
#endif

namespace mi {

// Sequence b of a call: its new tokens (rows first .. first + n - 1 of the
// packed tensors) and the tokens that the cache holds of it, the new ones
// among them.  A length outside [0, cap] makes the sequence empty (len 0) and
// is reported; starts are clamped into [0, tokens] and never run backwards.
struct Kv8Seq {
  int first;
  int n;
  int len;
  bool bad;
};

MI_HD int kv8_clamp(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

MI_HD Kv8Seq kv8_seq(int start, int next, int length, int tokens, int cap) {
  Kv8Seq s;
  s.first = kv8_clamp(start, 0, tokens);
  s.n = kv8_clamp(next, s.first, tokens) - s.first;
  s.bad = length < 0 || length > cap;
  s.len = s.bad ? 0 : length;
  return s;
}

// The page that a table entry names, or -1 if the cache has no such page.
MI_HD int kv8_page(int entry, int pages) { return entry >= 0 && entry < pages ? entry : -1; }

// Where the 16 keys from `pos` (a multiple of 16) on are loaded from: their own
// place, or behind the end of a sequence of `len` >= 1 the place of its last 16.
// Pages hold a multiple of 16, so the 16 slots from the result on lie in one page,
// and that page is one of the sequence's.
MI_HD int kv8_group_at(int pos, int len) {
  const int last = (len - 1) & ~15;
  return pos < last ? pos : last;
}

// One past the last position that new token i of a sequence sees: its own
// position is len - n + i.  0 when nothing is visible.
MI_HD int kv8_limit(const Kv8Seq& s, int i) {
  const int64_t at = (int64_t)s.len - s.n + i + 1;
  return at < 0 ? 0 : at > s.len ? s.len : (int)at;
}

// How a sequence's work is cut: its rows (new tokens x heads of a group, the
// token outermost) into tiles of rt, its keys into tiles of kt of which a part
// takes about `chunk`.  A sequence with rows but no keys keeps one part, which
// writes its empty rows.
struct Kv8Cut {
  int rows;       // n * group
  int row_tiles;
  int key_tiles;
  MI_HD float work() const { return (float)row_tiles * (float)key_tiles; }
  MI_HD int parts(int chunk) const { return key_tiles > chunk ? (key_tiles + chunk - 1) / chunk : 1; }
};

MI_HD Kv8Cut kv8_cut(const Kv8Seq& s, int group, int rt, int kt) {
  Kv8Cut c;
  c.rows = s.n * group;  // the host checked that tokens * group fits 31 bits
  c.row_tiles = (c.rows + rt - 1) / rt;
  c.key_tiles = (int)(((int64_t)s.len + kt - 1) / kt);
  return c;
}

// Row tiles of up to 64 sequences by how far their last tokens see, the farthest
// first: round k takes of each sequence the tile whose end lies about k tiles'
// tokens before the longest sequence's end, if it has one.
struct Kv8Rounds {
  int off;    // the round of the sequence's last tile
  int tiles;
  MI_HD Kv8Rounds(const Kv8Seq& s, const Kv8Cut& c, int longest, int group, int rt) {
    const int step = rt / group > 1 ? rt / group : 1;  // tokens of a row tile
    tiles = c.row_tiles;
    off = tiles > 0 ? (longest - s.len) / step : 0;
  }
  MI_HD int before(int k) const { return kv8_clamp(k - off, 0, tiles); }  // tiles in rounds 0 .. k - 1
  MI_HD bool in(int k) const { return k >= off && k - off < tiles; }
};

// How the key tiles of a call are cut into parts: `few` parts in all, or `many`
// where a part would be longer than `wide` tiles, none shorter than `least`.
struct Kv8Plan {
  int few, wide, least, many;  // few <= many
  // Key tiles a part takes.  work, of all sequences and k/v heads, is a float
  // sum, a few units of 2^-24 off, which the factor makes up for; the parts are
  // at most `many` more than the tiles of rows.
  MI_HD int chunk(float work) const {
    float c = work / (float)few * 1.00001f + 1.0f;
    if (c > (float)wide) c = work / (float)many * 1.00001f + 1.0f;
    return c < (float)least ? least : c > 1073741824.f ? 1073741824 : (int)c;
  }
};

// Row tiles that tokens x group rows in at most `seqs` sequences can make.
MI_HD int64_t kv8_row_tiles_most(int64_t tokens, int64_t seqs, int64_t group, int rt) {
  const int64_t some = seqs < tokens ? seqs : tokens;
  return (tokens * group + some * (rt - 1)) / rt;
}

// Pages that a sequence's new tokens fall into, and the most for a whole call.
MI_HD int kv8_touched(const Kv8Seq& s, int shift) {
  if (s.n == 0 || s.n > s.len) return 0;
  return ((s.len - 1) >> shift) - ((s.len - s.n) >> shift) + 1;
}
MI_HD int64_t kv8_touched_most(int64_t tokens, int64_t seqs, int shift) {
  const int64_t some = seqs < tokens ? seqs : tokens;
  return (tokens >> shift) + 2 * some;
}

// The scale of a block whose largest finite magnitude is amax: the smallest
// power of two s >= 2^-110 with amax <= 448 s (448 is the largest e4m3 number).
// amax = m 2^e with m in [1, 2), 448 = 1.75 * 2^8.
MI_HD float kv8_scale_of(float amax) {
  uint32_t u;
  __builtin_memcpy(&u, &amax, 4);
  int e = (int)(u >> 23) - 127 - 8;
  if ((u & 0x7fffffu) > 0x600000u) ++e;
  if (e < -110) e = -110;
  u = (uint32_t)(e + 127) << 23;
  float s;
  __builtin_memcpy(&s, &u, 4);
  return s;
}

}  // namespace mi
