// How the paged attention's line of items is cut: plain integers, for the kernel and for host code alike.
//
// Items (a request's 16 columns) stand one after the other, each on its tiles' places and a few more; workgroup w has
// the places [w * per, (w + 1) * per).  A stretch's end closer than kPiece tiles to an item's end moves there.
#pragma once

namespace paged {
constexpr int kPiece = 8;  // tiles of a cut item's piece, at least: one a wave

// where an end of a stretch, t places past an item's start, cuts the item's tiles
constexpr int cut_at(int t, int tiles) { return t < kPiece ? 0 : (tiles - t < kPiece ? tiles : t); }

// the workgroups that an item's first and last tiles go to
struct Parts {
  int first, last;
};
// `wgs` workgroups: an item whose length grew after the line was summed may reach past the line's end, what it is
// joined of may not
constexpr Parts parts_of(int start, int tiles, int per, int wgs) {
  const int end = start + tiles;
  int first = start / per, last = (end - 1) / per;
  if ((first + 1) * per - start < kPiece) ++first;
  if (end - last * per < kPiece) --last;
  return {first, last < wgs ? last : wgs - 1};
}
}  // namespace paged
