// What a wave of the MXFP4 tile kernel has in flight, as numbers: its loads into LDS, its stores and the counts that it
// waits with. Plain C++, so that a host program can replay a wave's operations against them.
#pragma once

namespace joy {

// vmcnt operations of one wave of a 64 FM x 64 FN tile with a ring of S slabs. They complete in order; a wait with count
// n leaves at most the n last ones in flight.
struct MxTileCounts {
  int fm, fn, ring;
  bool quant;  // MXFP4 output

  constexpr int a() const { return 2 * fm; }      // loads of a slab's A rows
  constexpr int w() const { return 2 * fn; }      // of its W rows
  constexpr int ws() const { return w() + 1; }    // and its scales
  constexpr int stores() const {                  // of a tile's epilogue, at least
    return fm * (quant ? (fn + 1) / 2 + (fn == 3 ? 3 : 1) : fn * 2);
  }
  // Before a slab's second phase the next slab is read from LDS. Behind its loads lie the A rows of the slabs from the
  // next but one on to the one S ahead, and the W rows and scales of all of these but the last.
  constexpr int next_slab() const { return (ring - 1) * a() + (ring - 2) * ws(); }
  // The same in a tile's first slab: the last epilogue's stores lie there too.
  constexpr int next_slab_first() const { return next_slab() + stores(); }
  // Before an epilogue that follows its tile's only slab. The tile's bias and gate were loaded in the second phase of the
  // last tile's first slab, in front of that phase's W rows and scales; behind those lie the last epilogue's stores, this
  // slab's A rows, the next tile's bias or gate, W rows and scales. With more slabs a tile, the wait of the second covers
  // the bias and gate for any ring, and with a ring of two that of the first: a whole slab's loads lie behind them.
  constexpr int side() const { return ws() + stores() + a() + 1 + ws(); }
  // Whether that wait is needed: it is not where the only slab's own wait, a + ws + stores operations behind the bias and
  // gate, counts no more than these.
  constexpr bool side_waits() const { return next_slab_first() > ws() + stores() + a(); }
};

// The loads of a workgroup's tiles first, first + P, ... below count as one stream of slabs, nk a tile: next() goes on by
// one and says whether the tile has changed. Past the last tile the stream goes on with slabs that fetch nothing, from an
// empty buffer range at offset 0: only against a range that holds them are scalar offsets sure to count as inside or
// outside (an unsigned range minus offset would wrap).
struct MxLoadStream {
  int tile, slab = 0;
  int k_off;       // the slab's bytes into a row
  unsigned s_off;  // and into the scales (a whole tile's may pass 2^31)

  constexpr MxLoadStream(int first, int row_bytes, int slab_stride)
      : tile(first), k_off(-row_bytes), s_off(0u - (unsigned)slab_stride) {}
  constexpr bool next(int nk, int P, int count, int row_bytes, int slab_stride) {
    k_off += row_bytes, s_off += (unsigned)slab_stride;
    if (slab++ != nk) return false;
    tile += P;
    slab = tile < count ? 1 : nk;  // behind the last tile every slab is as its first
    k_off = 0, s_off = 0;
    return true;
  }
};

// First column that the loads of a tile at column n0 take: column 0 where the tile lies behind N (the last 192-column tile
// of MXFP4 output may), whose results are not stored, so that its range of W holds every offset too.
constexpr int mx_load_column(int n0, int N) { return n0 < N ? n0 : 0; }

}  // namespace joy
