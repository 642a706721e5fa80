// Replays what one wave of the MXFP4 tile kernel issues, waits for and reads, with the counts that the kernel waits with
// (csrc/mxfp4_schedule.hpp): every read of LDS has to lie behind a wait for its load and a barrier, every load into LDS
// behind a barrier that follows the last read of what it overwrites. The four waves do the same in step, each a share of
// the loads, so that one wave's wait before a barrier is every wave's. And where the stream of loads is: on the slabs of
// the workgroup's tiles in turn, behind the last one at offset 0, at no time past a range.
//
// No arguments: the replay. Arguments fm fn ring quant: the count that the kernel waits with before the epilogue of a
// tile of one slab, -1 where no wait is needed there.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../joyai-video-edit_amd/csrc/mxfp4_schedule.hpp"

struct Wave {
  int issued = 0, done = 0, seen = 0, epoch = 0;
  bool ok = true;
  int issue() { return issued++; }
  void wait(int n) { done = issued - n > done ? issued - n : done; }
  void barrier() { seen = done, ++epoch; }
  void read(int op) { ok &= op < seen; }
};

struct Place {  // LDS that one load or group of loads fills
  int op = -1, read_at = -1;
  void load(Wave& w, int count) {
    w.ok &= read_at < w.epoch;
    for (int i = 0; i < count; ++i) op = w.issue();
  }
  void read(Wave& w) { w.read(op), read_at = w.epoch; }
};

// More operations than the counts say may be behind a load (a gated residual's rows), never fewer.
static bool replay(const joy::MxTileCounts& n, int nk, int tiles, bool residual) {
  Wave w;
  const int S = n.ring;
  std::vector<Place> a(S), ws(S);
  Place side[2];
  side[0].load(w, 1);
  for (int s = 0; s < S; ++s) a[s].load(w, n.a()), ws[s].load(w, n.ws());
  w.wait((S - 2) * (n.a() + n.ws()));
  w.barrier();
  a[0].read(w), ws[0].read(w);
  int g = 0;
  for (int t = 0; t < tiles; ++t) {
    for (int k = 0; k < nk; ++k, ++g) {
      const int slot = g % S, next = (g + 1) % S;
      ws[slot].read(w);  // the second half of its W units
      w.barrier();
      a[slot].load(w, n.a());
      w.wait(k == 0 ? n.next_slab_first() : n.next_slab());
      w.barrier();
      if (k == 0) side[(t + 1) & 1].load(w, 1);
      ws[next].read(w), a[next].read(w);
      ws[slot].load(w, n.ws());
    }
    if (n.side_waits() && nk == 1) w.wait(n.side()), w.barrier();
    side[t & 1].read(w);
    for (int i = 0; i < n.stores() * (residual ? 2 : 1); ++i) w.issue();
  }
  return w.ok;
}

static bool stream(int nk, int first, int P, int count, int slab_stride) {
  joy::MxLoadStream at = {first, 128, slab_stride};
  bool ok = true;
  for (int t = first; t < count; t += P)
    for (int k = 0; k < nk; ++k) {
      ok &= at.next(nk, P, count, 128, slab_stride) == (k == 0 && t != first);
      ok &= at.tile == t && at.k_off == 128 * k && at.s_off == (unsigned)slab_stride * (unsigned)k;
    }
  for (int i = 0; i < 4; ++i)  // a ring's slabs behind the last tile
    ok &= at.next(nk, P, count, 128, slab_stride) && at.tile >= count && at.k_off == 0 && at.s_off == 0;
  return ok;
}

int main(int argc, char** argv) {
  if (argc == 5) {
    const joy::MxTileCounts n = {atoi(argv[1]), atoi(argv[2]), atoi(argv[3]), atoi(argv[4]) != 0};
    printf("%d\n", n.side_waits() ? n.side() : -1);
    return 0;
  }
  int bad = 0, runs = 0;
  for (int fm = 1; fm <= 4; ++fm)
    for (int fn = 2; fn <= 4; ++fn)
      for (int ring = 2; ring <= 4; ++ring)
        for (int quant = 0; quant < 2; ++quant) {
          const joy::MxTileCounts n = {fm, fn, ring, quant != 0};
          if (n.next_slab_first() >= 64) continue;  // the kernel's static_assert refuses it
          if (n.side_waits() && n.side() >= 64) printf("wait count of %d x %d, ring %d\n", fm, fn, ring), ++bad;
          for (int nk = 1; nk <= 5; ++nk)
            for (int tiles = 1; tiles <= 5; ++tiles)
              for (int residual = 0; residual < 2 - quant; ++residual, ++runs)
                if (!replay(n, nk, tiles, residual))
                  printf("64 x %d rows, 64 x %d columns, ring of %d, %s output, %d slabs, %d tiles\n", fm, fn, ring,
                         quant ? "MXFP4" : "16-bit", nk, tiles), ++bad;
        }
  for (int nk = 1; nk <= 5; ++nk)
    for (int first = 0; first < 3; ++first)
      for (int P = 3; P <= 4; ++P)
        for (int count = first + 1; count <= 9; ++count)
          for (int stride : {8, 8 * 347, nk > 1 ? 0x7ffffff8 / (nk - 1) / 8 * 8 : 0x7ffffff8}) {  // the largest: 2^31 bytes in all
            ++runs;
            if (!stream(nk, first, P, count, stride))
              printf("stream of %d slabs, tiles %d, %d, ... below %d\n", nk, first, first + P, count), ++bad;
          }
  for (int N = 32; N <= 2048; N += 32)
    for (int n0 = 0; n0 < (N + 255) / 256 * 256; n0 += 192) {
      ++runs;
      const int c = joy::mx_load_column(n0, N);
      if (c >= N || (n0 < N && c != n0)) printf("column %d of %d: loads from %d\n", n0, N, c), ++bad;
    }
  printf("%d of %d\n", bad, runs);
  return bad != 0;
}
