// qz_moe_walk.cuh -- how the warps of a CTA share the units of one phase of the
// expert layer: plain index arithmetic, no device call, so that it also compiles
// for the host.
#pragma once

#ifdef __CUDACC__
#define QZ_HD __host__ __device__ __forceinline__
#else
#define QZ_HD inline
#endif

namespace qz {

constexpr int kMoeWarps = 16;  // of a CTA
constexpr int kMoePiece = 4;   // chunks per bulk copy

// This warp's part of a phase: `whole` units of its own, kMoeWarps apart, then
// perhaps a share of one more.
struct MoeWalk {
  int group, unit;             // current group and unit in it
  int units, chunks;           // per group; per unit
  int left;                    // units after the current one
  int c, c0, c1;               // current chunk; this warp's chunks of the current unit
  int share, part;             // warps that share the last unit, this warp's place among them; 0: no last unit
  int last_group, last_unit;
  bool whole;                  // the current unit is this warp's alone
  bool met;                    // this warp has joined the others of the shared unit

  QZ_HD MoeWalk(const int* bound, int units_, int chunks_, int warp) : units(units_), chunks(chunks_) {
    const int begin = bound[0], end = bound[1];
    const int rounds = (end - begin) / kMoeWarps, rest = (end - begin) % kMoeWarps;
    share = rest ? kMoeWarps / rest : 1;
    share = share < 8 ? share : 8;
    share = share < chunks ? share : chunks;
    const int last = begin + rounds * kMoeWarps + warp / share;
    if (last < end) {
      part = warp % share;
      last_group = last / units;
      last_unit = last % units;
    } else {
      share = 0;
    }
    left = rounds + (share ? 1 : 0);
    whole = true;
    met = false;
    c0 = 0;
    c1 = chunks;
    group = (begin + warp) / units;
    unit = (begin + warp) % units;
    enter();
  }
  QZ_HD bool done() const { return left < 0; }
  // The warps of the last unit wait for each other without a limit, so each has to
  // join, also one that gave up in an earlier unit.
  QZ_HD bool owes_meeting() const { return share > 1 && !met; }
  QZ_HD void enter() {  // the next unit's first chunk
    if (--left == 0 && share) {
      whole = share == 1;
      group = last_group;
      unit = last_unit;
      c0 = part * chunks / share;
      c1 = (part + 1) * chunks / share;
    }
    c = c0;
  }
  QZ_HD int piece() const { return c1 - c < kMoePiece ? c1 - c : kMoePiece; }
  QZ_HD bool advance() {  // true: a new unit
    c += kMoePiece;
    if (c < c1) return false;
    unit += kMoeWarps;
    while (unit >= units) { unit -= units; ++group; }
    enter();
    return true;
  }
};

}  // namespace qz
