// kv4_walk.h — which stages of a call each attention block works on (kv4.cu).
//
// A unit of work is one row group of one key/value head.  Units are numbered (entry,
// row group, head); their stages of a.keys keys, each unit's after a.pad places for what
// a unit costs besides, make one flat range that the blocks share evenly.
//
// `A`: the call's sizes (c.batch, c.heads, n_tokens, group, rows, n_rows, row_groups,
// keys, pad, splits) and len(b), an entry's length clamped to its cache.  The lengths are
// read again at every unit, by each warp for itself.  They must not change in between;
// if they do, results are lost but every loop here ends, and every unit, stage and
// block that it yields exists.  Plain C++, so that this can be shown on the CPU.
#pragma once

#ifdef __CUDACC__
#define MRI_WALK __device__ __forceinline__
#else
#define MRI_WALK inline
#endif

namespace mri {
namespace kv4 {

struct Unit {
  int b, rg, h;
  int tiles;  // places of this unit, its stages last
  int end;    // its last stage + 1, counted from the block's first stage
};

// The end of the unit after the last one, past every block's stages (below 2^32 in all,
// and shared by all SMs where there are more than a few).
constexpr int kPastUnits = 1 << 30;

MRI_WALK int lesser(int a, int b) { return a < b ? a : b; }
MRI_WALK int greater(int a, int b) { return a < b ? b : a; }

// What a unit counts in the flat range: the stages of its row group (up to the last key its
// last row sees, at least one: rows that see nothing are written too) after a.pad places.
template <typename A>
MRI_WALK int unit_tiles(const A& a, int b, int rg) {
  const int last = lesser((rg + 1) * a.n_rows, a.rows) - 1;
  const int seen = a.len(b) - a.n_tokens + 1 + last / a.group;
  return a.pad + greater(1, (seen + a.keys - 1) / a.keys);
}

template <typename A>
MRI_WALK void next_unit(const A& a, Unit& u) {
  if (++u.h == a.c.heads) {
    u.h = 0;
    if (++u.rg == a.row_groups) {
      u.rg = 0;
      ++u.b;
    }
    if (u.b < a.c.batch) {
      u.tiles = unit_tiles(a, u.b, u.rg);
    } else {
      u.tiles = 0;
      u.end = kPastUnits;
    }
  }
  u.end += u.tiles;
}

struct Plan {
  unsigned total, x0;     // stages of the call (below 2^32); the block's first
  int count;              // stages of the block
  unsigned blocks;        // blocks with a share
  unsigned each, longer;  // a share's stages; the first `longer` blocks have one more
  Unit first;
};

// Block `block`'s share of `total` stages (at least one); a block has `least` of them before the
// next one is used.  Its first unit is none until find_first knows better.
template <typename A>
MRI_WALK void share_out(const A& a, unsigned total, unsigned block, unsigned grid, unsigned least, Plan& plan) {
  const unsigned wanted = total / least + (total % least != 0);
  const unsigned blocks = grid < wanted ? grid : wanted;
  plan.total = total;
  plan.blocks = blocks;
  plan.each = total / blocks;
  plan.longer = total % blocks;
  plan.x0 = block < blocks ? block * plan.each + (block < plan.longer ? block : plan.longer) : total;
  plan.count = block < blocks ? static_cast<int>(plan.each + (block < plan.longer)) : 0;
  plan.first = Unit{a.c.batch, 0, 0, 0, kPastUnits};
}

// The unit that holds flat stage x0, if it is one of (entry, row group) pairs p0 to
// p1 - 1, whose stages begin at flat stage `before`.
template <typename A>
MRI_WALK bool find_first(const A& a, unsigned x0, unsigned before, unsigned p0, unsigned p1, Unit& first) {
  const unsigned groups = static_cast<unsigned>(a.row_groups), heads = static_cast<unsigned>(a.c.heads);
#ifdef __CUDACC__
#pragma unroll 1
#endif
  for (unsigned p = p0; p < p1; ++p) {
    const int b = static_cast<int>(p / groups), rg = static_cast<int>(p % groups);
    const unsigned tiles = static_cast<unsigned>(unit_tiles(a, b, rg));
    if (x0 - before < tiles * heads) {
      const unsigned h = (x0 - before) / tiles;
      first = Unit{b, rg, static_cast<int>(h), static_cast<int>(tiles), static_cast<int>((h + 1) * tiles - (x0 - before))};
      return true;
    }
    before += tiles * heads;
  }
  return false;
}

// The block whose share holds flat stage x.
MRI_WALK int owner_of(const Plan& p, unsigned x) {
  const unsigned edge = p.longer * (p.each + 1);
  const unsigned c = x < edge ? x / (p.each + 1) : p.longer + (x - edge) / p.each;
  return static_cast<int>(c < p.blocks ? c : p.blocks - 1);
}

// The first stage at or after `next` of the ring that takes every a.splits-th stage of the
// block, with the unit it belongs to in v; `count` or more if there is none.
template <typename A>
MRI_WALK int seek_stage(const A& a, Unit& v, int next, int count) {
  while (next < count) {
    while (next >= v.end) next_unit(a, v);
    const int first = v.end - v.tiles + a.pad;
    if (next >= first) break;
    next += (first - next + a.splits - 1) / a.splits * a.splits;
  }
  return next;
}

// Brings x and u to the block's next stage.  Its unit's stages begin at unit_begin and this
// block has [x, seg_end) of them.  False: there is none.
template <typename A>
MRI_WALK bool next_segment(const A& a, Unit& u, int& x, int count, int& unit_begin, int& seg_end) {
  while (x < count) {
    seg_end = lesser(u.end, count);
    unit_begin = u.end - u.tiles + a.pad;
    x = greater(x, unit_begin);
    if (x < seg_end) return true;
    x = seg_end;
    next_unit(a, u);
  }
  return false;
}

}  // namespace kv4
}  // namespace mri
