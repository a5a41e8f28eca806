// asmllm_b200/csrc/found.cuh -- records of where a unit's results are, from
// the passes of the decode attentions to their joins.
//
// A unit's tiles are cut over ranges; the range in which it begins leaves its
// record.  A join forms addresses from records alone, so that
//   * every unit has one, also where a wait has run out: abandon();
//   * what is no record of such a call (a workspace that another call writes
//     at the same time) has no parts: parts_of(), in_group().
// Plain C++, so that both can be run on a CPU.
#pragma once

#ifdef __CUDACC__
#define ASM_FOUND_FN __host__ __device__ __forceinline__
#else
#define ASM_FOUND_FN inline
#endif

namespace asmllm {

// 0 parts: no position; 1: whole, found by row; more: ranges first .. first + parts - 1 hold one part each, the first of them
// in slot `slot`, the others in slot 2 r of range r.
struct Found {
  int parts, first, slot, pad;
};

// Parts that may be read where there are `ranges` ranges of two slots each.
ASM_FOUND_FN int parts_of(const Found& f, int ranges) {
  if (f.parts == 1) return 1;
  const bool inside = f.parts > 1 && f.first >= 0 && f.first < ranges && f.parts <= ranges - f.first && f.slot >= 0 &&
                      f.slot < 2 * ranges;
  return inside ? f.parts : 0;
}

// Sequence s, of `batch`, is one of group `group`'s, of `groups`, which are [begin, end).
ASM_FOUND_FN bool in_group(int group, int begin, int end, int s, int groups, int batch) {
  return group >= 0 && group < groups && begin >= 0 && begin <= s && s < end && end <= batch;
}

// The rest of a walk whose work has been given up: leave() for each unit that begins in it, from the present one on.
// w: tiles [at, end) are left, tile t of a unit of nt is next; advance(n) goes n tiles on, to the end of a unit or of the walk.
template <class W, class Leave, class Advance>
ASM_FOUND_FN void abandon(W& w, Leave leave, Advance advance) {
  while (w.at < w.end) {
    if (w.t == 0) leave();
    const long long unit = w.nt - w.t, rest = w.end - w.at;
    advance((int)(unit < rest ? unit : rest));
  }
}

}  // namespace asmllm
