// The rounds of a ring of stages that two CTAs fill, each its own shared memory, against one barrier a stage (count 2: an
// arrival of each CTA with the bytes that it copies), and what is left of them when a CTA gives up. Plain C++: the host's
// tests compile it.
#pragma once

namespace psgd {

// How many of the first `rounds` rounds of a ring of `stages` were of stage i.
constexpr unsigned ring_uses(unsigned rounds, unsigned stages, unsigned i) { return rounds / stages + (i < rounds % stages ? 1u : 0u); }

// Stage i after one CTA of a pair has issued the copies of `own` rounds and the other those of `peer`, neither issuing any
// more. The barrier's phase k ends when both have arrived for their k-th use of the stage and all bytes have landed, and a
// stage is used again only after its phase before was used up, so the two are at most one use apart and one phase at most is
// open. Where they are one apart, the open phase lacks the arrival of the CTA that is behind (it copies nothing): `arrive`
// says that it has to be made up for. After that the last phase ends as soon as what is in flight has landed; `wait` says
// that there is one, `parity` is its parity.
struct StageLeft {
  bool arrive, wait;
  unsigned parity;
};
constexpr StageLeft stage_left(unsigned own, unsigned peer, unsigned stages, unsigned i) {
  const unsigned a = ring_uses(own, stages, i), b = ring_uses(peer, stages, i), most = a > b ? a : b;
  return StageLeft{a != b, most > 0, (most - 1u) & 1u};
}

}  // namespace psgd
