// How the rows of the 8-bit weight stream (op 317) are cut along K. No HIP here: tests compile it alone.
#pragma once

namespace kvm {

// Steps of all waves (512 bytes of a row) in one part of K: the fewest parts of which one's rows (`bytes` of LDS a step) fit into `room`, all
// alike. The last part may end behind K, by less than a step for each other part; the staged rows are 0 there. (Parts that divide the steps
// evenly would be one step each for a prime number of them: 16 rows of 8,704 bytes in 17 parts, 63 us where 8,192 take 44.)
constexpr int gq_part_steps(int steps, int bytes, int room) {
  const int most = room / bytes < 1 ? 1 : room / bytes < steps ? room / bytes : steps;
  const int parts = (steps + most - 1) / most;
  return (steps + parts - 1) / parts;
}

}  // namespace kvm
