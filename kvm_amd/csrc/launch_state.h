// What the host keeps about an executor's launches. No HIP here: tests compile it alone.
#pragma once

namespace kvm {

struct LaunchState {
  int seq = 0;                // sequence number of the last report asked for
  bool reported = false;      // the last launch's report is on its way
  bool self_timed = false;    // the last launch has its own time in its report
  bool clean = false;         // the device state is as a reset leaves it (untraced static launches)
  // The next report's number. Never 0, which in a launch's arguments says that it does not report itself: after 2^32 launches (a day
  // of short ones) the numbers start at 1 again.
  int next_seq() {
    const unsigned s = (unsigned)seq + 1u;
    return seq = (int)(s ? s : 1u);
  }
};

}  // namespace kvm
