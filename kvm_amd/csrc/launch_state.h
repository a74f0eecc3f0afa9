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
  // Around the enqueueing of a launch: whether a reset goes in front of it; it is enqueued; something about it failed. The state is
  // clean for the next launch only once a launch that clears it is known to be on its way.
  bool begin(bool light) {
    const bool reset = !(light && clean);
    clean = false;
    reported = light;
    return reset;
  }
  void enqueued(bool light) { clean = light; }
  void lost() { clean = false; }
};

}  // namespace kvm
