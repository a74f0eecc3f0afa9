// What the host keeps about an executor's launches. No HIP here: tests compile it alone.
#pragma once

namespace kvm {

// The second word of a launch's report: 16 bits of its sequence number (enough to know it from the report before) and 48 bits of the
// launch's time in ticks of 10 ns, a month of them. (32 bits, beside the whole number, are 43 seconds, and the timeout bounds only how
// long no task ends.)
constexpr unsigned long long report_time(int seq, unsigned long long ticks) { return (ticks << 16) | ((unsigned)seq & 0xffffu); }
constexpr bool report_time_is(unsigned long long word, int seq) { return (word & 0xffffu) == ((unsigned)seq & 0xffffu); }
constexpr float report_ms(unsigned long long word) { return (float)((double)(word >> 16) * 1e-5); }

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
