"""The host's bookkeeping of launches (kvm_amd/csrc/launch_state.h), compiled alone. No GPU needed."""
import subprocess

import pytest

from kvm_amd import build as kb


@pytest.fixture(scope='module')
def run(tmp_path_factory):
    """run(statements): a program of them, with `L` a LaunchState; CHECK ends it with the line that does not hold."""
    def go(body):
        d = tmp_path_factory.mktemp('ls')
        (d / 'a.cpp').write_text('#include "launch_state.h"\n#include <cstdio>\n#include <cstdlib>\n#include <initializer_list>\n'
                                 '#define CHECK(x) do { if (!(x)) { std::printf("%s\\n", #x); std::exit(1); } } while (0)\n'
                                 'using namespace kvm;\nint main() {\n  LaunchState L;\n' + body + '\n}\n')
        subprocess.run([kb.CXX, '-std=c++17', '-O1', f'-I{kb.CSRC}', str(d / 'a.cpp'), '-o', str(d / 'a')], check=True)
        r = subprocess.run([str(d / 'a')], capture_output=True, text=True)
        assert r.returncode == 0, r.stdout
    return go


def test_sequence_numbers_are_never_zero(run):
    run('CHECK(L.next_seq() == 1 && L.next_seq() == 2 && L.seq == 2);'
        'L.seq = 0x7fffffff; CHECK(L.next_seq() == (int)0x80000000u);'
        'L.seq = -1; CHECK(L.next_seq() == 1 && L.seq == 1);')


def test_a_reset_goes_in_front_after_anything_that_failed(run):
    run('CHECK(L.begin(true)); L.enqueued(true); CHECK(!L.begin(true)); L.enqueued(true);'        # the first one, the next one
        'CHECK(!L.begin(true)); CHECK(L.begin(true));'                                            # one that was not enqueued
        'L.enqueued(true); L.lost(); CHECK(L.begin(true)); L.enqueued(true);'                     # one without its report
        'CHECK(L.begin(false)); L.enqueued(false); CHECK(!L.reported && L.begin(true) && L.reported);')   # a traced one between


def test_launches_longer_than_32_bits_of_ticks(run):
    """43 seconds are 2^32 ticks of 10 ns."""
    run('const unsigned long long t = 100ull * 1000 * 1000 * 60 * 60 * 24;'                       # a day
        'for (int seq : {1, 65535, 65536, 65537, -1, (int)0x80000001u}) {'
        '  const unsigned long long w = report_time(seq, t);'
        '  CHECK(report_time_is(w, seq) && !report_time_is(w, seq + 1) && !report_time_is(w, seq - 1) && report_ms(w) == 86400000.f); }'
        'CHECK(report_ms(report_time(7, (1ull << 32) + 100000)) > 42949.f && report_ms(report_time(7, 100)) == 1e-3f);'
        'CHECK(!report_time_is(0, 1));')
