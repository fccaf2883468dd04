"""What the paged cache's attention decides on the host (csrc/wt_kv_plan.h), asked of a host program that includes the header."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "whisper-timestamped_amd", "csrc")


def host_program(folder, main, more=""):
    """The numbers that a host program over the header prints, line by line (nothing is launched)."""
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not found")
    src, exe = folder / "probe.hip", folder / "probe"
    src.write_text('#include <cstdio>\n#include "wt_kv_plan.h"\n' + more + 'using namespace wt;\nint main() {\n' + main + "\nreturn 0; }\n")
    subprocess.check_call([hipcc, "--offload-arch=gfx950", "-std=c++17", "-I" + CSRC, "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    return [tuple(map(int, line.split())) for line in subprocess.check_output([str(exe)], text=True).splitlines()]


def test_join_stays_in_its_workgroups_lds(tmp_path):
    """Six floats of LDS a thread: a thread that leads `lanes` of them reads those of the next lanes - 1 threads too.  The last
    threads of a workgroup that `lanes` does not divide lead nobody (head_dim 32, one query, 17 ... 24 parts: lanes 3, and
    thread 255 has multiples of 3 before it)."""
    found = host_program(tmp_path, """
        for (int rows = 1; rows <= 32; ++rows)
            for (int hd : {32, 64, 96, 128, 256})
                for (int count = 1; count <= 1024; ++count) {
                    const int lanes = kv_join_lanes(256, rows * hd / 4, count);
                    int far = 0, all = 0, led = 0;
                    for (int t = 0; t < 256; t += lanes) {
                        all = t + lanes - 1;
                        if (kv_join_grouped(t, lanes, 256)) far = t + lanes - 1, ++led;
                    }
                    std::printf("%d %d %d %d %d %d %d\\n", rows, hd, count, lanes, far, all, led);
                }""")
    assert len(found) == 32 * 5 * 1024
    assert all(far < 256 and led == 256 // lanes for *_, lanes, far, _, led in found)
    assert any(all_ >= 256 for *_, all_, _ in found), "the remainder that the rule is there for"
    assert (1, 32, 20, 3, 254, 257, 85) in found


def test_a_threads_own_stream_has_memory_of_its_own(tmp_path):
    """hipStreamPerThread is the same handle in every thread, and another stream: kept apart by thread; other handles are not."""
    found = host_program(tmp_path, """
        const hipStream_t other = reinterpret_cast<hipStream_t>(0x1000);
        StreamKey mine = stream_key(hipStreamPerThread), theirs, theirs_other, next;
        std::thread([&] { theirs = stream_key(hipStreamPerThread), theirs_other = stream_key(other); }).join();
        std::thread([&] { next = stream_key(hipStreamPerThread); }).join();
        std::printf("%d %d %d %d %d %d\\n", mine == stream_key(hipStreamPerThread), mine == theirs, theirs == next, mine == next,
                    theirs_other == stream_key(other), stream_key(nullptr) == StreamKey{nullptr, 0});""", "#include <thread>\n#include \"wt_stream_key.h\"\n")
    assert found == [(1, 0, 0, 0, 1, 1)]
