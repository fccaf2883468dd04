"""What the paged cache's attention decides on the host (csrc/wt_kv_plan.h), asked of a host program that includes the header."""
import os
import shutil
import subprocess

import pytest
import torch

import kv_known as K

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


CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.float8_e4m3fn: 3}
PLAN = """
    const auto plan = [](int cus, int dtype, int width, int page, int heads, int seqs, int q_heads, int columns) {
        wt_kv_cache c = {};
        c.dtype = dtype, c.head_dim = width, c.page_size = page, c.n_heads = heads;
        return kv_plan(cus, c, seqs, q_heads, columns);
    };"""


def test_every_schedule_has_its_shapes(tmp_path):
    """The shapes of kv_known take the schedules that they are there for, so that a rule that moves cannot quietly leave one untested;
    together they take every kernel that the library has."""
    shapes = K.shapes()
    lines = [f"{{{CODE[s.dtype]}, {s.width}, {s.page}, {s.heads}, {len(s.lengths)}, {s.heads * s.group}, {s.columns}}}" for s in shapes]
    found = host_program(tmp_path, PLAN + "const int shapes[][7] = {" + ", ".join(lines) + """};
        for (const auto &s : shapes) {
            const KvPlan p = plan(256, s[0], s[1], s[2], s[3], s[4], s[5], s[6]);
            std::printf("%d %d %d %d %d\\n", p.direct, p.waves, p.q_wide, p.min_share, p.q_tiles);
        }""")
    for s, (direct, waves, wide, least, tiles) in zip(shapes, found):
        assert (bool(direct), waves, wide) == (s.whole, s.waves, s.tiles), (s, direct, waves, wide)
        assert tiles == -(-s.group // (16 * s.tiles))
        assert max(s.lengths) <= s.columns * s.page
        if not s.whole:
            assert s.share() >= least and -(-(-(-max(s.lengths) // s.unit())) // s.share()) >= s.parts, (s, s.share())
    kinds = {(s.q_dtype, s.dtype, s.width, s.whole, s.waves, s.tiles) for s in shapes}
    for q, d in K.PAIRS:
        for width in (32, 64, 96, 128, 256):
            assert {(q, d, width, True, 2, 1), (q, d, width, False, 4, 1)} <= kinds
            assert width == 256 or {(q, d, width, True, 4, 2), (q, d, width, False, 4, 2)} <= kinds


def test_a_workspace_does_for_fewer_sequences_and_pages(tmp_path):
    """What wt_kv_attend_workspace gives (the larger of the call's own need and that of one sequence) is enough for any fewer of them."""
    found = host_program(tmp_path, PLAN + """
        const int widths[] = {32, 64, 96, 128, 256}, cus[] = {256, 304, 64, 32, 8, 1};
        unsigned r = 1;
        const auto next = [&](int n) { r = r * 1664525u + 1013904223u; return (int)((r >> 8) % n); };
        for (int i = 0; i < 4000; ++i) {
            const int c = cus[next(6)], d = next(4), w = widths[next(5)], page = 1 << next(9), heads = 1 + next(20), group = 1 + next(50);
            const int seqs = 1 + next(i % 2 ? 400 : 20), columns = 1 + next(i % 3 ? 200 : 20000);
            const auto bytes = [&](int s, int col) { return (long long)plan(c, d, w, page, heads, s, heads * group, col).bytes; };
            const long long given = std::max(bytes(seqs, columns), bytes(1, columns));
            long long most = 0;
            for (int s = 1; s <= seqs; ++s)
                for (int col = columns; col > 0; col = col > 64 ? col * 9 / 10 : col - 1) most = std::max(most, bytes(s, col));
            std::printf("%d %d\\n", (int)(most <= given), (int)(given > 0));
        }""", "#include <algorithm>\n")
    assert all(ok for ok, _ in found) and any(g for _, g in found) and not all(g for _, g in found)


def test_known_results_tell_a_lost_key():
    """The mistakes that the known results are there for, made on purpose: 16 keys left out, or taken twice, anywhere, show in every type."""
    g = torch.Generator().manual_seed(0)
    for s in K.shapes():
        n = max(s.lengths)
        v = K.counting_values(n, s.heads, s.width)
        right, _ = K.counted(v, n, s.q_dtype)
        for at in [0, (n - 1) // K.RUN * K.RUN] + (torch.randint(0, -(-n // K.RUN), (4,), generator=g) * K.RUN).tolist():
            for wrong in (dict(without=at), dict(twice=at)):
                assert not torch.equal(K.counted(v, n, s.q_dtype, **wrong)[0], right), (s, wrong)
        k, x, at = K.peaked(n, s.heads, s.width, s.dtype)
        q, columns = K.peak_queries(len(s.lengths), s.heads, s.group, s.width, s.q_dtype)
        columns = columns[0]
        want, allowed = K.peak_results(x, at, n, columns, s.q_dtype, s.depth())
        for p in [p for p in range(n) if int(at[p]) in columns.tolist()][::97]:
            wrong, _ = K.peak_results(x, at, n, columns, s.q_dtype, s.depth(), without=p // K.RUN * K.RUN)
            assert float(((wrong - want).abs() / allowed).max()) > 2.0, (s, p)


def test_very_many_heads_over_very_long_tables(tmp_path):
    """2^27 heads over tables of 2^40 bytes are more than 64 MB, although their product has no place in 64 bits."""
    found = host_program(tmp_path, PLAN + """
        for (int seqs : {1 << 10, 1 << 17, 1 << 22}) {
            const KvPlan p = plan(256, WT_DTYPE_BF16, 128, 1 << 20, 32, seqs, 32 * 24, 2047);
            std::printf("%d %d %d\\n", p.direct, p.q_wide, p.grid == 256);
        }""")
    assert found == [(0, 2, 1)] * 3
