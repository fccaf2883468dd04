#!/usr/bin/env python3
"""transcribe_batch with the decoder's text in the backend's concatenated caches and in paged ones (streams.PAGED_SELF_ATTENTION), in turn:
whisper-base of random weights, n recordings of 30 s stepping together, scripted transcripts (so that both decode the same
number of tokens).  The least of `--reps` runs of each; the words of both are compared.

    python tools/bench_paged_decoder.py [--streams 32,128] [--reps 5]
"""
import argparse
import os
import sys
import time

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (os.path.join(ROOT, "tests"), os.path.join(ROOT, "whisper-timestamped_amd"), ROOT):
    sys.path.insert(0, p)

import torch  # noqa: E402

import many_helper as H  # noqa: E402
import whisper_double as W  # noqa: E402
from golden import make_golden_transcribe as G  # noqa: E402
from whisper_double.decoding import Script, set_row_scripts  # noqa: E402

W.install()
import whisper_timestamped as wt  # noqa: E402
from whisper_timestamped import streams  # noqa: E402


def main():
    a = argparse.ArgumentParser()
    a.add_argument("--streams", default="32,128")
    a.add_argument("--reps", type=int, default=5)
    a = a.parse_args()
    model = H.load_base("cuda:0")
    g = torch.Generator().manual_seed(7)
    clips = [(0.05 * torch.randn(30 * 16000, generator=g)).float() for _ in range(4)]
    window = G.window_script(50364, 50257, [(s, [None] * n, e) for s, n, e in H.SEGMENTS], "eot")

    def batch(n, fp16):
        scripts = [Script([window]) for _ in range(n)]

        def on_group(idx):
            for i in idx:
                scripts[i].begin_window()
            set_row_scripts([scripts[i] for i in idx])
        streams.ON_GROUP_DECODE = on_group
        try:
            return wt.transcribe_batch(model, [clips[k % 4] for k in range(n)], max_streams=n, language="en", fp16=fp16)
        finally:
            streams.ON_GROUP_DECODE = None
            set_row_scripts(None)

    for fp16 in (False, True):
        for n in map(int, a.streams.split(",")):
            took, words = {False: [], True: []}, {}
            for rep in range(-1, a.reps):
                for paged in (False, True):
                    streams.PAGED_SELF_ATTENTION = paged
                    torch.cuda.synchronize()
                    t = time.perf_counter()
                    out = batch(n, fp16)
                    torch.cuda.synchronize()
                    if rep >= 0:
                        took[paged].append(time.perf_counter() - t)
                    words[paged] = [[w["text"] + "%.2f" % w["start"] for s in x["segments"] for w in s["words"]] for x in out]
            same = sum(x == y for x, y in zip(words[False], words[True]))
            print("%s %4d recordings: concatenated %.3f s (%s), paged %.3f s (%s); words and starts equal in %d" % (
                "f16" if fp16 else "f32", n, min(took[False]), " ".join("%.3f" % x for x in took[False]), min(took[True]),
                " ".join("%.3f" % x for x in took[True]), same), flush=True)


if __name__ == "__main__":
    main()
