"""Passes over performance cases of the context operators right behind the
making of their inputs and before the reading of their outputs, all asked for
without a wait and with work in front of the inputs: the same bits as with
waits between them, on torch's default stream and on another."""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from perf import operators as P  # noqa: E402


def passes(case, wait):
    big = torch.ones(4096, 4096, device="cuda")
    for _ in range(0 if wait else 20):  # milliseconds that the inputs stand behind
        big = big @ big * 2.0 ** -12
    state = P.prepare(case, 5)
    if wait:
        torch.cuda.synchronize()
    got = P.run(state)
    if wait:
        torch.cuda.synchronize()
    got = [t.clone() for t in (got.values() if isinstance(got, dict) else [got])]
    torch.cuda.synchronize()
    return got


def main():
    P.own = True
    for stream in (torch.cuda.default_stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            for case in P.listed():
                if case["name"] in ("append_1", "decode_1x777", "prompt_5x611", "step_1", "delta_3x251"):
                    want = passes(case, True)
                    for _ in range(3):
                        same = [torch.equal(g, w) for g, w in zip(passes(case, False), want)]
                        print(case["name"], stream.cuda_stream != 0, same, flush=True)
                        assert all(same)
    print("ordered")


if __name__ == "__main__":
    main()
