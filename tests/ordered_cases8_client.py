"""As ordered_cases_client.py, for the performance cases of the context in 8
bits: inputs, calls and outputs asked for without a wait give the same bits as
with waits between them, on torch's default stream and on another."""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from ordered_cases_client import passes  # noqa: E402
import ordered_cases_client  # noqa: E402
from perf import more_operators as P  # noqa: E402


def main():
    P.own = True
    ordered_cases_client.P = P
    for stream in (torch.cuda.default_stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            for case in P.listed():
                if case["name"] in ("plan_1", "append8_1", "append8_200", "decode8_1x777", "prompt8_5x611"):
                    want = passes(case, True)
                    for _ in range(3):
                        same = [torch.equal(g.view(torch.uint8), w.view(torch.uint8)) for g, w in zip(passes(case, False), want)]
                        print(case["name"], stream.cuda_stream != 0, same, flush=True)
                        assert all(same)
    print("ordered")


if __name__ == "__main__":
    main()
