"""Paged attention in a process where about one in TL_PAGED_FAIL_WAITS waits of the kernels gives up (read once a
process): rows whose copies or products were not waited for are done over, and come out right all the same.

    python paged_waits_child.py decode|chunks
"""
import os
import sys

sys.path[:0] = [os.path.dirname(os.path.abspath(__file__)), os.path.dirname(os.path.dirname(os.path.abspath(__file__)))]
import numpy as np  # noqa: E402
import torch  # noqa: E402

from test_paged_gpu import DT, TYPES, attend_case, check_attend, i32, ops, run_attend  # noqa: E402


def done_over(new):
    """The share of a call's rows that were done over: a weight of 2^-129 is 0 in the kernels' exponentials, but not there."""
    q, kc, vc, table, q_start, ln = attend_case([2000] * len(new), new, 1, 1, 64, 16, "f32")
    dtype = torch.float32 if max(new) == 1 else torch.bfloat16
    q, kc, vc = torch.zeros_like(q).to(dtype), torch.zeros_like(kc).to(dtype), torch.zeros_like(vc).to(dtype)
    q[..., 0], kc[..., 0] = 1, -200
    for t in table:
        kc[t[0], 0, 0, 0], kc[t[0], 0, 1, 0], vc[t[0], 0, 1] = 0, -89.5, 1e30
    out = torch.full(q.shape, 3.0, device="cuda", dtype=dtype)
    ops().paged_attention(out, q, kc, vc, i32(table), i32(q_start), i32(ln), 1.0)
    want = np.exp(-89.5) * 1e30
    assert ((out == 0) | ((out - want).abs() < 0.02 * want)).all()
    return (out != 0).float().mean().item()


def main(kind):
    one_in = os.environ.get("TL_PAGED_FAIL_WAITS")
    for dtype in TYPES if kind == "decode" else ("f16", "bf16"):
        for again in range(4):
            if kind == "decode":
                run_attend([700, 1, 64, 130, 0], [1] * 5, 8, 2, 128, 16, dtype, seed=again)
                run_attend([3000, 90], [1, 1], 4, 1, 64, 32, dtype, seed=again, window=1500)
                run_attend([300] * 40, [1] * 40, 8, 2, 64, 8, dtype, seed=again)
            else:
                run_attend([700, 1, 300, 130], [300, 1, 20, 70], 8, 2, 128, 16, dtype, seed=again)  # tiles of 256 rows and fewer
                run_attend([600] * 6, [20] * 6, 4, 1, 64, 32, dtype, seed=again)  # both streams have each row
                run_attend([1500], [90], 3, 1, 128, 64, dtype, seed=again, window=1000)  # Q by lanes
    share = done_over([1] * 64 if kind == "decode" else [30, 40])
    assert share == 1 if one_in == "1" else share == 0 if one_in is None else True, (one_in, share)
    torch.cuda.synchronize()
    print("right", one_in, share)


if __name__ == "__main__":
    main(sys.argv[1])
