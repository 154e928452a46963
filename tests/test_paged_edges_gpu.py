"""Edges of the paged serving operators, against the plain 64-bit forms."""
import math
import os
import subprocess
import sys
import threading

import numpy as np
import pytest

import paged_plain as plain
from test_paged_gpu import DT, TYPES, attend_case, check_attend, check_rope, f32, f64, i32, ops, rope_case, run_sample, u

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)


def attend(q, kc, vc, table, q_start, lens, scale=None, window=0):
    out = torch.full(q.shape, 3.0, device="cuda", dtype=q.dtype)
    ops().paged_attention(out, q, kc, vc, i32(table), i32(q_start), i32(lens), scale, window)
    return out


# ---------------------------------------------------------------- sampling

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 3, 1001, 4093, 32001, 270001])
def test_masked_logits_are_not_drawn_at_very_large_temperatures(dtype, n):
    """All weights are 1 but those of -inf, which stay 0 at any temperature; rows begin off 16 bytes (odd n)."""
    rng = np.random.default_rng(n)
    temps = np.array([1e36, 1.3e37, 1e38, 3.4e38, np.inf], np.float32)
    rows = 4 * len(temps)
    x = rng.standard_normal((rows, n)).astype(np.float32)
    x[rng.random((rows, n)) < 0.3] = -np.inf
    x[::4] = rng.standard_normal((len(temps), n))
    x[1::4, : n // 2] = -np.inf
    x[:, n // 3] = 0.5
    T = np.repeat(temps, 4)
    t = torch.as_tensor(x).cuda().to(DT[dtype])
    xs = t.float().cpu().numpy()
    for k, p, m in ((0, 1.0, 0.0), (2, 1.0, 0.0), (700, 1.0, 0.5), (0, 0.37, 0.0), (900, 0.61, 1.0)):
        for r in (0.0, 0.43, float(np.nextafter(np.float32(1), np.float32(0)))):
            full = [np.full(rows, v, np.float32) for v in (r, p, m)]
            got = ops().sample_rows(t, f32(full[0]), f32(T), i32(np.full(rows, k)), f32(full[1]), f32(full[2])).cpu().numpy()
            # (x - max) / T of these rows is 0 to within 1e-35, and the quotient -inf / inf is read as -inf
            want = [plain.sample(xs[i], r, min(T[i], np.float32(3.4e38)), k, p, m) for i in range(rows)]
            np.testing.assert_array_equal(got, want, err_msg=str((k, p, m, r)))


def test_sample_from_several_threads():
    """Rows of two sizes, which take unlike amounts of shared memory, from host threads at once."""
    from torchless_b200 import lib
    rng = np.random.default_rng(1)
    jobs, bad = [], []
    for n in (777, 32000):
        x = rng.standard_normal((1, n)).astype(np.float32)
        r, T = rng.random(1).astype(np.float32), np.full(1, 0.9, np.float32)
        jobs.append((torch.as_tensor(x).cuda(), f32(r), f32(T), plain.sample(x[0], r[0], T[0])))

    def work(x, r, T, want):
        side, out, L = torch.cuda.Stream(), i32([-1]), lib()
        n, args = x.shape[1], (r.data_ptr(), T.data_ptr(), None, None, None, side.cuda_stream)
        torch.cuda.synchronize()
        status = [L.tl_sample_rows(out.data_ptr(), x.data_ptr(), 0, n, 1, n, *args) for _ in range(4000)]
        side.synchronize()
        if any(status) or out.item() != want:
            bad.append((n, sum(map(bool, status)), out.item(), want))

    threads = [threading.Thread(target=work, args=job) for job in jobs for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("n", [7, 1500, 32000, 270000])
def test_min_p_above_one_keeps_the_first_of_the_order(n):
    """No weight reaches it: one logit is kept all the same, the largest with the lowest index."""
    rng = np.random.default_rng(n)
    x = rng.integers(0, 4, (4, n)).astype(np.float32)
    r, T = np.array([0.0, 0.3, 0.7, 0.99], np.float32), np.full(4, 0.8, np.float32)
    m = np.array([1.0001, 2.0, np.inf, 1.0], np.float32)
    for k, p in ((None, None), ([3] * 4, None), ([n // 2] * 4, [0.9] * 4), (None, [0.5] * 4)):
        run_sample(x, r, T, k, p, m)


# ---------------------------------------------------------------- attention

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [[1, 1], [90, 33]])
@pytest.mark.parametrize("scale", [1e6, 1e7, 1e9, 3e36, 1e37, -1e37, 2e38])
def test_scores_that_pass_fp32_through_the_scale(dtype, new, scale):
    """Products of small whole numbers are exact, so the largest has all the weight, however large the scale (ties share
    it).  One kv head's products are all negative."""
    q, kc, vc, table, q_start, ln = attend_case([90, 333], new, 8, 2, 64, 16, dtype)
    g = torch.Generator(device="cuda").manual_seed(5)
    q.copy_(torch.randint(1, 4, q.shape, generator=g, device="cuda"))
    k = torch.randint(-3, 4, kc.shape, generator=g, device="cuda")
    k[:, 1] = -k[:, 1].abs() - 1
    kc.copy_(k)
    out = attend(q, kc, vc, table, q_start, ln, scale)
    want, ao, _, _, _ = plain.attend(f64(q), f64(kc), f64(vc), table, q_start, ln, scale, 0)
    # the weights of the largest are alike and exact, the sum over ties (fewer than 64) and the quotient round in 32 bits
    tol = u(DT[dtype]) * np.abs(want) * (1 + 2.0 ** -8) + 80 * 2.0 ** -24 * ao
    assert np.all(np.abs(f64(out) - want) <= tol)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens,new", [([50, 200], [1, 1]), ([6000], [1]), ([140, 50], [140, 40]), ([3000, 40], [30, 20])])
def test_values_near_the_largest_of_the_type(dtype, lens, new):
    """A mean of finite values is finite, although their sum is not."""
    q, kc, vc, table, q_start, ln = attend_case(lens, new, 4, 1, 64, 16, dtype)
    vc[..., 3] = 3e38
    vc[..., 7] = torch.where(torch.rand(vc.shape[:-1], device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) < 0.5,
                             3e38, -3e38).to(vc.dtype)
    check_attend(attend(q, kc, vc, table, q_start, ln), q, kc, vc, table, q_start, ln, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n,ln", [(64, 300), (30, 300), (30, 100)])
def test_a_column_that_is_not_finite_leaves_the_other_half_alone(dtype, n, ln):
    """As many equal row tiles as SMs, so that each block has a whole one.  The threads that hold the columns of the other
    half do not see the infinity, and what they write must not depend on who is faster."""
    seqs = torch.cuda.get_device_properties(0).multi_processor_count
    q, kc, vc, table, q_start, lens = attend_case([ln] * seqs, [n] * seqs, 4, 1, 128, 16, dtype)
    clean = attend(q, kc, vc, table, q_start, lens)
    for b in range(seqs):
        vc[table[b, (ln - 3) // 16], 0, (ln - 3) % 16, 5] = float("inf")
    for _ in range(5):
        out = attend(q, kc, vc, table, q_start, lens)
        assert torch.equal(out[..., 64:], clean[..., 64:])
        rows = out.view(seqs, n, 4, 128)
        assert torch.isfinite(rows[:, : n - 3]).all() and torch.isposinf(rows[:, n - 3:, :, 5]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 20])
@pytest.mark.parametrize("n", [2500, 20000])
def test_many_small_weights_add_up(dtype, rows, n):
    """One key with nearly all the weight and n of 2^-25.2 each: the small ones are the whole result.  As many sequences
    (over the same pages) as SMs, so that a block has the whole of one."""
    hd, bs = 64, 16
    seqs = torch.cuda.get_device_properties(0).multi_processor_count
    table = np.tile(np.arange(-(-n // bs), dtype=np.int32), (seqs, 1))
    kc = torch.zeros(table.shape[1], 1, bs, hd, device="cuda", dtype=DT[dtype])
    vc = torch.ones_like(kc)
    kc[..., 0] = -17.5
    kc[0, 0, 0], vc[0, 0, 0] = 0, 0
    q = torch.zeros(rows * seqs, 1, hd, device="cuda", dtype=DT[dtype])
    q[..., 0] = 1
    out = f64(attend(q, kc, vc, table, rows * np.arange(seqs + 1), [n] * seqs, 1.0))
    w = np.tile(n - rows + np.arange(rows), seqs) * math.exp(-17.5)  # the keys of the small weight
    want = (w / (1 + w))[:, None, None]
    # the score and its factor log2(e) round to 2^-24 of 25.2 log2 units (ln 2 of that in the weight), the weight and the
    # result round to the type, and the running sums to 32 bits, one step a key at worst
    rel = 4 * 25.2 * 2.0 ** -24 + n * 2.0 ** -24 + (3 * u(DT[dtype]) if dtype != "f32" else 0)
    assert np.all(np.abs(out - want) <= rel * want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [40, 20, 33, 25]])
def test_lengths_below_zero(dtype, new):
    """Queries of a length at or near the smallest whole number stand before position 0: zeros."""
    q, kc, vc, table, q_start, ln = attend_case([90, 64, 64, 64], new, 8, 2, 64, 16, dtype)
    ln[1:] = -2 ** 31, -2 ** 31 + 10, -1
    for window in (0, 20):
        out = attend(q, kc, vc, table, q_start, ln, window=window)
        check_attend(out, q, kc, vc, table, q_start, ln, dtype, window=window)
        assert (out[q_start[1]:] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,new", [([3, 90, 2], [8, 1, 1]), ([10, 90], [60, 40])])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 8, 2 ** 31, 2 ** 40])
def test_the_largest_windows(dtype, lens, new, window):
    """More than any length is no window, also beside queries that stand before position 0."""
    q, kc, vc, table, q_start, ln = attend_case(lens, new, 4, 2, 64, 16, dtype)
    out = attend(q, kc, vc, table, q_start, ln, window=window)
    check_attend(out, q, kc, vc, table, q_start, ln, dtype)
    assert torch.equal(out, attend(q, kc, vc, table, q_start, ln))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 30])
def test_one_kv_head_and_one_page_in_any_layout(dtype, tokens):
    """A dimension of size 1 has no layout: a cache kept as [n_blocks, block_size, 1, head_dim] is the same pages, and K may
    come that way beside V in its own."""
    q, kc, vc, table, q_start, ln = attend_case([60, 40], [tokens, tokens], 4, 1, 64, 16, dtype)

    def turn(c):
        return torch.empty(c.shape[0], 16, 1, 64, device="cuda", dtype=c.dtype).copy_(c.transpose(1, 2)).transpose(1, 2)

    turned = turn(kc)
    assert turned.shape == kc.shape and turned.stride(1) == 64
    want = attend(q, kc, vc, table, q_start, ln)
    assert torch.equal(attend(q, turned, vc, table, q_start, ln), want)
    assert torch.equal(attend(q, turned, turn(vc), table, q_start, ln), want)
    # one page
    kk, vv = kc[table[1, 0]][None], vc[table[1, 0]].clone()[None]
    odd = torch.empty(5, *kk.shape[1:], device="cuda", dtype=kk.dtype)[:1].copy_(vv)
    odd = odd.as_strided(odd.shape, (3, *odd.stride()[1:]))
    one = [np.zeros((1, 1), np.int32), [0, tokens], [16]]
    assert torch.equal(attend(q[:tokens], kk, odd, *one), attend(q[:tokens], kk, vv, *one))


def test_pages_that_are_not_contiguous_are_refused():
    kc = torch.zeros(6, 2, 16, 64, device="cuda")
    q = torch.zeros(1, 4, 64, device="cuda")
    for bad in (kc.transpose(1, 2).contiguous().transpose(1, 2), kc[:, :, ::2], torch.zeros(6, 2, 16, 128, device="cuda")[..., ::2]):
        with pytest.raises(ValueError, match="contiguous"):
            attend(q, bad, bad, np.zeros((1, 1), np.int32), [0, 1], [1])
    with pytest.raises(ValueError, match="layout"):  # unlike strides between the pages
        attend(q, kc[::2], kc[:3], np.zeros((1, 1), np.int32), [0, 1], [1])


# ---------------------------------------------------------------- cache writes

@pytest.mark.parametrize("dtype", TYPES)
def test_two_tokens_with_one_slot_leave_every_other_row_right(dtype):
    q_out, kc, vc, big, qkv, pos, slots, cos, sin, wq, wk = rope_case(30, 4, 2, 64, 16, 64, "f32", dtype, "both", page_pad=16)
    slots[9] = slots[4]
    before = [f64(t) for t in (q_out, kc, vc)]
    ops().qk_norm_rope(q_out, kc, vc, qkv, pos, slots, cos, sin, wq, wk)
    page, row = divmod(int(slots[4]), 16)
    kept = kc[page, :, row].clone(), vc[page, :, row].clone()
    # either token's values may stand in the shared slot: the two are compared with each token in its turn
    right = []
    for last in (4, 9):
        s = slots.clone()
        s[13 - last] = -1  # the other of 4 and 9
        c = [torch.from_numpy(b).cuda().to(kc.dtype) for b in before]
        ops().qk_norm_rope(*c, qkv, pos, s, cos, sin, wq, wk)
        right.append([x[page, :, row] for x in c[1:]])
        check_rope(*c, qkv, pos, s, cos, sin, wq, wk, dtype, before)
        for x, y in zip((q_out, kc, vc), c):
            y = y.clone()
            if x is not q_out:
                y[page, :, row] = x[page, :, row]
            assert torch.equal(x, y)
    for got, a, b in zip(kept, *right):
        assert ((got == a) | (got == b)).all()
    assert (big[:, :, 2 * 16 * 64:] == 7).all()


# ---------------------------------------------------------------- waits that run out

def child(kind, one_in):
    env = dict(os.environ, **({} if one_in is None else dict(TL_PAGED_FAIL_WAITS=str(one_in))))
    r = subprocess.run([sys.executable, os.path.join(os.path.dirname(__file__), "paged_waits_child.py"), kind], env=env,
                       capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and f"right {one_in}" in r.stdout, r.stdout[-500:] + r.stderr[-3000:]


@pytest.mark.parametrize("one_in", [None, 1, 100, 1000])
def test_decode_rows_whose_copies_were_not_waited_for_are_done_over(one_in):
    child("decode", one_in)


@pytest.mark.parametrize("one_in", [None, 1, 100, 1000])
def test_chunk_rows_whose_products_were_not_waited_for_are_done_over(one_in):
    child("chunks", one_in)
