"""The operators of the paged serving step against plain 64-bit forms."""
import numpy as np
import pytest

import paged_plain as plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)


def ops():
    from torchless_b200 import ops as o
    return o


def i32(v):
    return torch.as_tensor(np.asarray(v), dtype=torch.int32).cuda()


def f64(t):
    return t.detach().double().cpu().numpy()


# ---------------------------------------------------------------- plan

def run_plan(table, cached, new, free, bs, n_tokens):
    want = plain.plan(table, cached, new, free, bs, n_tokens)
    dev = i32(table)
    got = ops().paged_plan(dev, i32(cached), i32(new), i32(free), bs, n_tokens)
    for name, g, w in zip(("table", "q_start", "seq_lens", "positions", "slots", "counts"), (dev, *got), want):
        np.testing.assert_array_equal(g.cpu().numpy(), w, err_msg=name)


@pytest.mark.parametrize("n_req,width,bs,most_cached,most_new,pad,seed", [
    (1, 1, 8, 1, 1, 0, 0), (1, 9, 16, 100, 40, 3, 1), (7, 5, 8, 40, 20, 0, 2), (33, 12, 256, 2000, 900, 11, 3),
    (1023, 6, 16, 90, 3, 5, 4), (1024, 6, 16, 90, 3, 0, 5), (1025, 6, 16, 90, 3, 1, 6), (2500, 20, 64, 1200, 80, 77, 7),
])
def test_plan_matches_request_by_request(n_req, width, bs, most_cached, most_new, pad, seed):
    rng = np.random.default_rng(seed)
    cached = rng.integers(0, most_cached + 1, n_req)
    new = rng.integers(0, most_new + 1, n_req)
    ids = rng.permutation(n_req * width + 50).astype(np.int32)
    table = np.full((n_req, width), -1, np.int32)
    at = 0
    for b in range(n_req):
        h = min(-(-int(cached[b]) // bs), width)
        table[b, :h] = ids[at:at + h]
        at += h
    run_plan(table, cached, new, ids[at:], bs, int(new.sum()) + pad)


@pytest.mark.parametrize("what", ["short list", "empty list", "narrow table", "few rows", "no rows", "no new", "negative",
                                  "missing page", "all zero"])
def test_plan_edges(what):
    rng = np.random.default_rng(3)
    n_req, width, bs = 6, 4, 8
    cached = np.array([0, 5, 8, 17, 31, 1])
    new = np.array([9, 0, 8, 3, 1, 7])
    table = rng.permutation(100)[: n_req * width].reshape(n_req, width).astype(np.int32)
    free = np.arange(200, 240, dtype=np.int32)
    n = int(new.sum()) + 2
    if what == "short list":
        free = free[:2]
    elif what == "empty list":
        free = free[:0]
    elif what == "narrow table":
        table = table[:, :2].copy()
    elif what == "few rows":
        n = 13
    elif what == "no rows":
        n = 0
    elif what == "no new":
        new = new * 0
    elif what == "negative":
        cached, new = np.array([0, -5, 8, -1, 31, 1]), np.array([9, -3, 8, 3, -100, 7])
    elif what == "missing page":
        table[3, 2] = -1
    elif what == "all zero":
        cached, new = cached * 0, new * 0
    run_plan(table, cached, new, free, bs, n)


def test_plan_without_requests():
    q_start, lens, pos, slots, counts = ops().paged_plan(torch.empty(0, 3, dtype=torch.int32, device="cuda"), i32([]),
                                                         i32([]), i32([4]), 16, 5)
    assert q_start.tolist() == [0] and lens.numel() == 0 and counts.tolist() == [0, 0]
    assert pos.tolist() == [-1] * 5 and slots.tolist() == [-1] * 5


# ---------------------------------------------------------------- norm, rotation, cache write

def u(dtype):
    """Half a step of the type, relative."""
    return torch.finfo(dtype).eps / 2


def rope_case(T, H, KV, hd, bs, rot, src, dst, norm, stride_pad=0, page_pad=0, seed=0, n_pos=50):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = (H + 2 * KV) * hd
    qkv = torch.randn(T, n + stride_pad, generator=g, device="cuda").to(DT[src])[:, :n]
    nb = -(-T // bs) + 2
    big = torch.full((2, nb, KV * bs * hd + page_pad), 7.0, device="cuda", dtype=DT[dst])
    kc, vc = (big[i][:, :KV * bs * hd].view(nb, KV, bs, hd) for i in (0, 1))
    pos = torch.randint(0, n_pos, (T,), generator=g, device="cuda", dtype=torch.int32)
    slots = torch.randperm(nb * bs, generator=g, device="cuda")[:T].to(torch.int32)
    ang = torch.arange(n_pos, device="cuda")[:, None].double() * 100.0 ** (-torch.arange(rot // 2, device="cuda") / (rot / 2))
    wq = (1 + 0.3 * torch.randn(hd, generator=g, device="cuda")) if norm in ("both", "q") else None
    wk = (1 + 0.3 * torch.randn(hd, generator=g, device="cuda")) if norm in ("both", "k") else None
    q_out = torch.full((T, H, hd), 5.0, device="cuda", dtype=DT[dst])
    return q_out, kc, vc, big, qkv, pos, slots, ang.cos().float(), ang.sin().float(), wq, wk


def check_rope(q_out, kc, vc, qkv, pos, slots, cos, sin, wq, wk, dst, before):
    T, H, hd = q_out.shape
    nb, KV, bs, _ = kc.shape
    x = f64(qkv).reshape(T, H + 2 * KV, hd)
    p, sl = pos.cpu().numpy(), slots.cpu().numpy()
    live = (p >= 0) & (p < cos.shape[0])
    c, s = f64(cos)[np.where(live, p, 0)][:, None], f64(sin)[np.where(live, p, 0)][:, None]
    wqn, wkn = (None if w is None else f64(w) for w in (wq, wk))
    yq = plain.norm_rope(x[:, :H], wqn, c, s, 1e-5)
    yk = plain.norm_rope(x[:, H:H + KV], wkn, c, s, 1e-5)
    want_q = before[0].copy()
    want_q[live] = yq[live]
    want = [b.copy() for b in before[1:]]
    for t in range(T):
        if live[t] and 0 <= sl[t] < nb * bs:
            want[0][sl[t] // bs, :, sl[t] % bs] = yk[t]
            want[1][sl[t] // bs, :, sl[t] % bs] = x[t, H + KV:]
    for got, w in ((q_out, want_q), (kc, want[0]), (vc, want[1])):
        # one rounding to the type, and fp32 arithmetic on pairs whose larger member is below the
        # head's largest value M: about 12 roundings in the sum of squares (halved by the root), the
        # root, the quotient, two products and the rotation's two: under 16 of them on 2 M
        M = np.abs(w).max(-1, keepdims=True)
        assert np.all(np.abs(f64(got) - w) <= u(DT[dst]) * np.abs(w) + 32 * 2.0 ** -24 * M + 2.0 ** -25), dst


@pytest.mark.parametrize("T,H,KV,hd,bs,rot,src,dst,norm,sp,pp", [
    (1, 4, 1, 128, 16, 128, "bf16", "bf16", "both", 0, 0), (1, 1, 1, 64, 8, 64, "f32", "f32", "none", 0, 0),
    (37, 6, 2, 64, 16, 32, "f16", "f16", "both", 8, 64), (130, 5, 5, 128, 32, 64, "f32", "f16", "q", 4, 0),
    (61, 8, 2, 128, 16, 16, "f32", "bf16", "k", 0, 8), (19, 32, 8, 128, 256, 128, "bf16", "f32", "both", 16, 0),
    (700, 4, 1, 128, 64, 128, "f16", "bf16", "none", 0, 0), (5, 7, 7, 64, 8, 48, "bf16", "f16", "both", 0, 24),
    (3, 3, 1, 128, 16, 112, "f32", "f32", "both", 12, 4), (4099, 8, 2, 128, 16, 128, "bf16", "bf16", "both", 0, 0),
])
def test_norm_rope(T, H, KV, hd, bs, rot, src, dst, norm, sp, pp):
    q_out, kc, vc, big, qkv, pos, slots, cos, sin, wq, wk = rope_case(T, H, KV, hd, bs, rot, src, dst, norm, sp, pp, seed=T)
    before = [f64(t) for t in (q_out, kc, vc)]
    ops().qk_norm_rope(q_out, kc, vc, qkv, pos, slots, cos, sin, wq, wk)
    check_rope(q_out, kc, vc, qkv, pos, slots, cos, sin, wq, wk, dst, before)
    if pp:  # what lies between the pages is not the cache's
        assert (big[:, :, KV * bs * hd:] == 7).all()


def test_norm_rope_padding_and_missing_pages():
    """Rows without a position are left alone; rows without a page get q only."""
    q_out, kc, vc, _, qkv, pos, slots, cos, sin, wq, wk = rope_case(40, 4, 2, 64, 16, 64, "f32", "f16", "both")
    pos[3], pos[7], pos[39] = -1, cos.shape[0], 2 ** 31 - 1
    slots[4], slots[5], slots[6] = -1, kc.shape[0] * 16, 2 ** 31 - 1
    before = [f64(t) for t in (q_out, kc, vc)]
    ops().qk_norm_rope(q_out, kc, vc, qkv, pos, slots, cos, sin, wq, wk)
    check_rope(q_out, kc, vc, qkv, pos, slots, cos, sin, wq, wk, "f16", before)


def test_norm_rope_zero_rows_and_extremes():
    """A head of zeros stays zero under the norm; no tokens is no work."""
    q_out, kc, vc, _, qkv, pos, slots, cos, sin, wq, wk = rope_case(4, 4, 2, 64, 16, 64, "f32", "f32", "both")
    qkv.zero_()
    ops().qk_norm_rope(q_out, kc, vc, qkv, pos, slots, cos, sin, wq, wk)
    assert (q_out == 0).all()
    e = q_out[:0]
    ops().qk_norm_rope(e, kc, vc, qkv[:0], pos[:0], slots[:0], cos, sin)


# ---------------------------------------------------------------- attention

def attend_case(lens, new, H, KV, hd, bs, dtype, seed=0, extra=3, page_pad=0, q_pad=0, kscale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    need = [-(-n // bs) for n in lens]
    nb = sum(need) + extra
    ids = rng.permutation(nb)
    table = np.full((len(lens), max(need + [1]) + 1), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    big = torch.full((2, nb, KV * bs * hd + page_pad), float("nan"), device="cuda", dtype=DT[dtype])
    kc, vc = (big[i][:, :KV * bs * hd].view(nb, KV, bs, hd) for i in (0, 1))
    # only rows that belong to a sequence hold numbers: the rest of the cache is NaN
    for b, n in enumerate(lens):
        for j in range(need[b]):
            m = min(bs, n - j * bs)
            for c in (kc, vc):
                c[table[b, j], :, :m] = (torch.randn(KV, m, hd, generator=g, device="cuda") * (kscale if c is kc else 1)).to(DT[dtype])
    q_start = np.concatenate([[0], np.cumsum(new)]).astype(np.int64)
    T = int(q_start[-1])
    q = torch.randn(T, H * hd + q_pad, generator=g, device="cuda").to(DT[dtype])[:, :H * hd].unflatten(1, (H, hd))
    return q, kc, vc, table, q_start, np.array(lens, np.int64)


def check_attend(got, q, kc, vc, table, q_start, lens, dtype, scale=None, window=0, rows=None):
    hd = q.shape[2]
    scale = hd ** -0.5 if scale is None else scale
    out, ao, asc, keys, sv = plain.attend(f64(q), f64(kc), f64(vc), table, q_start, lens, scale, window)
    d = DT[dtype]
    # weights: a score is off by (hd + 2) roundings of sum |q k| and enters both the weight and the
    # sum; the running sums add one rounding a key, the exponential two units; half types round each
    # weight once (fp16: at worst 2^-25 absolute below its normal range, on weights whose sum is
    # at least 1); the result is rounded once
    e32 = 2.0 ** -24
    rel = 2 * (hd + 2) * e32 * asc + (keys + 16) * e32 + (u(d) if dtype != "f32" else 0)
    tol = u(d) * np.abs(out) + rel * ao * (1 + u(d)) + (2.0 ** -25 * sv if dtype == "f16" else 0) + 2.0 ** -40
    g = f64(got)
    if rows is not None:
        g, out, tol = g[rows], out[rows], tol[rows]
    bad = ~(np.abs(g - out) <= tol)
    assert not bad.any(), (int(bad.sum()), float(np.nanmax(np.abs(g - out) / tol)), np.argwhere(bad)[:3].tolist())


def run_attend(lens, new, H, KV, hd, bs, dtype, window=0, scale=None, **kw):
    c = attend_case(lens, new, H, KV, hd, bs, dtype, **kw)
    q, kc, vc, table, q_start, ln = c
    out = torch.full(q.shape, 3.0, device="cuda", dtype=q.dtype)
    ops().paged_attention(out, q, kc, vc, i32(table), i32(q_start), i32(ln), scale, window)
    check_attend(out, *c, dtype, scale, window)
    return c, out


TYPES = ["f32", "f16", "bf16"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,KV,hd", [(8, 2, 128), (4, 4, 64), (3, 1, 128), (16, 1, 64), (40, 2, 128)])
@pytest.mark.parametrize("bs", [8, 16, 64])
def test_decode_lengths(dtype, H, KV, hd, bs):
    """One token for each of many sequences, of lengths around the tile and page borders."""
    lens = [1, 2, bs - 1, bs, bs + 1, 63, 64, 65, 127, 128, 129, 200, 511]
    run_attend(lens, [1] * len(lens), H, KV, hd, bs, dtype, seed=bs)


@pytest.mark.parametrize("dtype", TYPES)
def test_decode_long_context_is_split(dtype):
    run_attend([4001], [1], 8, 2, 128, 16, dtype)
    run_attend([3000, 1, 700], [1, 1, 1], 4, 1, 64, 32, dtype, window=1500)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,KV,hd,bs", [(8, 2, 128, 16), (3, 1, 64, 8), (2, 2, 128, 128), (6, 2, 64, 256)])
def test_chunks(dtype, H, KV, hd, bs):
    """Chunks and single tokens together, chunks that are whole sequences, empty requests."""
    lens = [70, 1, 300, 33, 5, 129, 64]
    new = [70, 1, 45, 0, 5, 2, 17]
    run_attend(lens, new, H, KV, hd, bs, dtype, seed=hd + bs)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window", [1, 7, 64, 100, 1000])
def test_windows(dtype, window):
    run_attend([150, 90, 260, 1], [150, 3, 30, 1], 8, 2, 128, 16, dtype, window=window)
    run_attend([150, 90, 260, 1], [1, 1, 1, 1], 4, 1, 64, 16, dtype, window=window)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,new", [([513], [1]), ([140, 200], [140, 61])])
def test_strides_scale_and_large_scores(dtype, lens, new):
    run_attend(lens, new, 8, 2, 128, 16, dtype, scale=0.3, page_pad=64, q_pad=136)
    run_attend(lens, new, 8, 2, 64, 16, dtype, kscale=8.0)  # scores of some tens: weights near 0 and 1
    run_attend(lens, new, 8, 2, 64, 16, dtype, scale=0.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [40, 20, 33, 25]])
def test_missing_pages_and_queries_without_keys(dtype, new):
    """Table entries out of range are not attended; queries before the first token get zeros."""
    lens = [100, 64, 0, 10]
    q, kc, vc, table, q_start, ln = attend_case(lens, new, 8, 2, 128, 16, dtype)
    table[0, 1], table[0, 4], table[1, 0] = -1, kc.shape[0], 2 ** 31 - 1
    out = torch.full(q.shape, 3.0, device="cuda", dtype=q.dtype)
    ops().paged_attention(out, q, kc, vc, i32(table), i32(q_start), i32(ln))
    check_attend(out, q, kc, vc, table, q_start, ln, dtype)
    assert (out[q_start[2]:q_start[3]] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [[1, 1], [70, 9]])
def test_rows_of_no_sequence_stay(dtype, new):
    """Rows before q_start[0] and behind q_start[n] keep what they held; lengths past the table are cut."""
    q, kc, vc, table, q_start, ln = attend_case([90, 40], new, 4, 2, 64, 16, dtype)
    T = q.shape[0]
    qq = torch.cat([q[:2], q, q[:5]])
    out = torch.full(qq.shape, 3.0, device="cuda", dtype=q.dtype)
    ops().paged_attention(out, qq, kc, vc, i32(table), i32(q_start + 2), i32(ln))
    assert (out[:2] == 3).all() and (out[2 + T:] == 3).all()
    check_attend(out[2:2 + T], q, kc, vc, table, q_start, ln, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_value_that_a_query_does_not_attend_to_does_not_reach_it(dtype):
    """Infinity and NaN in K and V of later tokens of the same chunk: the queries before stay clean,
    those behind get what the formula gives."""
    q, kc, vc, table, q_start, ln = attend_case([150, 20], [100, 3], 8, 2, 128, 16, dtype)
    at = 90  # position of the bad key: queries of sequence 0 stand at 50 ..
    vc[table[0, at // 16], 0, at % 16, 5] = float("inf")
    vc[table[0, at // 16], 1, at % 16, 7] = float("nan")
    kc[table[1, 1], 1, 3, :] = float("nan")  # position 19 of sequence 1: its last query's own key
    out = torch.full(q.shape, 3.0, device="cuda", dtype=q.dtype)
    ops().paged_attention(out, q, kc, vc, i32(table), i32(q_start), i32(ln))
    clean = [t for t in range(103) if t < 40 or 100 <= t < 102]
    check_attend(out, q, kc, vc, table, q_start, ln, dtype, rows=clean)
    o = out.float().cpu().numpy()
    assert np.isposinf(o[40:100, :4, 5]).all() and np.isnan(o[40:100, 4:, 7]).all()
    assert np.isfinite(o[40:100, :4, 6]).all() and np.isfinite(o[40:100, 4:, 6]).all()
    assert np.isnan(o[102, 4:]).all() and np.isfinite(o[102, :4]).all()


def test_attention_of_nothing():
    q, kc, vc, table, q_start, ln = attend_case([20], [1], 4, 2, 64, 16, "f16")
    ops().paged_attention(q[:0].contiguous(), q[:0], kc, vc, i32(table), i32([0, 0]), i32(ln))
    out = torch.full(q.shape, 3.0, device="cuda", dtype=q.dtype)
    ops().paged_attention(out, q, kc, vc, i32(table[:0]), i32([0]), i32([]))
    assert (out == 3).all()


# ---------------------------------------------------------------- sampling

def f32(v):
    return torch.as_tensor(np.asarray(v, np.float32)).cuda()


def run_sample(x, r, T, k=None, p=None, m=None, dtype="f32"):
    t = torch.as_tensor(np.asarray(x, np.float32)).cuda().to(DT[dtype])
    xs = t.float().cpu().numpy()
    got = ops().sample_rows(t, f32(r), f32(T), None if k is None else i32(k), None if p is None else f32(p),
                            None if m is None else f32(m)).cpu().numpy()
    want = [plain.sample(xs[i], r[i], T[i], None if k is None else k[i], None if p is None else p[i],
                         None if m is None else m[i]) for i in range(len(xs))]
    np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 2, 31, 777, 1000, 1025, 32000, 50003])
@pytest.mark.parametrize("mode", ["plain", "k", "p", "m", "all"])
def test_sample_matches_the_sorted_form(dtype, n, mode):
    rng = np.random.default_rng(n)
    rows = 9
    x = rng.standard_normal((rows, n)) * 2.5
    r = rng.random(rows, np.float32)
    T = rng.uniform(0.2, 1.5, rows).astype(np.float32)
    k = rng.integers(-1, max(2, min(n + 2, 300)), rows) if mode in ("k", "all") else None
    p = rng.uniform(0.1, 1.02, rows).astype(np.float32) if mode in ("p", "all") else None
    m = rng.uniform(-0.02, 0.3, rows).astype(np.float32) if mode in ("m", "all") else None
    run_sample(x, r, T, k, p, m, dtype)


@pytest.mark.parametrize("n", [3, 40, 2049, 32000])
def test_sample_ties_go_to_the_lowest_index(n):
    """Few distinct logits: the cuts of top-k and top-p fall inside runs of equal values."""
    rng = np.random.default_rng(n)
    rows = 40
    x = rng.integers(0, 4, (rows, n)).astype(np.float32) * 0.5
    x[0] = 1.0
    x[1, : n // 2] = -0.0
    x[1, n // 2:] = 0.0
    r = rng.random(rows, np.float32)
    T = np.where(np.arange(rows) % 5 == 4, 0.0, rng.uniform(0.5, 1.5, rows)).astype(np.float32)
    k = rng.integers(0, n + 1, rows)
    p = rng.uniform(0.05, 1.0, rows).astype(np.float32)
    run_sample(x, r, T, k, None, None)
    run_sample(x, r, T, None, p, None)
    run_sample(x, r, T, k, p, None)


def test_sample_border_settings():
    rng = np.random.default_rng(5)
    n = 1500
    x = rng.standard_normal((1, n)).astype(np.float32) * 2
    x[0, 100:400] = -np.inf
    big = np.nextafter(np.float32(1), np.float32(0))
    cases = []
    for r in (0.0, 0.5, float(big)):
        for T in (0.0, -1.0, float("nan"), 1e-6, 1e-30, 1.0, 100.0, 1e30):
            for k in (0, 1, 2, n - 1, n, n + 5, -3):
                for p in (-1.0, 0.0, 1e-9, 0.5, float(big), 1.0, 2.0, float("nan")):
                    cases.append((r, T, k, p, rng.choice([0.0, 1.0, -1.0, 0.5, float("nan")])))
    r, T, k, p, m = (np.array(v) for v in zip(*cases))
    run_sample(np.repeat(x, len(cases), 0), r.astype(np.float32), T.astype(np.float32), k, p.astype(np.float32),
               m.astype(np.float32))


@pytest.mark.parametrize("T", [0.0, 0.7])
def test_sample_rows_that_cannot_be_sampled(T):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((8, 2000)).astype(np.float32)
    x[0, 5] = np.nan
    x[1, 0] = np.nan
    x[2, 7] = np.inf
    x[3] = -np.inf
    x[4] = np.nan
    x[5, 1:] = -np.inf
    x[6, :-1] = -np.inf
    x[7] = -3e38
    r = np.full(8, 0.3, np.float32)
    run_sample(x, r, np.full(8, T), [5] * 8, [0.9] * 8, [0.01] * 8)
    run_sample(x, r, np.full(8, T))


@pytest.mark.parametrize("n", [4093, 4096, 45000, 128001, 270000])
@pytest.mark.parametrize("off", [0, 1, 3])
def test_sample_sizes_and_alignments(n, off):
    """Rows around a segment's size, rows that do not fit shared memory, rows longer than the cells; rows
    that begin off 16 bytes.  Peaked and flat rows, with few and many logits kept."""
    rng = np.random.default_rng(n + off)
    x = torch.as_tensor((rng.standard_normal((4, n + 5)) * np.array([[0.3], [1.0], [3.0], [8.0]])).astype(np.float32)).cuda()
    v = x[:, off:off + n]
    xs = v.cpu().numpy()
    for k, p, m in ((None, None, None), (40, 0.9, 0.02), (3000, 0.97, None), (None, 0.5, None), (None, 0.999, 1e-5)):
        r, T = rng.random(4).astype(np.float32), rng.uniform(0.5, 1.2, 4).astype(np.float32)
        full = lambda a, f: None if a is None else f([a] * 4)
        got = ops().sample_rows(v, f32(r), f32(T), full(k, i32), full(p, f32), full(m, f32)).cpu().numpy()
        want = [plain.sample(xs[i], r[i], T[i], k, p, m) for i in range(4)]
        np.testing.assert_array_equal(got, want)


def test_sample_strided_rows():
    rng = np.random.default_rng(8)
    x = torch.as_tensor(rng.standard_normal((6, 1111)).astype(np.float32)).cuda()
    v = x[:, 7:1008]
    r, T = rng.random(6).astype(np.float32), np.full(6, 0.8, np.float32)
    got = ops().sample_rows(v, f32(r), f32(T)).cpu().numpy()
    want = [plain.sample(v[i].cpu().numpy(), r[i], T[i]) for i in range(6)]
    np.testing.assert_array_equal(got, want)
    assert ops().sample_rows(x[:0], f32([]), f32([])).numel() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n", [(700, 257), (310, 1500), (160, 30000)])
def test_sample_more_rows_than_run_at_once(dtype, rows, n):
    """Greedy rows, short lists, cuts by top-p and none, side by side: every row gets its answer."""
    rng = np.random.default_rng(rows)
    x = rng.standard_normal((rows, n)) * 2
    kind = rng.integers(0, 4, rows)
    T = np.where(kind == 0, 0.0, rng.uniform(0.4, 1.3, rows)).astype(np.float32)
    k = np.where(kind == 1, rng.integers(1, 300, rows), 0)
    p = np.where(kind == 2, rng.uniform(0.3, 0.99, rows), 1.0).astype(np.float32)
    run_sample(x, rng.random(rows, np.float32), T, k, p, None, dtype)
    run_sample(x, rng.random(rows, np.float32), T, None, p, None, dtype)


# ---------------------------------------------------------------- together

def step_state(dtype, seed):
    """Three requests of a two-layer toy: what a serving loop holds."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    H, KV, hd, bs, V = 8, 2, 128, 16, 500
    s = dict(H=H, KV=KV, hd=hd, bs=bs, V=V, dtype=dtype)
    s["table"] = torch.full((3, 8), -1, dtype=torch.int32, device="cuda")
    s["free"] = torch.randperm(24, generator=g, device="cuda").to(torch.int32)
    s["kc"] = torch.full((2, 24, KV, bs, hd), float("nan"), device="cuda", dtype=DT[dtype])
    s["vc"] = torch.full_like(s["kc"], float("nan"))
    ang = torch.arange(128, device="cuda")[:, None].double() * 1e4 ** (-torch.arange(hd // 2, device="cuda") / (hd / 2))
    s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    s["wq"], s["wk"] = (1 + 0.1 * torch.randn(2, hd, generator=g, device="cuda")).unbind()
    s["wq"], s["wk"] = s["wq"].contiguous(), s["wk"].contiguous()
    s["w_qkv"] = torch.randn(2, 64, (H + 2 * KV) * hd, generator=g, device="cuda") / 8
    s["w_o"] = torch.randn(2, H * hd, 64, generator=g, device="cuda") / 32
    s["head"] = torch.randn(64, V, generator=g, device="cuda") / 4
    s["embed"] = torch.randn(V, 64, generator=g, device="cuda")
    return s


def serve(s, ids, cached, new, n_rows, r, used):
    """One step; ids [n_rows].  Returns (tokens of each request's last row, counts)."""
    o = ops()
    q_start, lens, pos, slots, counts = o.paged_plan(s["table"], cached, new, s["free"][used:], s["bs"], n_rows)
    x = s["embed"][ids]
    for layer in range(2):
        qkv = (x @ s["w_qkv"][layer]).contiguous()
        q = torch.zeros(n_rows, s["H"], s["hd"], device="cuda", dtype=DT[s["dtype"]])
        a = torch.zeros_like(q)
        o.qk_norm_rope(q, s["kc"][layer], s["vc"][layer], qkv, pos, slots, s["cos"], s["sin"], s["wq"], s["wk"])
        o.paged_attention(a, q, s["kc"][layer], s["vc"][layer], s["table"], q_start, lens, window=40)
        x = x + a.flatten(1).float() @ s["w_o"][layer]
    logits = x[(q_start[1:] - 1).clamp(min=0).long()] @ s["head"]
    n = logits.shape[0]
    tok = o.sample_rows(logits, r, torch.full((n,), 0.9, device="cuda"), torch.full((n,), 40, dtype=torch.int32, device="cuda"),
                        torch.full((n,), 0.95, device="cuda"), torch.full((n,), 0.01, device="cuda"))
    return tok, logits, counts


@pytest.mark.parametrize("dtype", TYPES)
def test_a_run_of_steps_is_the_same_in_chunks_and_token_by_token(dtype):
    """The prompts of three requests go in at once, or in pieces beside single tokens: the logits of
    their last tokens agree (the pages, the masks and the splits of the two ways differ)."""
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, 500, n) for n in (37, 5, 61)]

    def feed(pieces):
        s, used, at, logits = step_state(dtype, 4), 0, [0, 0, 0], [None] * 3
        for new in pieces:
            ids = np.concatenate([prompts[b][at[b]:at[b] + n] for b, n in enumerate(new)] + [[0, 0]])  # 2 padding rows
            _, lg, counts = serve(s, torch.as_tensor(ids).cuda().long(), i32(at), i32(new), len(ids), f32([0.5] * 3), used)
            used += int(counts[0])
            assert int(counts[1]) == 0
            at = [a + n for a, n in zip(at, new)]
            for b in range(3):
                if new[b] and at[b] == len(prompts[b]):
                    logits[b] = f64(lg[b])
        assert used == sum(-(-len(p) // 16) for p in prompts)
        return np.stack(logits)

    whole = feed([[37, 5, 61]])
    pieces = feed([[20, 1, 0], [1, 1, 50], [1, 1, 1], [15, 2, 10]])
    # each way's rows pass two layers whose q, k, v and weights round to the type (6 roundings a
    # layer, each on values of the residual's size or below, through maps of gain near 1)
    tol = {"f32": 2e-4, "f16": 24 * 2.0 ** -11, "bf16": 24 * 2.0 ** -8}[dtype]
    assert np.abs(whole - pieces).max() <= tol * np.abs(whole).max()


def test_a_captured_step_replays_with_new_lengths():
    """The whole step in one CUDA graph: replays read the lengths, tables and draws of the moment."""
    s, e = step_state("f16", 9), step_state("f16", 9)
    n_rows = 12
    ids = torch.zeros(n_rows, dtype=torch.long, device="cuda")
    cached, new, r = i32([0, 0, 0]), i32([5, 1, 3]), f32([0.1, 0.5, 0.9])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm up aside, on a state of its own
        serve(step_state("f16", 9), ids, cached, new, n_rows, r, 0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tok, logits, counts = serve(s, ids, cached, new, n_rows, r, 0)
    rng = np.random.default_rng(2)
    at, free = np.zeros(3, int), s["free"].clone()
    used = 0
    for new_np in ([5, 1, 3], [1, 1, 10], [4, 0, 1], [1, 1, 1], [0, 7, 2]):
        ids.copy_(torch.as_tensor(rng.integers(0, 500, n_rows)).cuda())
        cached.copy_(i32(at))
        new.copy_(i32(new_np))
        r.copy_(f32(rng.random(3)))
        s["free"].copy_(torch.roll(free, -used))
        graph.replay()
        want_tok, want, want_counts = serve(e, ids, i32(at), i32(new_np), n_rows, r, used)
        live = [b for b in range(3) if new_np[b]]
        assert torch.equal(logits[live], want[live]) and torch.equal(tok[live], want_tok[live])
        assert int(counts[0]) == int(want_counts[0])
        used += int(counts[0])
        at += np.array(new_np)


def test_another_stream_and_repeated_calls_agree():
    q, kc, vc, table, q_start, ln = attend_case([700, 90], [1, 60], 8, 2, 128, 16, "bf16")
    args = (i32(table), i32(q_start), i32(ln))
    outs = []
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for n in range(6):
        with torch.cuda.stream(side if n % 2 else torch.cuda.current_stream()):
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            ops().paged_attention(out, q, kc, vc, *args)
            outs.append(out)
    torch.cuda.synchronize()
    assert all(torch.equal(outs[0], x) for x in outs[1:])


# ---------------------------------------------------------------- more of attention

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_seq", [257, 700])
@pytest.mark.parametrize("most", [1, 12])
def test_more_sequences_than_a_block_has_threads(dtype, n_seq, most):
    """Decode steps (most = 1) and short chunks, some without tokens."""
    rng = np.random.default_rng(n_seq + most)
    new = rng.integers(0, most + 1, n_seq)
    lens = new + rng.integers(0, 30, n_seq)
    run_attend(lens.tolist(), new.tolist(), 4, 1, 64, 8, dtype, seed=most)


@pytest.mark.parametrize("dtype", TYPES)
def test_more_row_tiles_than_a_warp_has_lanes(dtype):
    run_attend([1200, 3], [1100, 1], 8, 1, 64, 64, dtype)
    run_attend([300] + [5] * 59, [130] + [1] * 59, 4, 1, 64, 16, dtype)  # few rows a sequence on average


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,KV", [(24, 1), (100, 1), (14, 2)])
def test_groups_of_odd_sizes(dtype, H, KV):
    run_attend([77, 5, 300], [1, 1, 1], H, KV, 64, 16, dtype)
    run_attend([77, 5, 300], [13, 5, 2], H, KV, 128, 32, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [[1, 1], [90, 33]])
def test_signs_and_sizes_of_the_scale(dtype, new):
    """A negative scale, a tiny one, and 0 with scores that are far from 1: all weights alike."""
    run_attend([90, 333], new, 8, 2, 128, 16, dtype, scale=-0.2)
    run_attend([90, 333], new, 8, 2, 64, 16, dtype, scale=1e-38)
    run_attend([90, 333], new, 8, 2, 64, 16, dtype, scale=0.0, kscale=1e4 if dtype == "f16" else 1e33)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [[1, 1, 1], [80, 20, 33]])
@pytest.mark.parametrize("window", [5, 40])
def test_missing_pages_under_a_window(dtype, new, window):
    q, kc, vc, table, q_start, ln = attend_case([200, 64, 90], new, 8, 2, 64, 8, dtype)
    table[0, 23:25], table[0, 15], table[1, 7], table[2, 3:12] = -1, kc.shape[0], -2 ** 31, -1
    out = torch.full(q.shape, 3.0, device="cuda", dtype=q.dtype)
    ops().paged_attention(out, q, kc, vc, i32(table), i32(q_start), i32(ln), None, window)
    check_attend(out, q, kc, vc, table, q_start, ln, dtype, window=window)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_offsets_past_32_bits(dtype):
    """Pages 2^25 elements apart: the last ones lie more than 2^31 elements behind the first.  K and V are
    written there by qk_norm_rope and read by both kinds of attention."""
    KV, hd, bs, n_blocks, stride, H = 1, 64, 8, 68, 1 << 25, 4
    big = torch.zeros(2 * n_blocks * stride, device="cuda", dtype=DT[dtype])
    kc, vc = (big[i * n_blocks * stride:][:n_blocks * stride].view(n_blocks, stride)[:, :KV * bs * hd].view(n_blocks, KV, bs, hd)
              for i in (0, 1))
    n = 540
    g = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn(n, (H + 2 * KV) * hd, generator=g, device="cuda")
    pos = torch.arange(n, device="cuda", dtype=torch.int32)
    table = torch.arange(n_blocks, device="cuda", dtype=torch.int32)[None]
    cos, sin = torch.ones(n, 32, device="cuda"), torch.zeros(n, 32, device="cuda")
    q = torch.empty(n, H, hd, device="cuda", dtype=DT[dtype])
    ops().qk_norm_rope(q, kc, vc, qkv, pos, pos, cos, sin)
    assert torch.equal(kc.reshape(-1, hd)[:n], qkv[:, H * hd:(H + 1) * hd].to(DT[dtype]))
    assert torch.equal(vc.reshape(-1, hd)[:n], qkv[:, (H + 1) * hd:].to(DT[dtype]))
    small = kc.contiguous(), vc.contiguous()
    for rows in (1, 200):
        qq, args = q[n - rows:], (table, i32([0, rows]), i32([n]))
        a, b = torch.empty_like(qq), torch.empty_like(qq)
        ops().paged_attention(a, qq, kc, vc, *args)
        ops().paged_attention(b, qq, *small, *args)
        assert torch.equal(a, b)
        check_attend(a, qq, *small, np.arange(n_blocks)[None], np.array([0, rows]), np.array([n]), dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_two_streams_at_once(dtype):
    """Steps of two batches in two streams, each call with a workspace of its own, give what they give alone."""
    cases = [attend_case([900, 90, 14], [1, 1, 1], 8, 2, 128, 16, dtype, seed=1),
             attend_case([700, 260], [300, 60], 8, 2, 128, 16, dtype, seed=2)]
    args = [(i32(t), i32(s), i32(n)) for _, _, _, t, s, n in cases]
    want = []
    for (q, kc, vc, *_), a in zip(cases, args):
        want.append(torch.empty(q.shape, device="cuda", dtype=q.dtype))
        ops().paged_attention(want[-1], q, kc, vc, *a)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(20):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                q, kc, vc = cases[k][:3]
                outs[k].append(torch.empty(q.shape, device="cuda", dtype=q.dtype))
                ops().paged_attention(outs[k][-1], q, kc, vc, *args[k])
    torch.cuda.synchronize()
    for k in (0, 1):
        assert all(torch.equal(x, want[k]) for x in outs[k])


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("tokens", [1, 64])
def test_workspaces_that_do_not_do_are_refused(dtype, tokens):
    import ctypes
    from torchless_b200 import lib, tl_paged_cache
    L = lib()
    kc = torch.zeros(4, 1, 16, 64, device="cuda", dtype=[torch.float32, torch.float16][dtype])
    q = torch.zeros(tokens, 4, 64, device="cuda", dtype=kc.dtype)
    out = torch.full_like(q, 3.0)
    table, start, lens = i32([[0, 1, 2, 3]]), i32([0, tokens]), i32([64])
    c = tl_paged_cache(kc.data_ptr(), kc.data_ptr(), 4, 1, 16, 64, 16 * 64, dtype)
    need = ctypes.c_size_t()
    assert L.tl_paged_attention_workspace(ctypes.byref(c), tokens, 4, 1, 4, ctypes.byref(need)) == 0
    ws = torch.zeros(need.value + 16, device="cuda", dtype=torch.uint8)

    def call(p, size):
        return L.tl_paged_attention(out.data_ptr(), q.data_ptr(), 256, ctypes.byref(c), table.data_ptr(), 4,
                                    start.data_ptr(), lens.data_ptr(), 1, tokens, 4, 0.1, 0, p, size, None)
    assert call(None, need.value) and call(ws.data_ptr(), need.value - 1) and call(ws.data_ptr() + 8, need.value)
    torch.cuda.synchronize()
    assert (out == 3).all()
    assert call(ws.data_ptr(), need.value) == 0
    torch.cuda.synchronize()
    assert (out == 0).all()


def test_two_tokens_with_one_slot():
    """The slot holds numbers of the two; nothing else changes."""
    q_out, kc, vc, _, qkv, pos, slots, cos, sin, wq, wk = rope_case(30, 4, 2, 64, 16, 64, "f32", "f32", "none")
    slots[9] = slots[4]
    before = [f64(t) for t in (q_out, kc, vc)]
    ops().qk_norm_rope(q_out, kc, vc, qkv, pos, slots, cos, sin)
    got = []
    for drop in (4, 9):  # either alone
        kk, vv = kc.clone().fill_(7), vc.clone().fill_(7)
        s = slots.clone()
        s[drop] = -1
        ops().qk_norm_rope(torch.empty_like(q_out), kk, vv, qkv, pos, s, cos, sin)
        got.append((kk, vv))
    for x, a, b in zip((kc, vc), got[0], got[1]):
        assert ((x == a) | (x == b)).all()
    assert before[1].shape == kc.shape
