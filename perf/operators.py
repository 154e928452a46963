"""The operators of one serving step over a paged KV cache, measured apart.

A step that mixes prompt chunks and decoding requests runs, in this order:

* ``plan``    block tables and slot maps from the request lengths (once a step);
* ``rope``    norms of the q and k heads, rotation, write into the pages (once a layer);
* ``attend``  attention of the new tokens over the pages (once a layer);
* ``sample``  temperature, top-k, top-p and min-p per request (once a step).

Where ``own`` is false each is computed in its plain form by elementary torch
operations in 32 bits (64 where a border decides about a whole number).
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
DEV = "cuda"


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------

def listed():
    heads = dict(H=32, KV=8, hd=128)  # the 7B configuration of this repository
    return [
        # one new token for each of 64 requests: every decode step of a server plans this
        dict(name="plan decode 64", op="plan", B=64, ctx=4096, new=1, page=16, pad=0),
        # a full step of prompt chunks of all sizes, with padding rows of a fixed token budget
        dict(name="plan chunks 16384", op="plan", B=509, ctx=8192, new=61, page=16, pad=131),
        # one request decoding, heads normalised: the smallest call
        dict(name="rope 1 bf16 norm", op="rope", T=1, **heads, page=16, rot=128, src="bf16", dst="bf16", norm=True),
        # 64 requests decoding from the fp32 rows of a GEMM into fp16 pages, rotation alone
        dict(name="rope 64 f32 to f16", op="rope", T=64, **heads, page=16, rot=128, src="f32", dst="f16", norm=False),
        # a long prompt pass
        dict(name="rope 16381 bf16 norm", op="rope", T=16381, **heads, page=64, rot=128, src="bf16", dst="bf16", norm=True),
        # one request with a long context: few rows, a long axis
        dict(name="decode 1x8192 bf16", op="attend", B=1, q=1, ctx=8192, ragged=False, **heads, page=16, dtype="bf16", window=0),
        # the batched decode configuration, requests of unlike lengths
        dict(name="decode 64x4096 f16 ragged", op="attend", B=64, q=1, ctx=4096, ragged=True, **heads, page=16, dtype="f16", window=0),
        # the same with the fp32 cache that the framework's own batches keep
        dict(name="decode 64x4096 f32", op="attend", B=64, q=1, ctx=4096, ragged=False, **heads, page=32, dtype="f32", window=0),
        # the second half of a 4096-token prompt under the sliding window of the configuration
        dict(name="chunk 2048 of 4096 bf16", op="attend", B=1, q=2048, ctx=4096, ragged=False, **heads, page=64, dtype="bf16", window=4096),
        # chunks and single tokens together, odd lengths, pages that end inside a tile
        dict(name="chunks 9x<=389 f16 ragged", op="attend", B=9, q=389, ctx=5003, ragged=True, **heads, page=16, dtype="f16", window=0),
        # one request's token
        dict(name="sample 1x32000", op="sample", B=1, V=32000, mode="all"),
        # a server's step: every request with its own settings
        dict(name="sample 256x32000 mixed", op="sample", B=256, V=32000, mode="mixed"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "rope", "rope", "attend", "attend", "attend", "sample", "sample"])
    page = rng.choice([16, 32, 64])
    if op == "plan":
        B = _log(rng, 1, 700)
        return dict(op=op, B=B, ctx=_log(rng, 16, 8192), new=_log(rng, 1, max(1, 32000 // B)), page=page, pad=rng.choice([0, rng.randint(1, 300)]))
    if op == "rope":
        hd = rng.choice([64, 128])
        KV = rng.choice([1, 2, 4, 8])
        src = rng.choice(["f32", "f16", "bf16"])
        return dict(op=op, T=_log(rng, 1, 8000), H=KV * rng.choice([1, 2, 4, 5]), KV=KV, hd=hd, page=page, rot=rng.choice([hd, hd, hd // 2]),
                    src=src, dst=rng.choice([src, "f16", "bf16"]), norm=rng.random() < 0.7)
    if op == "attend":
        KV = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 3, 4, 4, 8])
        hd = rng.choice([64, 128, 128])
        q = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 17, 700)])
        ctx = _log(rng, max(32, q), 8192)
        q = min(q, max(1, int(100e9 / (4 * ctx * group * KV * hd))))
        most = max(1, int(min(100e9 / (4 * q * ctx * group * KV * hd), 60e6 / (q * ctx * group * KV / 8), 64 * 4096 / ctx)))
        return dict(op=op, B=_log(rng, 1, min(64, most)), q=q, ctx=ctx, ragged=rng.random() < 0.7, H=KV * group, KV=KV, hd=hd, page=page,
                    dtype=rng.choice(["f32", "f16", "bf16"]), window=rng.choice([0, 0, _log(rng, 16, 4096)]))
    return dict(op=op, B=_log(rng, 1, 200), V=_log(rng, 777, 40000), mode=rng.choice(["all", "mixed", "top_p", "plain"]))


def _lengths(case):
    """Cached and new tokens of every request: a matter of the case alone."""
    rng = random.Random("%(op)s %(B)d %(ctx)d" % case)
    cached, new = [], []
    for b in range(case["B"]):
        if case["op"] == "plan":
            n = case["new"] if case["new"] == 1 else rng.randint(0, case["new"])
            c = _log(rng, 1, case["ctx"]) - 1
        elif case["ragged"] and b:
            n = rng.choice([1, rng.randint(1, case["q"])])
            c = _log(rng, max(n, case["ctx"] // 16), case["ctx"]) - n
        else:
            n, c = case["q"], case["ctx"] - case["q"]
        cached.append(c)
        new.append(n)
    return cached, new


# --------------------------------------------------------------------------
# what a user has in hand
# --------------------------------------------------------------------------

def _pages(lens, page, gen):
    """A table of pages in random order for sequences of `lens` tokens, and their number with some to spare."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + 7
    ids = torch.randperm(total, generator=gen, device=DEV).to(torch.int32)
    width = max(max(need), 1)
    col = torch.arange(width, device=DEV)
    n = torch.tensor(need, device=DEV)
    first = torch.cumsum(n, 0) - n
    src = first[:, None] + col
    table = torch.where(col < n[:, None], ids[src.clamp(max=total - 1)], torch.full_like(src, -1, dtype=torch.int32))
    return table.contiguous(), total


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32 if dtype == torch.float32 else dtype)

    s = dict(case)
    if case["op"] == "plan":
        cached, new = _lengths(case)
        page = case["page"]
        have = [-(-c // page) for c in cached]
        need = [-(-(c + n) // page) for c, n in zip(cached, new)]
        width, total = max(max(need), 1), sum(need) + 100
        ids = torch.randperm(total, generator=gen, device=DEV).to(torch.int32)
        col = torch.arange(width, device=DEV)
        h = torch.tensor(have, device=DEV)
        src = (torch.cumsum(h, 0) - h)[:, None] + col
        s["table"] = torch.where(col < h[:, None], ids[src.clamp(max=total - 1)], torch.full_like(src, -1, dtype=torch.int32)).contiguous()
        s["free"] = ids[sum(have):].contiguous()
        s["cached"], s["new_tokens"], s["T"] = _ints(cached), _ints(new), sum(new) + case["pad"]
    elif case["op"] == "rope":
        T, H, KV, hd, page = case["T"], case["H"], case["KV"], case["hd"], case["page"]
        blocks = -(-T // page) + 3
        s["qkv"] = randn(T, (H + 2 * KV) * hd, dtype=DTYPES[case["src"]])
        s["positions"] = torch.randint(0, 4096, (T,), generator=gen, device=DEV, dtype=torch.int32)
        s["slots"] = torch.randperm(blocks * page, generator=gen, device=DEV)[:T].to(torch.int32)
        inv = 10000.0 ** (-torch.arange(case["rot"] // 2, device=DEV, dtype=torch.float64) / (case["rot"] // 2))
        ang = torch.arange(4096, device=DEV, dtype=torch.float64)[:, None] * inv
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
        s["wq"] = 1 + 0.2 * randn(hd) if case["norm"] else None
        s["wk"] = 1 + 0.2 * randn(hd) if case["norm"] else None
        s["k_cache"] = torch.zeros(blocks, KV, page, hd, device=DEV, dtype=DTYPES[case["dst"]])
        s["v_cache"] = torch.zeros_like(s["k_cache"])
    elif case["op"] == "attend":
        cached, new = _lengths(case)
        dtype = DTYPES[case["dtype"]]
        lens = [c + n for c, n in zip(cached, new)]
        s["table"], blocks = _pages(lens, case["page"], gen)
        s["q_in"] = randn(sum(new), case["H"], case["hd"], dtype=dtype)
        s["k_cache"] = randn(blocks, case["KV"], case["page"], case["hd"], dtype=dtype)
        s["v_cache"] = randn(blocks, case["KV"], case["page"], case["hd"], dtype=dtype)
        start = [0]
        for n in new:
            start.append(start[-1] + n)
        s["q_start"], s["seq_lens"] = _ints(start), _ints(lens)
        s["max_q"] = max(new)
    else:
        B, V = case["B"], case["V"]
        s["logits"] = 2.5 * randn(B, V)

        def uniform(lo, hi):
            return lo + (hi - lo) * torch.rand(B, generator=gen, device=DEV)

        s["r"] = torch.rand(B, generator=gen, device=DEV)
        s["temperature"] = uniform(0.3, 1.3)
        k, p, m = torch.randint(1, 200, (B,), generator=gen, device=DEV), uniform(0.5, 0.99), uniform(0.0, 0.1)
        if case["mode"] == "mixed":  # each setting is off in some rows, and some rows are greedy
            off = torch.rand(4, B, generator=gen, device=DEV)
            k = torch.where(off[0] < 0.4, torch.zeros_like(k), k)
            p = torch.where(off[1] < 0.4, torch.ones_like(p), p)
            m = torch.where(off[2] < 0.4, torch.zeros_like(m), m)
            s["temperature"] = torch.where(off[3] < 0.1, torch.zeros_like(m), s["temperature"])
        s["top_k"] = k.to(torch.int32) if case["mode"] in ("all", "mixed") else None
        s["top_p"] = p if case["mode"] != "plain" else None
        s["min_p"] = m if case["mode"] in ("all", "mixed") else None
    return s


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

def run(s):
    return {"plan": _plan, "rope": _rope, "attend": _attend, "sample": _sample}[s["op"]](s)


def _plan(s):
    if own:
        from torchless_b200 import ops
        q_start, seq_lens, positions, slots, counts = ops.paged_plan(s["table"], s["cached"], s["new_tokens"], s["free"], s["page"], s["T"])
        return s["table"], q_start, seq_lens, positions, slots, counts
    table, free, page, T = s["table"], s["free"], s["page"], s["T"]
    width = table.shape[1]
    cached, new = s["cached"].long(), s["new_tokens"].long()
    q_start = torch.nn.functional.pad(torch.cumsum(new, 0), (1, 0)).clamp(max=T)
    seq_lens = cached + q_start.diff()
    have = (cached + page - 1) // page
    need = (((seq_lens + page - 1) // page).clamp(max=width) - have).clamp(min=0)
    end = torch.cumsum(need, 0)
    j = torch.arange(width, device=DEV) - have[:, None]
    src = (end - need)[:, None] + j
    ids = torch.where(src < free.numel(), free[src.clamp(0, free.numel() - 1)], -1)
    table.copy_(torch.where((j >= 0) & (j < need[:, None]), ids, table))
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(q_start[1:], t, right=True)
    inside = b < cached.numel()
    b = b.clamp(max=cached.numel() - 1)
    pos = cached[b] + t - q_start[b]
    blk = table[b, (pos // page).clamp(max=width - 1)].long()
    slots = torch.where(inside & (pos // page < width) & (blk >= 0), blk * page + pos % page, -1)
    positions = torch.where(inside, pos, -1)
    counts = torch.stack([end[-1].clamp(max=free.numel()), (end[-1] - free.numel()).clamp(min=0)])
    return table, q_start.int(), seq_lens.int(), positions.int(), slots.int(), counts.int()


def _rope(s):
    H, KV, hd = s["H"], s["KV"], s["hd"]
    T = s["qkv"].shape[0]
    kc, vc = s["k_cache"], s["v_cache"]
    if own:
        from torchless_b200 import ops
        q_out = torch.empty(T, H, hd, dtype=kc.dtype, device=DEV)
        ops.qk_norm_rope(q_out, kc, vc, s["qkv"], s["positions"], s["slots"], s["cos"], s["sin"], s["wq"], s["wk"], 1e-5)
        return q_out, kc, vc
    x = s["qkv"].float().view(T, H + 2 * KV, hd)
    cos, sin = s["cos"][s["positions"].long()][:, None], s["sin"][s["positions"].long()][:, None]

    def turned(x, w):
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w
        h = s["rot"] // 2
        a, b = x[..., :h], x[..., h:2 * h]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., 2 * h:]], -1).to(kc.dtype)

    q_out = turned(x[:, :H], s["wq"])
    page, off = s["slots"].long() // s["page"], s["slots"].long() % s["page"]
    kc[page, :, off] = turned(x[:, H:H + KV], s["wk"])
    vc[page, :, off] = x[:, H + KV:].to(vc.dtype)
    return q_out, kc, vc


def _attend(s):
    q, kc, vc = s["q_in"], s["k_cache"], s["v_cache"]
    if own:
        from torchless_b200 import ops
        out = torch.empty_like(q)
        ops.paged_attention(out, q, kc, vc, s["table"], s["q_start"], s["seq_lens"], window=s["window"])
        return out
    T, H, hd = q.shape
    B, KV, n, start, lens = s["B"], s["KV"], s["max_q"], s["q_start"].long(), s["seq_lens"].long()
    pages = s["table"].clamp(min=0).long()
    k, v = (c[pages].transpose(1, 2).reshape(B, KV, -1, hd).float() for c in (kc, vc))
    i = torch.arange(n, device=DEV)
    x = q[(start[:-1, None] + i).clamp(max=T - 1)].float()  # [B, n, H, hd]
    x = x.view(B, n, KV, H // KV, hd).permute(0, 2, 3, 1, 4).reshape(B, KV, -1, hd)
    scores = (x @ k.transpose(-1, -2)).view(B, KV, H // KV, n, -1) * hd ** -0.5
    at = (lens - start.diff())[:, None] + i  # the queries' positions
    j = torch.arange(k.shape[2], device=DEV)
    seen = (j <= at[..., None]) & (j < lens[:, None, None])
    if s["window"]:
        seen &= j > at[..., None] - s["window"]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True).clamp(min=-1e30)
    e = scores.exp_()
    total = e.sum(-1, keepdim=True)
    o = (e.view(B, KV, -1, k.shape[2]) @ v).view(B, KV, H // KV, n, hd) / total.clamp(min=1e-30)
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(start[1:], t, right=True)
    return o[b, :, :, t - start[b]].reshape(T, H, hd).to(q.dtype)


def _sample(s):
    x, r, T, k, p, m = s["logits"], s["r"], s["temperature"], s["top_k"], s["top_p"], s["min_p"]
    if own:
        from torchless_b200 import ops
        return ops.sample_rows(x, r, T, k, p, m)
    B, V = x.shape
    # 64 bits: a running sum next to a border decides which token it is
    ordered, index = torch.sort(x, dim=-1, descending=True, stable=True)
    greedy = (T <= 0)[:, None]
    t = torch.where(greedy, torch.ones_like(T)[:, None], T[:, None]).double()
    w = torch.exp((ordered.double() - ordered[:, :1].double()) / t)
    place = torch.arange(V, device=DEV)
    keep = torch.ones_like(w, dtype=torch.bool)
    if k is not None:
        keep &= (place < k[:, None]) | (k <= 0)[:, None]
    if p is not None:
        sums = torch.cumsum(w * keep, -1)
        keep &= (sums - w < p[:, None].double() * sums[:, -1:]) | (p >= 1)[:, None]
    if m is not None:
        keep &= w >= m[:, None].double()
    keep[:, 0] = True
    kept = torch.zeros_like(w).scatter_(1, index, w * keep)
    sums = torch.cumsum(kept, -1)
    reached = (sums >= r[:, None].double() * sums[:, -1:]) & (kept > 0)
    first = torch.where(reached, place, V).amin(-1)
    last = torch.where(kept > 0, place, 0).amax(-1)
    return torch.where(greedy[:, 0], index[:, 0], torch.minimum(first, last)).int()


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------

def work(case):
    if case["op"] == "plan":
        cached, new = _lengths(case)
        taken = sum(-(-(c + n) // case["page"]) - -(-c // case["page"]) for c, n in zip(cached, new))
        # lengths in, offsets and lengths out, ids from the list into the table, one table entry read
        # and a position and a slot written for each token
        return {"bytes": 4 * (4 * case["B"] + 3 + 2 * taken + 3 * sum(new) + 2 * case["pad"]), "flops": 0}
    if case["op"] == "rope":
        n = case["T"] * (case["H"] + 2 * case["KV"]) * case["hd"]
        rows = case["T"] * (case["H"] + case["KV"]) * case["hd"]
        return {"bytes": n * (SIZES[case["src"]] + SIZES[case["dst"]]) + case["T"] * 8 + min(case["T"], 4096) * case["rot"] * 4,
                "flops": rows * (3 + 4 * bool(case["norm"]))}
    if case["op"] == "attend":
        cached, new = _lengths(case)
        W = case["window"] or 1 << 30
        keys = sum(c + n - max(0, c + 1 - W) for c, n in zip(cached, new))
        pairs = sum(min(W, c + i + 1) for c, n in zip(cached, new) for i in range(n))
        size, hd = SIZES[case["dtype"]], case["hd"]
        return {"bytes": 2 * size * hd * (keys * case["KV"] + sum(new) * case["H"]) + 4 * (keys // case["page"] + 2 * case["B"]),
                "flops": 4 * pairs * case["H"] * hd}
    return {"bytes": 4 * case["B"] * (case["V"] + 6), "flops": 3 * case["B"] * case["V"]}


# --------------------------------------------------------------------------
# the definition in 64 bits
# --------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] in ("plan", "sample"):
        return None  # whole numbers
    s = prepare(case, seed)
    H, KV, hd = case["H"], case["KV"], case["hd"]
    if case["op"] == "rope":
        T, half = case["T"], case["rot"] // 2
        x = s["qkv"].to(torch.float64).reshape(T, H + 2 * KV, hd)
        if case["norm"]:
            g = torch.cat([s["wq"].double().expand(H, hd), s["wk"].double().expand(KV, hd)])
            scale = (x[:, :H + KV].pow(2).sum(-1, keepdim=True) / hd + 1e-5).sqrt()
            x[:, :H + KV] = x[:, :H + KV] / scale * g
        turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()][:, None, :]
        z = torch.complex(x[:, :H + KV, :half], x[:, :H + KV, half:2 * half]) * turn
        x[:, :H + KV, :half], x[:, :H + KV, half:2 * half] = z.real, z.imag
        blocks, page = s["k_cache"].shape[0], case["page"]
        flat = [torch.zeros(blocks * page, KV, hd, dtype=torch.float64, device=DEV) for _ in range(2)]
        flat[0][s["slots"].long()] = x[:, H:H + KV]
        flat[1][s["slots"].long()] = x[:, H + KV:]
        k, v = (f.view(blocks, page, KV, hd).transpose(1, 2).contiguous() for f in flat)
        return x[:, :H].contiguous(), k, v
    cached, new = _lengths(case)
    out = torch.empty(sum(new), H, hd, dtype=torch.float64, device=DEV)
    W = case["window"] or 1 << 30
    t = 0
    for b, (c, n) in enumerate(zip(cached, new)):
        lo, end = max(0, c + 1 - W), c + n
        j = torch.arange(lo, end, device=DEV)
        page = s["table"][b, j // case["page"]].long()
        pos = torch.arange(c, end, device=DEV)[:, None]
        bias = torch.where((j <= pos) & (j > pos - W), 0.0, -math.inf).double()
        for g in range(KV):
            k, v = (a[page, g, j % case["page"]].double() for a in (s["k_cache"], s["v_cache"]))
            for h in range(g * (H // KV), (g + 1) * (H // KV)):
                p = torch.softmax(s["q_in"][t:t + n, h].double() @ k.T / math.sqrt(hd) + bias, -1)
                out[t:t + n, h] = p @ v
        t += n
    return out
