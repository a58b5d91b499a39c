"""Measured cases of the serving operators: paged append, paged attention, sampling.

A serving step of the engine appends the new rows to a paged cache (`append`), attends over it
(`attention`) and draws the next tokens (`sample`).  All three are integer operators, so the plain
forms below give the same integers: products of more than 32 bits are taken in int64 or in float64
where every partial sum stays below 2^53.
"""
import math
import os
import sys
from decimal import Decimal, getcontext

import numpy as np
import torch

own = False

DMAX = 1536
C1, C2, C3, C4 = 744163075, 257059888, 57045411, 7277686  # 2^-u on [0, 1), Q30
LOG2E_Q24 = 24204406
MASKED = -(1 << 31)


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one new token of one sequence: the smallest call of a decoding step, latency
        dict(name="append_1_4bit", op="append", rows=1, seqs=1, heads=9, kv=3, hd=64, page=16, bits=4, inp=16,
             n_pos=512, mode="decode"),
        # a decoding step of 512 sequences, straight from a device linear's int32 outputs
        dict(name="append_512_4bit", op="append", rows=512, seqs=512, heads=9, kv=3, hd=64, page=32, bits=4, inp=32,
             n_pos=512, mode="decode"),
        # a chunk of prompts (65536 rows, the engine's chunk), kept at 16 bits
        dict(name="append_65536_16bit", op="append", rows=65536, seqs=150, heads=9, kv=3, hd=64, page=16, bits=16,
             inp=32, n_pos=512, mode="prompt"),
        # a ragged prompt batch of a wider model, compressed on the way
        dict(name="append_20011_hd128_4bit", op="append", rows=20011, seqs=7, heads=32, kv=8, hd=128, page=64, bits=4,
             inp=16, n_pos=8192, mode="prompt"),
        # one short conversation: latency of a single call
        dict(name="attention_1x200_16bit", op="attention", seqs=1, per=1, length=200, spread=0.0, heads=9, kv=3, hd=64,
             page=16, bits=16, pb=16, bits_c=16),
        # one sequence with a long cache: the long axis has to be split
        dict(name="attention_1x65521_4bit", op="attention", seqs=1, per=1, length=65521, spread=0.0, heads=9, kv=3,
             hd=64, page=64, bits=4, pb=19, bits_c=16),
        # a serving batch of ragged sequences at the model's table length
        dict(name="attention_512x512_4bit", op="attention", seqs=512, per=1, length=512, spread=1.0, heads=9, kv=3,
             hd=64, page=16, bits=4, pb=16, bits_c=16),
        # the benchmark's decoding batch: 4096 sequences of up to 128 tokens
        dict(name="attention_4096x128_16bit", op="attention", seqs=4096, per=1, length=128, spread=0.3, heads=9, kv=3,
             hd=64, page=32, bits=16, pb=16, bits_c=32),
        # wide heads and long caches, four query rows of each sequence (drafts being verified)
        dict(name="attention_32x4x6000_hd128_4bit", op="attention", seqs=32, per=4, length=6000, spread=0.5, heads=32,
             kv=8, hd=128, page=64, bits=4, pb=18, bits_c=16),
        # one row of the model's vocabulary: latency
        dict(name="sample_1x49152", op="sample", rows=1, vocab=49152, pad=0, mode="k_p"),
        # the benchmark's decoding batch, nucleus sampling
        dict(name="sample_4096x49152", op="sample", rows=4096, vocab=49152, pad=0, mode="p"),
        # an odd, larger vocabulary in padded rows, every row with parameters of its own
        dict(name="sample_100x128003", op="sample", rows=100, vocab=128003, pad=5, mode="mixed"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("append", "attention", "sample"))
    heads, kv, hd = rng.choice(((9, 3, 64), (9, 3, 64), (8, 8, 64), (16, 2, 64), (15, 5, 64), (32, 8, 128), (14, 2, 128)))
    page, bits = rng.choice((16, 32, 64, 128)), rng.choice((4, 4, 16))
    if op == "append":
        mode = rng.choice(("decode", "prompt"))
        rows = _log(rng, 1, 4096 if mode == "decode" else 65536 * 9 // heads)
        return dict(op=op, rows=rows, seqs=rows if mode == "decode" else min(rows, rng.randint(1, 64)), heads=heads, kv=kv,
                    hd=hd, page=page, bits=bits, inp=rng.choice((16, 32)), n_pos=rng.choice((512, 2048, 8192)), mode=mode)
    if op == "attention":
        length = _log(rng, 1, 65536)
        row = kv * 2 * (hd * 2 if bits == 16 else hd // 2 + hd // 16)
        per = rng.choice((1, 1, 1, 2, 4))
        most = min(4096 // per, 150_000_000 // (length * row * per), 2_300_000_000 // (length * heads * per * hd))
        seqs = _log(rng, 1, most) if most > 1 else 1
        return dict(op=op, seqs=seqs, per=per if most >= 1 else 1, length=length, spread=rng.choice((0.0, 0.5, 1.0)),
                    heads=heads, kv=kv, hd=hd, page=page, bits=bits, pb=rng.choice((16, 17, 18, 19)),
                    bits_c=rng.choice((16, 32)))
    vocab = _log(rng, 1000, 200_000)
    return dict(op=op, rows=_log(rng, 1, min(4096, 150_000_000 // vocab)), vocab=vocab, pad=rng.choice((0, 0, 1, 13)),
                mode=rng.choice(("t", "k", "p", "k_p", "min_p", "mixed")))


def _rowbytes(c):
    """Bytes of one cached row of one kv head."""
    return c["hd"] * 2 if c["bits"] == 16 else c["hd"] // 2 + c["hd"] // 16


def _lengths(c):
    """Cached tokens of each sequence: `spread` is the share by which the shortest falls behind."""
    r = np.random.RandomState(c["length"] * 31 + c["seqs"])
    n = np.round(c["length"] * (1.0 - c["spread"] * r.rand(c["seqs"]))).astype(np.int64)
    n[0] = c["length"]
    return np.maximum(n, 1)


def work(case):
    c = case
    if c["op"] == "append":
        q, k = c["heads"] * c["hd"], c["kv"] * c["hd"]
        rope = min(c["rows"], c["n_pos"]) * c["hd"] * 4
        by = c["rows"] * ((q + 2 * k) * c["inp"] // 8 + 2 * q + 2 * c["kv"] * _rowbytes(c) + 2 * k * 4 + 8) + rope
        return {"bytes": by, "flops": c["rows"] * (q + k) * 3}
    if c["op"] == "attention":
        n = _lengths(c)
        tok = int(n.sum())
        seen = int(sum(max(int(x) - (c["per"] - 1 - i), 0) for x in n for i in range(c["per"])))
        rows = c["seqs"] * c["per"]
        by = tok * c["kv"] * 2 * _rowbytes(c) + rows * c["heads"] * c["hd"] * 6 + 4 * int((-(-n // c["page"])).sum())
        return {"bytes": by, "flops": 4 * seen * c["heads"] * c["hd"]}
    return {"bytes": c["rows"] * (c["vocab"] * 4 + 36), "flops": c["rows"] * c["vocab"] * 12}


# ----------------------------------------------------------------------------------------- inputs
def _exp_table():
    """E[d] = floor(2^30 exp(-d / 128) + 1/2)."""
    getcontext().prec = 40
    return [int(((Decimal(-d) / 128).exp() * (1 << 30) + Decimal("0.5")).__floor__()) for d in range(DMAX + 1)]


def _rope(n_pos, hd):
    """Q30 cosines and sines [n_pos][hd / 2] of angles p 100000^(-2 j / hd)."""
    ang = np.arange(n_pos, dtype=np.float64)[:, None] * 100000.0 ** (-2.0 * np.arange(hd // 2) / hd)[None, :]
    return (np.floor(np.cos(ang) * 2.0 ** 30 + 0.5).astype(np.int64), np.floor(np.sin(ang) * 2.0 ** 30 + 0.5).astype(np.int64))


def _normal(g, shape, std, dtype):
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).round_()
    return x.clamp_(-32768, 32767).to(dtype)


def _gains(g, hd, n):
    """A few channels of keys are several times larger than the rest, as in trained models."""
    x = torch.ones(n, hd, device="cuda")
    for i in range(n):
        x[i, torch.randperm(hd, generator=g, device="cuda")[: hd // 16]] = 4.0
    return x


def _pages_of(c, blocks):
    """Pool views (values, scales) of a uint8 pool: values [page][kv][slot][bytes], scales [page][kv][slot][group][4]."""
    n = c["page"] * (c["hd"] * 2 if c["bits"] == 16 else c["hd"] // 2)
    if c["bits"] == 16:
        return blocks.view(torch.int16).unflatten(2, (c["page"], c["hd"])), None
    return (blocks[:, :, :n].unflatten(2, (c["page"], c["hd"] // 2)),
            blocks[:, :, n:].unflatten(2, (c["page"], c["hd"] // 64, 4)))


def _quantise(x):
    """int64 [..., hd] -> (nibble bytes [..., hd / 2], scale bytes [..., hd / 64, 4], the values they stand for)."""
    g = x.unflatten(-1, (-1, 64))
    z, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    m = ((hi - z + 14) // 15).clamp_(min=1)
    n = (2 * (g - z) + m) // (2 * m)
    b = (n[..., :32] | (n[..., 32:] << 4)).flatten(-2).to(torch.uint8)
    sc = torch.cat([m & 255, m >> 8, z & 255, (z >> 8) & 255], -1).to(torch.uint8)
    return b, sc, (z + m * n).flatten(-2)


def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(c)
    if c["op"] == "sample":
        n, v = c["rows"], c["vocab"]
        lg = torch.empty(n, v + c["pad"], device="cuda", dtype=torch.int32)
        for r in range(0, n, 256):
            x = torch.randn(min(256, n - r), v + c["pad"], generator=g, device="cuda").mul_(2.6)
            up = torch.randint(0, v, (x.shape[0], 20), generator=g, device="cuda")
            x.scatter_add_(1, up, torch.rand(up.shape, generator=g, device="cuda").mul_(8.0))
            ban = torch.rand(x.shape, generator=g, device="cuda") < 0.001
            lg[r:r + 256] = torch.where(ban, MASKED, (x * 65536).round_().to(torch.int32))
        s["logits"] = lg
        i32 = dict(device="cuda", dtype=torch.int32)
        t = 0.5 + 0.8 * torch.rand(n, generator=g, device="cuda")
        s["inv_temp"] = (65536.0 / t).round_().to(torch.int32)
        on = torch.randint(0, 2, (3, n), generator=g, **i32) if c["mode"] == "mixed" else None
        k = torch.randint(1, 200, (n,), generator=g, **i32) if on is not None else torch.full((n,), 50, **i32)
        s["top_k"] = k * on[0] if on is not None else (k if c["mode"] in ("k", "k_p") else None)
        p = torch.full((n,), int(0.95 * 65536), **i32)
        if on is not None:
            p = torch.where(on[1] == 1, torch.randint(6554, 65500, (n,), generator=g, **i32), 65536).to(torch.int32)
        s["top_p"] = p if c["mode"] in ("p", "k_p", "mixed") else None
        mp = torch.full((n,), int(0.05 * 65536), **i32)
        s["min_p"] = mp * on[2] if on is not None else (mp if c["mode"] == "min_p" else None)
        s["u"] = torch.randint(-(1 << 31), 1 << 31, (n,), generator=g, **i32)
        s["token"] = torch.zeros(n, device="cuda", dtype=torch.int64)
        s["kept"], s["prob"] = torch.zeros(n, **i32), torch.zeros(n, **i32)
        return s
    hd, kv, heads, page = c["hd"], c["kv"], c["heads"], c["page"]
    if c["op"] == "append":
        n, dt = c["rows"], torch.int16 if c["inp"] == 16 else torch.int32
        # q | k | v of a row lie side by side, as one projection leaves them
        qkv = _normal(g, (n, (heads + 2 * kv) * hd), 1500.0, dt)
        s["q"], s["k"], s["v"] = qkv[:, :heads * hd], qkv[:, heads * hd:(heads + kv) * hd], qkv[:, (heads + kv) * hd:]
        r = np.random.RandomState(seed % (1 << 31))
        if c["mode"] == "decode":
            pos = r.randint(0, c["n_pos"], n)
            seq = np.arange(n)
        else:
            per = np.full(c["seqs"], n // c["seqs"])
            per[: n % c["seqs"]] += 1
            seq = np.repeat(np.arange(c["seqs"]), per)
            start = r.randint(0, max(1, c["n_pos"] - int(per.max()) + 1), c["seqs"])
            pos = np.arange(n) - np.repeat(np.cumsum(per) - per, per)
            pos = (pos + np.repeat(start, per)) % c["n_pos"] if per.max() <= c["n_pos"] else pos
        s["rope"] = _rope(max(c["n_pos"], int(pos.max()) + 1), hd)
        # pages as an allocator hands them out; the pool has room for every page that the rows can touch
        cols = int(pos.max()) // page + 1
        key = seq * cols + pos // page
        used = np.unique(key)
        table = np.full(c["seqs"] * cols, -1, np.int64)
        n_pages = n if c["mode"] == "decode" else int((-(-per // page) + 1).sum())
        table[used] = r.permutation(n_pages)[:len(used)]
        s["table"] = torch.from_numpy(table.reshape(c["seqs"], cols).astype(np.int32)).cuda()
        s["seq"], s["pos"] = (torch.from_numpy(x.astype(np.int32)).cuda() for x in (seq, pos))
        s["q_out"] = torch.zeros(n, heads * hd, device="cuda", dtype=torch.int16)
        s["kv_out"] = torch.zeros(n, 2, kv, hd, device="cuda", dtype=torch.int32)
        for p in ("k_pool", "v_pool"):
            s[p] = torch.zeros(n_pages, kv, page * _rowbytes(c), device="cuda", dtype=torch.uint8)
        return s
    lens = _lengths(c)
    cols = -(-int(lens.max()) // page)
    need = -(-lens // page)
    n_pages = int(need.sum())
    perm = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((c["seqs"], cols), -1, device="cuda", dtype=torch.int32)
    mask = torch.arange(cols, device="cuda")[None, :] < torch.from_numpy(need).cuda()[:, None]
    table[mask] = perm
    s["table"] = table
    gains = _gains(g, hd, kv)
    for p, gain in (("k_pool", gains), ("v_pool", torch.ones_like(gains))):
        pool = torch.empty(n_pages, kv, page * _rowbytes(c), device="cuda", dtype=torch.uint8)
        val, sc = _pages_of(c, pool)
        step = max(1, (1 << 25) // (kv * page * hd))
        for i in range(0, n_pages, step):
            m = min(step, n_pages - i)
            x = (torch.randn(m, kv, page, hd, generator=g, device="cuda") * gain[None, :, None, :] * 1500.0).round_()
            x = x.clamp_(-32768, 32767)
            if c["bits"] == 16:
                val[i:i + m] = x.to(torch.int16)
            else:
                b, w, _ = _quantise(x.to(torch.int32))
                val[i:i + m], sc[i:i + m] = b, w
        s[p] = pool
    rows = c["seqs"] * c["per"]
    s["q"] = _normal(g, (rows, heads * hd), 1500.0, torch.int16)
    s["seq"] = torch.arange(c["seqs"], device="cuda", dtype=torch.int32).repeat_interleave(c["per"])
    # row i of a sequence sees all but the rows after it
    back = torch.arange(c["per"] - 1, -1, -1, device="cuda", dtype=torch.int32).repeat(c["seqs"])
    s["len"] = (torch.from_numpy(lens.astype(np.int32)).cuda().repeat_interleave(c["per"]) - back).clamp_(min=0)
    s["max_len"] = int(lens.max())
    s["shift_s"], s["shift_c"] = 17, c["pb"]
    s["out"] = torch.zeros(rows, heads * hd, device="cuda", dtype=torch.int32)
    return s


def _library():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "exact-integer-inference_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import _eii
    return _eii


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        eii = _library()
        if case["op"] == "sample":
            s["handle"] = eii.Sampler(torch.cuda.current_device())
        else:
            rope = s["rope"] if case["op"] == "append" else _rope(512, case["hd"])
            s["handle"] = eii.Paged(case["heads"], case["kv"], case["hd"], case["page"], case["bits"], rope=rope,
                                    device=torch.cuda.current_device())
            s["pages"] = eii.Pages(s["k_pool"].data_ptr(), s["v_pool"].data_ptr(), s["k_pool"].shape[0],
                                   s["table"].data_ptr(), s["table"].shape[1], s["table"].shape[0])
    elif case["op"] == "append":
        s["cos"], s["sin"] = (torch.from_numpy(x).cuda() for x in s["rope"])
    elif case["op"] == "attention":
        s["exp"] = torch.tensor(_exp_table(), device="cuda")
    return s


# -------------------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return {"append": _own_append, "attention": _own_attention, "sample": _own_sample}[state["op"]](state)
    return {"append": _append, "attention": _attention, "sample": _sample}[state["op"]](state)


def _own_append(s):
    s["handle"].append(s["pages"], s["k"].data_ptr(), s["v"].data_ptr(), s["rows"], s["pos"].data_ptr(), 30,
                       seq_ptr=s["seq"].data_ptr(), q_ptr=s["q"].data_ptr(), q_out_ptr=s["q_out"].data_ptr(), shift_q=30,
                       in_bits=s["inp"], ldq=s["q"].stride(0), ldk=s["k"].stride(0), ldv=s["v"].stride(0),
                       kv_out_ptr=s["kv_out"].data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    return [s["q_out"], s["kv_out"], s["k_pool"], s["v_pool"]]


def _own_attention(s):
    s["handle"].attention(s["pages"], s["q"].data_ptr(), s["q"].shape[0], s["len"].data_ptr(), s["max_len"], s["shift_s"],
                          s["shift_c"], s["bits_c"], s["out"].data_ptr(), seq_ptr=s["seq"].data_ptr(), prob_bits=s["pb"],
                          stream=torch.cuda.current_stream().cuda_stream)
    return s["out"]


def _own_sample(s):
    p = {k + "_ptr": s[k].data_ptr() for k in ("inv_temp", "top_k", "top_p", "min_p") if s[k] is not None}
    s["handle"].sample(s["logits"].data_ptr(), s["rows"], s["vocab"], s["u"].data_ptr(), s["token"].data_ptr(),
                       ld=s["logits"].stride(0), kept_ptr=s["kept"].data_ptr(), prob_ptr=s["prob"].data_ptr(),
                       stream=torch.cuda.current_stream().cuda_stream, **p)
    return [s["token"], s["kept"], s["prob"]]


def _rs(x, n):
    return (x + (1 << (n - 1))) >> n


def _rotate(x, c, sn, shift):
    """int64 [n][heads][hd], Q30 tables [n][hd / 2]."""
    h = x.shape[-1] // 2
    a, b, c, sn = x[..., :h], x[..., h:], c[:, None, :], sn[:, None, :]
    return _rs(torch.cat([a * c - b * sn, b * c + a * sn], -1), shift).clamp_(-32768, 32767)


def _append(s):
    hd, page = s["hd"], s["page"]
    pos = s["pos"].long()
    c, sn = s["cos"][pos], s["sin"][pos]
    s["q_out"].copy_(_rotate(s["q"].long().unflatten(1, (-1, hd)), c, sn, 30).flatten(1))
    k = _rotate(s["k"].long().unflatten(1, (-1, hd)), c, sn, 30)
    v = s["v"].long().unflatten(1, (-1, hd))
    pid, slot = s["table"][s["seq"].long(), pos // page].long(), pos % page
    for i, (x, pool) in enumerate(((k, s["k_pool"]), (v, s["v_pool"]))):
        val, sc = _pages_of(s, pool)
        if s["bits"] == 16:
            val[pid, :, slot] = x.to(torch.int16)
        else:
            b, w, x = _quantise(x)
            val[pid, :, slot], sc[pid, :, slot] = b, w
        s["kv_out"][:, i] = x
    return [s["q_out"], s["kv_out"], s["k_pool"], s["v_pool"]]


def _gather(s, pool, pid):
    """Rows of pages pid [b][cols] as float64 [b][kv][cols * page][hd]."""
    val, sc = _pages_of(s, pool)
    x = val[pid].to(torch.int32)
    if s["bits"] == 4:
        w = sc[pid].to(torch.int32)
        m, z = w[..., 0] | (w[..., 1] << 8), w[..., 2] | (w[..., 3] << 8)
        z = z - ((z >> 15) << 16)
        x = x.unflatten(-1, (-1, 32))
        x = torch.cat([x & 15, x >> 4], -1) * m[..., None] + z[..., None]
        x = x.flatten(-2)
    return x.transpose(1, 2).flatten(2, 3).double()


def _attention(s):
    heads, kv, hd, page, pb = s["heads"], s["kv"], s["hd"], s["page"], s["pb"]
    rows, g = s["q"].shape[0], heads // kv
    cols = s["table"].shape[1]
    step = max(1, (1 << 26) // (cols * page * kv * hd))
    ctx = torch.empty_like(s["out"])
    at = torch.arange(cols * page, device="cuda")
    for r in range(0, rows, step):
        pid = s["table"][s["seq"][r:r + step].long()].clamp(min=0).long()
        q = s["q"][r:r + step].double().unflatten(1, (kv, g, hd))
        acc = (q @ _gather(s, s["k_pool"], pid).transpose(2, 3)).long()
        sc = _rs(acc, s["shift_s"]).clamp_(-32768, 32767)
        seen = (at[None, :] < s["len"][r:r + step, None])[:, None, None, :]
        d = sc.masked_fill(~seen, -(1 << 20)).amax(-1, keepdim=True) - sc
        e = torch.where(seen & (d <= DMAX), s["exp"][d.clamp(0, DMAX)], 0)
        z = e.sum(-1, keepdim=True)
        p = ((e << pb) + (z >> 1)) // z.clamp(min=1)
        o = (p.double() @ _gather(s, s["v_pool"], pid)).long()
        lim = 1 << (s["bits_c"] - 1)
        ctx[r:r + step] = _rs(o, s["shift_c"]).clamp_(-lim, lim - 1).flatten(1).to(torch.int32)
    return ctx


def _weights(lg, beta):
    """Integer weights 2^30 exp(-(max - l) / T) of int64 logits [n][V]; masked logits have none."""
    dist = (lg.amax(1, keepdim=True) - lg)
    x = dist * ((beta * LOG2E_Q24 + (1 << 15)) >> 16)[:, None]
    n, f = x >> 40, ((x >> 16) & 0xFFFFFF) << 7
    y = C3 - ((C4 * f) >> 31)
    y = C2 - ((y * f) >> 31)
    y = C1 - ((y * f) >> 31)
    y = (1 << 30) - ((y * f) >> 31)
    w = torch.where(n <= 30, (y + ((1 << n.clamp(max=31)) >> 1)) >> n.clamp(max=31), 0)
    return w.masked_fill(lg == MASKED, 0)


def _sample(s):
    n, v = s["rows"], s["vocab"]
    tok, num, prob = (torch.empty_like(s[k]) for k in ("token", "kept", "prob"))
    at = torch.arange(v, device="cuda")
    step = max(1, (1 << 26) // v)
    for r in range(0, n, step):
        sl = slice(r, r + step)
        w = _weights(s["logits"][sl, :v].long(), s["inv_temp"][sl].long())
        srt, idx = torch.sort(w, dim=1, descending=True, stable=True)
        keep = srt > 0
        if s["top_k"] is not None:
            k = s["top_k"][sl].long()[:, None]
            keep &= (k <= 0) | (at[None, :] < k)
        if s["min_p"] is not None:
            keep &= srt >= (s["min_p"][sl].long() << 14)[:, None]
        cum = torch.where(keep, srt, 0).cumsum(1)
        if s["top_p"] is not None:
            p, mass = s["top_p"][sl].long()[:, None], cum[:, -1:]
            goal = (p * (mass >> 16) + ((p * (mass & 0xFFFF) + 0xFFFF) >> 16)).clamp_(min=1)
            keep &= (cum - srt) < goal
        kept = torch.zeros_like(w).scatter_(1, idx, torch.where(keep, srt, 0)).cumsum(1)
        mass, u = kept[:, -1], s["u"][sl].long() & 0xFFFFFFFF
        goal = (u * (mass >> 24) + ((u * (mass & 0xFFFFFF)) >> 24)) >> 8
        t = (kept <= goal[:, None]).sum(1)
        won = w.gather(1, t.clamp(max=v - 1)[:, None])[:, 0]
        tok[sl] = torch.where(mass > 0, t, -1)
        num[sl] = keep.sum(1).to(torch.int32)
        prob[sl] = (((won << 30) + (mass >> 1)) // mass.clamp(min=1)).to(torch.int32)
    return [tok, num, prob]


# ------------------------------------------------------------------------- definitions in 64 bits
def exact(case, seed):
    """The operators' integers by their definition, row by row in numpy int64; None where that takes long."""
    c = case
    if c["op"] == "append" and c["rows"] * (c["heads"] + 2 * c["kv"]) * c["hd"] > 1 << 25:
        return None
    if c["op"] == "attention" and c["length"] * c["seqs"] * c["per"] * c["heads"] * c["hd"] > 1 << 29:
        return None
    if c["op"] == "sample" and c["rows"] * c["vocab"] > 1 << 25:
        return None
    s = {k: v.cpu().numpy() if isinstance(v, torch.Tensor) else v for k, v in _inputs(c, seed).items()}
    return {"append": _exact_append, "attention": _exact_attention, "sample": _exact_sample}[c["op"]](s)


def _exact_rs(x, n):
    return np.floor_divide(x + (1 << (n - 1)), 1 << n)


def _exact_append(s):
    hd, kv, page, n = s["hd"], s["kv"], s["page"], s["rows"]
    h = hd // 2
    cos, sin = s["rope"]
    vb = page * (hd * 2 if s["bits"] == 16 else hd // 2)

    def turn(x, p):
        o = np.empty_like(x)
        o[:, :h] = x[:, :h] * cos[p] - x[:, h:] * sin[p]
        o[:, h:] = x[:, h:] * cos[p] + x[:, :h] * sin[p]
        return np.clip(_exact_rs(o, 30), -32768, 32767)

    for r in range(n):
        p = int(s["pos"][r])
        s["q_out"][r] = turn(s["q"][r].astype(np.int64).reshape(-1, hd), p).reshape(-1)
        k = turn(s["k"][r].astype(np.int64).reshape(-1, hd), p)
        v = s["v"][r].astype(np.int64).reshape(-1, hd)
        pid, slot = int(s["table"][s["seq"][r], p // page]), p % page
        for i, (x, pool) in enumerate(((k, s["k_pool"]), (v, s["v_pool"]))):
            if s["bits"] == 16:
                for j in range(kv):
                    pool[pid, j, slot * hd * 2:(slot + 1) * hd * 2] = x[j].astype("<i2").view(np.uint8)
                s["kv_out"][r, i] = x
                continue
            for j in range(kv):
                for a in range(hd // 64):
                    y = x[j, 64 * a:64 * a + 64]
                    z = int(y.min())
                    m = max(1, -((z - int(y.max())) // 15))
                    t = (2 * (y - z) + m) // (2 * m)
                    at = slot * (hd // 2) + 32 * a
                    pool[pid, j, at:at + 32] = t[:32] + 16 * t[32:]
                    at = vb + (slot * (hd // 64) + a) * 4
                    pool[pid, j, at:at + 4] = [m % 256, m // 256, z % 256, (z // 256) % 256]
                    s["kv_out"][r, i, j, 64 * a:64 * a + 64] = z + m * t
    return [s["q_out"], s["kv_out"], s["k_pool"], s["v_pool"]]


def _exact_rows(s, pool, pids, j, n):
    hd, page = s["hd"], s["page"]
    x = pool[pids, j]
    if s["bits"] == 16:
        return np.ascontiguousarray(x).view("<i2").reshape(-1, hd)[:n].astype(np.int64)
    nib = x[:, :page * hd // 2].reshape(-1, hd // 64, 32).astype(np.int64)[:n]
    sc = np.ascontiguousarray(x[:, page * hd // 2:]).reshape(-1, hd // 64, 4)[:n]
    m = sc[..., 0].astype(np.int64) + 256 * sc[..., 1].astype(np.int64)
    z = np.ascontiguousarray(sc[..., 2:]).view("<i2")[..., 0].astype(np.int64)
    return (np.concatenate([nib % 16, nib // 16], -1) * m[..., None] + z[..., None]).reshape(n, hd)


def _exact_attention(s):
    hd, kv, heads, pb = s["hd"], s["kv"], s["heads"], s["pb"]
    e_tab = np.array(_exp_table(), np.int64)
    lim = 1 << (s["bits_c"] - 1)
    for r in range(s["q"].shape[0]):
        n = int(s["len"][r])
        pids = s["table"][s["seq"][r], :-(-n // s["page"])]
        for j in range(kv):
            k, v = (_exact_rows(s, s[p], pids, j, n) for p in ("k_pool", "v_pool"))
            for h in range(j * (heads // kv), (j + 1) * (heads // kv)):
                q = s["q"][r, h * hd:(h + 1) * hd].astype(np.int64)
                sc = np.clip(_exact_rs(k @ q, s["shift_s"]), -32768, 32767)
                d = sc.max(initial=-32768) - sc
                e = np.where(d <= DMAX, e_tab[np.minimum(d, DMAX)], 0)
                z = max(1, int(e.sum()))
                p = (e * (1 << pb) + z // 2) // z
                s["out"][r, h * hd:(h + 1) * hd] = np.clip(_exact_rs(p @ v, s["shift_c"]), -lim, lim - 1)
    return s["out"]


def _exact_sample(s):
    out, num, prob = s["token"], s["kept"], s["prob"]
    for r in range(s["rows"]):
        lg = s["logits"][r, :s["vocab"]].astype(np.int64)
        b2 = (int(s["inv_temp"][r]) * LOG2E_Q24 + (1 << 15)) // (1 << 16)
        x = (lg.max() - lg) * b2
        octave, f = x // (1 << 40), (x // (1 << 16)) % (1 << 24) * 128
        y = np.full_like(f, C4)
        for c in (C3, C2, C1, 1 << 30):
            y = c - y * f // (1 << 31)
        half = np.where(octave > 0, 1 << np.maximum(np.minimum(octave, 31) - 1, 0), 0)
        w = np.where((octave <= 30) & (lg != MASKED), (y + half) // (1 << np.minimum(octave, 31)), 0)
        order = np.lexsort((np.arange(w.size), -w))
        order = order[w[order] > 0]
        if s["top_k"] is not None and s["top_k"][r] > 0:
            order = order[: int(s["top_k"][r])]
        if s["min_p"] is not None:
            order = order[w[order] >= int(s["min_p"][r]) * (1 << 14)]
        if s["top_p"] is not None and order.size:
            goal = max(1, -(-int(s["top_p"][r]) * int(w[order].sum()) // 65536))
            order = order[: int(np.searchsorted(np.cumsum(w[order]), goal)) + 1]
        mass = int(w[order].sum())
        num[r] = order.size
        if not mass:
            out[r], prob[r] = -1, 0
            continue
        goal = ((int(s["u"][r]) & 0xFFFFFFFF) * mass) >> 32
        ids = np.sort(order)
        out[r] = ids[int(np.searchsorted(np.cumsum(w[ids]), goal, side="right"))]
        prob[r] = (int(w[out[r]]) * (1 << 30) + mass // 2) // mass
    return [out, num, prob]
