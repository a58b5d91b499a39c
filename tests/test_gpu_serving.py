"""The serving operators on the GPU against their numpy oracle: paged append, paged attention,
sampling.  Every result is an integer and has to be equal."""
import numpy as np
import pytest

from oracle import serving as osv

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def st(torch):
    return torch.cuda.current_stream().cuda_stream


def random_rope(rng, n_pos, hd):
    a = rng.uniform(0, 2 * np.pi, (n_pos, hd // 2))
    return np.round(np.cos(a) * 2 ** 30).astype(np.int64), np.round(np.sin(a) * 2 ** 30).astype(np.int64)


class Cache:
    """A cache on both sides: device pools and the oracle's, with the same page table."""

    def __init__(self, torch, rng, heads, kv, hd, page, bits, lens, rope=None, n_pos=512, spare=3):
        import _eii
        self.t, self.heads, self.kv, self.hd, self.page, self.bits = torch, heads, kv, hd, page, bits
        self.rope = rope if rope is not None else random_rope(rng, n_pos, hd)
        self.p = _eii.Paged(heads, kv, hd, page, bits, rope=self.rope)
        need = [-(-int(n) // page) for n in lens]
        cols = max(max(need), 1) + 1
        self.n_pages = sum(need) + spare
        ids = rng.permutation(self.n_pages)
        # entries that no call reaches hold indices that must not be followed
        self.table = np.full((len(lens), cols), 1 << 30, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = ids[at:at + n]
            at += n
        size = self.p.pool_bytes(self.n_pages)
        self.host = [rng.integers(0, 256, size, dtype=np.uint8) for _ in range(2)]
        self.dev = [torch.from_numpy(x.copy()).cuda() for x in self.host]
        self.k, self.v = (osv.Pool(x, kv, hd, page, bits) for x in self.host)
        self.dtable = torch.from_numpy(self.table).cuda()
        self.pages = _eii.Pages(self.dev[0].data_ptr(), self.dev[1].data_ptr(), self.n_pages, self.dtable.data_ptr(), cols,
                                len(lens))

    def fill(self, rng, lens, std=1500.0):
        """Random rows at positions 0 .. lens[s] - 1 of both sides."""
        for s, n in enumerate(lens):
            for t in range(int(n)):
                for h in range(self.kv):
                    for pool in (self.k, self.v):
                        x = rng.normal(0, std, self.hd).round().clip(-32768, 32767).astype(np.int64)
                        pool.put(int(self.table[s, t // self.page]), h, t % self.page, x)
        self.upload()

    def upload(self):
        for d, h in zip(self.dev, self.host):
            d.copy_(self.t.from_numpy(h))

    def check_pools(self):
        for d, h in zip(self.dev, self.host):
            assert np.array_equal(d.cpu().numpy(), h)


# ----------------------------------------------------------------------------------------- append
APPEND = [(9, 3, 64, 16, 16, 16), (9, 3, 64, 16, 4, 32), (9, 3, 64, 128, 4, 16), (4, 4, 128, 32, 4, 32),
          (16, 2, 128, 16, 16, 16), (1, 1, 64, 1024, 4, 16), (6, 1, 128, 64, 16, 32)]


@pytest.mark.parametrize("heads,kv,hd,page,bits,inp", APPEND)
@pytest.mark.parametrize("n", [1, 2, 77])
@pytest.mark.parametrize("shape", ["dense", "fused", "offset"])
def test_append(torch, heads, kv, hd, page, bits, inp, n, shape):
    """Ragged rows with padding among them; dense rows, q | k | v side by side, and odd strides."""
    rng = np.random.default_rng(n + hd + bits)
    lens = [300, 1, 511, 64]
    c = Cache(torch, rng, heads, kv, hd, page, bits, lens)
    rows = [(s, t) for s, m in enumerate(lens) for t in range(m)]
    rows = [rows[i] for i in rng.permutation(len(rows))[:n]]
    seq, pos = (np.array(x, np.int32) for x in zip(*rows))
    if n > 2:
        seq[3], pos[5] = -1, -7
    dt = np.int16 if inp == 16 else np.int32
    widths = [heads * hd, kv * hd, kv * hd]
    data = rng.normal(0, 6000, (n, sum(widths))).round().clip(-32768, 32767)
    data[0, :7] = [-32768, 32767, 0, 1, -1, 32767, -32768]
    data[-1] = 5  # a row without spread: m = 1
    data = data.astype(dt)
    pad, off = {"dense": (0, 0), "fused": (0, 0), "offset": (3, 1)}[shape]
    cuts = np.cumsum([0] + widths)
    parts = [data[:, cuts[i]:cuts[i + 1]] for i in range(3)]
    if shape == "fused":
        full = torch.from_numpy(data).cuda()
        dev = [full[:, cuts[i]:cuts[i + 1]] for i in range(3)]
    else:
        dev = []
        for x in parts:
            buf = torch.full((n * (x.shape[1] + pad) + off + 8,), 17, dtype=torch.from_numpy(x).dtype, device="cuda")
            view = buf[off:off + n * (x.shape[1] + pad)].view(n, -1)[:, :x.shape[1]]
            view.copy_(torch.from_numpy(np.ascontiguousarray(x)))
            dev.append(view)
    q_out = torch.full((n, heads * hd + pad), 99, dtype=torch.int16, device="cuda")
    kv_out = torch.full((n, 2, kv, hd), 98, dtype=torch.int32, device="cuda")
    dseq, dpos = torch.from_numpy(seq).cuda(), torch.from_numpy(pos).cuda()
    c.p.append(c.pages, dev[1].data_ptr(), dev[2].data_ptr(), n, dpos.data_ptr(), 29, seq_ptr=dseq.data_ptr(),
               q_ptr=dev[0].data_ptr(), q_out_ptr=q_out.data_ptr(), shift_q=31, in_bits=inp, ldq=dev[0].stride(0),
               ldk=dev[1].stride(0), ldv=dev[2].stride(0), ldqo=heads * hd + pad, kv_out_ptr=kv_out.data_ptr(),
               stream=st(torch))
    c.p.sync(st(torch))
    wq, wkv = np.full((n, heads, hd), 99, np.int64), np.full((n, 2, kv, hd), 98, np.int64)
    osv.append(parts[0].reshape(n, heads, hd), parts[1].reshape(n, kv, hd), parts[2].reshape(n, kv, hd), seq, pos, c.table,
               c.k, c.v, c.rope, 31, 29, wq, wkv)
    got = q_out.cpu().numpy()
    assert np.array_equal(got[:, :heads * hd], wq.reshape(n, -1)) and (got[:, heads * hd:] == 99).all()
    assert np.array_equal(kv_out.cpu().numpy(), wkv)
    c.check_pools()


def test_append_without_q_in_place_and_default_sequences(torch):
    rng = np.random.default_rng(4)
    c = Cache(torch, rng, 9, 3, 64, 16, 4, [512, 40, 512])
    x = [rng.integers(-32768, 32768, (3, h, 64)) for h in (9, 3, 3)]
    pos = np.array([511, 33, 0], np.int32)
    d = [torch.from_numpy(a.astype(np.int16)).cuda() for a in x]
    dpos = torch.from_numpy(pos).cuda()
    wq, wkv = np.zeros((3, 9, 64), np.int64), np.zeros((3, 2, 3, 64), np.int64)
    osv.append(*x, np.arange(3), pos, c.table, c.k, c.v, c.rope, 30, 30, wq, wkv)
    c.p.append(c.pages, d[1].data_ptr(), d[2].data_ptr(), 3, dpos.data_ptr(), 30, stream=st(torch))
    c.p.sync(st(torch))
    c.check_pools()
    c.p.append(c.pages, d[1].data_ptr(), d[2].data_ptr(), 3, dpos.data_ptr(), 30, q_ptr=d[0].data_ptr(),
               q_out_ptr=d[0].data_ptr(), shift_q=30, stream=st(torch))
    c.p.sync(st(torch))
    c.check_pools()
    assert np.array_equal(d[0].cpu().numpy(), wq)
    c.p.append(c.pages, d[1].data_ptr(), d[2].data_ptr(), 0, dpos.data_ptr(), 30, stream=st(torch))
    c.p.append(c.pages, None, None, 0, None, 30, stream=st(torch))  # (an empty tensor's pointer)
    c.p.attention(c.pages, None, 0, None, 512, 17, 16, 16, None, stream=st(torch))
    c.p.sync(st(torch))
    c.check_pools()


# -------------------------------------------------------------------------------------- attention
def check_attention(torch, c, rng, seq, length, max_len, shift_s=17, pb=16, shift_c=16, bits_c=16, q=None, pad=0):
    import _eii
    n = len(length)
    if q is None:
        q = rng.normal(0, 1500, (n, c.heads, c.hd)).round().clip(-32768, 32767)
    q = q.astype(np.int64)
    width = c.heads * c.hd
    dq = torch.zeros(n * (width + pad) + pad, dtype=torch.int16, device="cuda")
    vq = dq[pad:].view(n, width + pad)[:, :width]
    vq.copy_(torch.from_numpy(q.reshape(n, -1).astype(np.int16)))
    out = torch.full((n, width + pad), 12345, dtype=torch.int32, device="cuda")
    dlen = torch.from_numpy(np.asarray(length, np.int32)).cuda()
    dseq = None if seq is None else torch.from_numpy(np.asarray(seq, np.int32)).cuda()
    c.p.attention(c.pages, vq.data_ptr(), n, dlen.data_ptr(), max_len, shift_s, shift_c, bits_c, out.data_ptr(),
                  seq_ptr=None if seq is None else dseq.data_ptr(), prob_bits=pb, ldq=width + pad, ldc=width + pad,
                  stream=st(torch))
    c.p.sync(st(torch))
    want = np.full((n, c.heads, c.hd), 12345, np.int64)
    osv.attention(q, np.arange(n) if seq is None else seq, length, c.table, c.k, c.v, _eii.table_exp(), shift_s, pb, shift_c,
                  bits_c, want)
    got = out.cpu().numpy()
    bad = np.argwhere(got[:, :width].reshape(want.shape) != want)
    assert bad.size == 0, (len(bad), bad[:4].tolist())
    assert (got[:, width:] == 12345).all()


@pytest.mark.parametrize("heads,kv,hd,page,bits", [(9, 3, 64, 16, 16), (9, 3, 64, 16, 4), (9, 3, 64, 64, 4), (8, 8, 64, 32, 16),
                                                   (8, 1, 128, 32, 4), (8, 1, 64, 16, 16), (4, 2, 128, 16, 16), (7, 1, 64, 128, 4),
                                                   (18, 2, 64, 16, 4), (16, 1, 128, 64, 16), (1, 1, 64, 1024, 4)])
def test_attention_lengths(torch, heads, kv, hd, page, bits):
    """Lengths around every tile and page edge, an empty sequence and padding rows among them."""
    rng = np.random.default_rng(heads * hd + page)
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 200, 257]
    c = Cache(torch, rng, heads, kv, hd, page, bits, lens)
    c.fill(rng, lens)
    check_attention(torch, c, rng, None, lens, 257)
    check_attention(torch, c, rng, [3, -1, 17, 17, 17, 0, 9, -5], [15, 4, 257, 256, 1, -3, 40, 0], 1000, pb=18, shift_c=19,
                    bits_c=32, pad=3)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("hd,n", [(64, 1100), (64, 5003), (128, 2049)])
def test_attention_long(torch, bits, hd, n):
    """One long sequence among short ones (the long axis is split over blocks)."""
    rng = np.random.default_rng(n + bits)
    lens = [n, 3, 700]
    c = Cache(torch, rng, 6, 2, hd, 64, bits, lens)
    c.fill(rng, lens)
    for max_len, pb in ((n, 16), (65536, 19)):
        check_attention(torch, c, rng, None, lens, max_len, pb=pb, shift_c=pb)
    check_attention(torch, c, rng, [0], [n - 1], n, shift_s=20)


@pytest.mark.parametrize("heads,kv,hd", [(9, 3, 64), (8, 2, 64), (14, 2, 128)])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("n", [1, 5, 20, 130, 700])
def test_attention_shapes(torch, heads, kv, hd, bits, n):
    """What a launch is laid out by: rows from one to many, each against length bounds from short to the longest."""
    rng = np.random.default_rng(n + hd + bits)
    lens = [300, 37, 1, 640]
    c = Cache(torch, rng, heads, kv, hd, 32, bits, lens)
    c.fill(rng, lens)
    seq = rng.integers(-1, 4, n)
    length = np.where(rng.random(n) < min(1, 8 / n), np.take(lens, seq), rng.integers(0, 50, n).clip(max=np.take(lens, seq)))
    for max_len in (640, 1200, 5000, 20000, 70000, 131072):
        check_attention(torch, c, rng, seq, length, max_len, shift_c=16)


@pytest.mark.parametrize("bits", [16, 4])
def test_attention_extremes(torch, bits):
    """Saturated scores, one key that takes all the weight, equal keys, keys beyond the table's end,
    the largest values with the smallest shifts."""
    rng = np.random.default_rng(7)
    c = Cache(torch, rng, 9, 3, 64, 16, bits, [150])
    q = np.full((1, 9, 64), -32768)
    q[0, 3:6] = 32767
    q[0, 6:] = rng.integers(-32768, 32768, (3, 64))
    for t in range(150):
        for h in range(3):
            k = np.full(64, [-32768, 32767, 1][t % 3]) if t < 100 else rng.integers(-32768, 32768, 64)
            c.k.put(int(c.table[0, t // 16]), h, t % 16, k.astype(np.int64))
            v = np.full(64, [-32768, 32767][t % 2]) if t < 75 else rng.integers(-32768, 32768, 64)
            c.v.put(int(c.table[0, t // 16]), h, t % 16, v.astype(np.int64))
    c.upload()
    for shift_s in (1, 10, 22, 30, 62):
        for n in (1, 75, 150):
            check_attention(torch, c, rng, [0], [n], 150, shift_s=shift_s, q=q)
            check_attention(torch, c, rng, [0], [n], 150, shift_s=shift_s, q=q, pb=19, shift_c=1, bits_c=32)
            check_attention(torch, c, rng, [0], [n], 150, shift_s=shift_s, q=q, pb=19, shift_c=30, bits_c=2)
            check_attention(torch, c, rng, [0], [n], 150, shift_s=shift_s, q=q, shift_c=-16, bits_c=32)
            check_attention(torch, c, rng, [0], [n], 150, shift_s=shift_s, q=q, shift_c=0, bits_c=32)


def test_attention_tables_in_used_memory(torch):
    """Keys too far from the maximum to weigh anything, and keys behind the last, with handles whose tables lie where
    other tables have been."""
    import _eii
    rng = np.random.default_rng(12)
    one = np.full((4096, 32), 1 << 30, np.int64)
    old = [_eii.Paged(9, 3, 64, 16, 16, rope=(one, one)) for _ in range(4)]
    for p in old:
        p.close()
    kept = []
    for i in range(12):
        lens = [150, 33, 7]
        c = Cache(torch, rng, 9, 3, 64, 16, 16 if i % 2 else 4, lens, n_pos=64 + 96 * i)
        c.fill(rng, lens)
        kept.append(c)
        for n, max_len in ((100, 600), (40, 600), (10, 5000), (1, 70000)):
            seq = rng.integers(0, 3, n)
            check_attention(torch, c, rng, seq, np.take(lens, seq), max_len, shift_s=12)


def test_attention_shared_pages(torch):
    """Two sequences that share their first pages (a common prompt)."""
    rng = np.random.default_rng(8)
    lens = [100, 70, 1]
    c = Cache(torch, rng, 9, 3, 64, 16, 4, lens)
    c.table[1, :4] = c.table[0, :4]
    c.dtable.copy_(torch.from_numpy(c.table))
    c.fill(rng, lens)
    check_attention(torch, c, rng, [0, 1, 1], [100, 70, 64], 128)


def test_attention_beyond_4gb(torch):
    """A pool of more than 2^32 bytes: rows in its last pages."""
    import _eii
    rng = np.random.default_rng(9)
    page, n_pages = 1024, 11000  # 11000 x 3 x 1024 x 128 bytes = 4.3 GB
    c = Cache(torch, rng, 9, 3, 64, page, 16, [40, 1030])
    c.fill(rng, [40, 1030])
    big = [torch.empty(c.p.pool_bytes(n_pages), dtype=torch.uint8, device="cuda") for _ in range(2)]
    shift = n_pages - c.n_pages
    for b, h in zip(big, c.host):
        b[-h.size:].copy_(torch.from_numpy(h))
    table = torch.from_numpy(np.where(c.table < c.n_pages, c.table + shift, c.table).astype(np.int32)).cuda()
    c.pages = _eii.Pages(big[0].data_ptr(), big[1].data_ptr(), n_pages, table.data_ptr(), c.table.shape[1], 2)
    assert big[0].numel() > 1 << 32
    check_attention(torch, c, rng, None, [40, 1030], 1030)
    x = [rng.integers(-32768, 32768, (2, h, 64)) for h in (9, 3, 3)]
    d = [torch.from_numpy(a.astype(np.int16)).cuda() for a in x]
    pos = np.array([39, 1024], np.int32)
    dpos = torch.from_numpy(pos).cuda()
    c.rope = tuple(np.tile(t, (3, 1))[:1100] for t in c.rope)
    p = _eii.Paged(9, 3, 64, page, 16, rope=c.rope)
    p.append(c.pages, d[1].data_ptr(), d[2].data_ptr(), 2, dpos.data_ptr(), 30, stream=st(torch))
    p.sync(st(torch))
    osv.append(None, x[1], x[2], np.arange(2), pos, c.table, c.k, c.v, c.rope, 30, 30, None, np.zeros((2, 2, 3, 64), np.int64))
    for b, h in zip(big, c.host):
        assert np.array_equal(b[-h.size:].cpu().numpy(), h)


def test_cache_refusals(torch):
    """Host refusals leave everything alone; device-side ones are reported once and the handle goes on."""
    import _eii
    rng = np.random.default_rng(10)
    c = Cache(torch, rng, 9, 3, 64, 16, 4, [64, 64])
    c.fill(rng, [64, 64])
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    kv = torch.ones(2, 192, dtype=torch.int32, device="cuda")
    q = torch.ones(2, 576, dtype=torch.int16, device="cuda")
    out = torch.zeros(2, 576, dtype=torch.int32, device="cuda")

    def append(n=2, pos=i32(0, 1), seq=None, k=kv, **kw):
        kw = dict(in_bits=32, seq_ptr=None if seq is None else seq.data_ptr(), stream=st(torch)) | kw
        c.p.append(c.pages, k.data_ptr(), kv.data_ptr(), n, pos.data_ptr(), kw.pop("shift_k", 30), **kw)

    def attend(n=2, length=i32(3, 4), max_len=64, seq=None, **kw):
        kw = dict(seq_ptr=None if seq is None else seq.data_ptr(), stream=st(torch)) | kw
        c.p.attention(c.pages, q.data_ptr(), n, length.data_ptr(), max_len, kw.pop("shift_s", 17), kw.pop("shift_c", 16),
                      kw.pop("bits_c", 16), out.data_ptr(), **kw)
    for bad in (lambda: append(n=3), lambda: append(n=-1), lambda: append(in_bits=8), lambda: append(shift_k=0),
                lambda: append(shift_k=63), lambda: append(ldk=191), lambda: append(q_ptr=q.data_ptr()),
                lambda: append(q_out_ptr=q.data_ptr()), lambda: append(q_ptr=q.data_ptr(), q_out_ptr=q.data_ptr(), shift_q=0),
                lambda: attend(n=3), lambda: attend(max_len=131073), lambda: attend(max_len=-1), lambda: attend(prob_bits=15),
                lambda: attend(prob_bits=20), lambda: attend(shift_s=0), lambda: attend(shift_c=63), lambda: attend(shift_c=-17), lambda: attend(bits_c=33),
                lambda: attend(seq_ptr=q.data_ptr() + 2), lambda: append(seq_ptr=q.data_ptr() + 2),
                lambda: append(kv_out_ptr=out.data_ptr() + 2), lambda: attend(ldq=575), lambda: attend(ldc=575), lambda: c.p.pool_bytes(0)):
        with pytest.raises(_eii.EiiError) as e:
            bad()
        assert e.value.code == _eii.EII_ERR_ARG
    good, c_pages = c.pages, []
    for field, value in (("k_pool", None), ("table", None), ("n_pages", 0), ("ld_table", 0), ("n_seq", 0),
                         ("v_pool", c.dev[1].data_ptr() + 8)):
        c.pages = _eii.Pages.from_buffer_copy(good)
        setattr(c.pages, field, value)
        with pytest.raises(_eii.EiiError):
            attend()
    c.pages = good
    c.p.sync(st(torch))
    wide = kv.clone()
    wide[1, 100] = 32768
    broken = c.table.copy()
    for value in (c.n_pages, -1):
        broken[1, 0] = value
        c.dtable.copy_(torch.from_numpy(broken))
        for call in (append, attend):
            call()
            with pytest.raises(_eii.EiiError, match="page"):
                c.p.sync(st(torch))
    c.dtable.copy_(torch.from_numpy(c.table))
    for call, text in ((lambda: append(seq=i32(0, 2)), "sequence"), (lambda: append(pos=i32(0, 512)), "position"),
                       (lambda: append(pos=i32(0, 5 * 16)), "position"), (lambda: append(k=wide), "int16"),
                       (lambda: attend(seq=i32(0, 2)), "sequence"), (lambda: attend(length=i32(65, 3)), "length"),
                       (lambda: attend(length=i32(5 * 16 + 1, 3), max_len=1000), "length")):
        call()
        with pytest.raises(_eii.EiiError, match=text) as e:
            c.p.sync(st(torch))
        assert e.value.code == _eii.EII_ERR_ARG
        c.p.sync(st(torch))
    c.fill(rng, [64, 64])
    check_attention(torch, c, rng, None, [64, 50], 64)


# --------------------------------------------------------------------------------------- sampling
def check_draw(torch, s, row_data, u, ld_pad=0, offset=0, **params):
    n, v = row_data.shape
    buf = torch.full((n * (v + ld_pad) + offset,), (1 << 31) - 1, dtype=torch.int32, device="cuda")
    view = buf[offset:].view(n, v + ld_pad)[:, :v]
    view.copy_(torch.from_numpy(row_data.astype(np.int32)))
    dev = {k + "_ptr": torch.from_numpy(np.asarray(x, np.int32)).cuda() for k, x in params.items()}
    du = torch.from_numpy(np.asarray(u, np.uint32).view(np.int32)).cuda()
    tok = torch.full((n,), -9, dtype=torch.int64, device="cuda")
    kept, prob = (torch.full((n,), -9, dtype=torch.int32, device="cuda") for _ in range(2))
    s.sample(view.data_ptr(), n, v, du.data_ptr(), tok.data_ptr(), ld=v + ld_pad, kept_ptr=kept.data_ptr(),
             prob_ptr=prob.data_ptr(), stream=st(torch), **{k: x.data_ptr() for k, x in dev.items()})
    s.sync(st(torch))
    got = list(zip(tok.tolist(), kept.tolist(), prob.tolist()))
    want = [osv.draw(row_data[r], u[r], **{k: int(x[r]) for k, x in params.items()}) for r in range(n)]
    assert got == want, [(r, g, w) for r, (g, w) in enumerate(zip(got, want)) if g != w][:5]


@pytest.fixture(scope="module")
def sampler():
    import _eii
    s = _eii.Sampler(0)
    yield s
    s.close()


def words(rng, n):
    u = rng.integers(0, 1 << 32, n, dtype=np.uint64)
    u[0] = 0
    u[-1] = (1 << 32) - 1
    return u


@pytest.mark.parametrize("v,pad,offset", [(1, 0, 0), (2, 0, 1), (31, 2, 0), (1000, 0, 0), (1001, 7, 3), (49152, 0, 0), (50257, 3, 1)])
def test_sampling_parameters(torch, sampler, v, pad, offset):
    """Every parameter on its own and together; vocabularies and row strides of every alignment."""
    rng = np.random.default_rng(v)
    n = 12 if v > 2000 else 40
    lg = (rng.normal(0, 2.6, (n, v)) * 65536).round().astype(np.int64)
    lg[rng.random((n, v)) < 0.05] = osv.MASKED
    if v > 40:
        lg[1, 5:25] = lg[1, 30]                  # ties
        lg[2, :20] += 8 << 16
    u = words(rng, n)
    t = (65536 / rng.uniform(.2, 3, n)).round().astype(np.int64)
    k = rng.integers(1, max(2, min(v, 300)), n)
    p = rng.integers(0, 65537, n)
    m = rng.integers(0, 9000, n)
    for kw in ({}, dict(inv_temp=t), dict(top_k=k), dict(top_p=p), dict(min_p=m), dict(top_k=np.ones(n, int)),
               dict(inv_temp=t, top_k=k, top_p=p), dict(inv_temp=t, top_k=k * (k % 2), top_p=np.where(k % 3, p, 65536), min_p=m)):
        check_draw(torch, sampler, lg, u, pad, offset, **kw)


def test_sampling_edges(torch, sampler):
    """All equal, all masked but one, all masked, the whole int32 range, ties across the cut, limits of
    every parameter."""
    rng = np.random.default_rng(3)
    v, n = 3001, 24
    lg = np.zeros((n, v), np.int64)
    lg[1] = osv.MASKED
    lg[2] = osv.MASKED
    lg[2, 1717] = osv.MASKED + 1
    lg[3] = rng.integers(-(1 << 31) + 1, 1 << 31, v)
    lg[4, ::2] = (1 << 31) - 1
    lg[4, 1::2] = -(1 << 31) + 1
    lg[5, 100:200] = 65536
    lg[6:] = rng.integers(-4, 5, (n - 6, v)) * 20000     # nine levels: ties everywhere
    u = words(rng, n)
    for beta in (1, 65536, 1 << 22):
        b = np.full(n, beta)
        for k in (0, 1, 7, 150, v, v + 5, (1 << 31) - 1):
            for p, m in ((65536, 0), (0, 0), (1, 65536), (40000, 1), (65535, 30000)):
                check_draw(torch, sampler, lg, u, inv_temp=b, top_k=np.full(n, k), top_p=np.full(n, p), min_p=np.full(n, m))


def test_sampling_masses(torch, sampler):
    """Every border of a small row's distribution: words around each cumulative mass."""
    row = np.round(np.log([8, 1, 4, 2, 1, 3, 3]) * 65536).astype(np.int64)
    w = osv.weights(row, 65536)
    cum, mass = np.cumsum(w), int(w.sum())
    edges = [(int(c) << 32) // mass for c in cum]
    u = np.array([min(max(e + d, 0), (1 << 32) - 1) for e in edges for d in (-2, -1, 0, 1, 2)], np.uint64)
    check_draw(torch, sampler, np.tile(row, (len(u), 1)), u)
    for p in range(0, 65537, 4096):
        check_draw(torch, sampler, np.tile(row, (len(u), 1)), u, top_p=np.full(len(u), p))


def test_sampling_many_rows(torch, sampler):
    """More rows than blocks are resident, and a large vocabulary."""
    rng = np.random.default_rng(6)
    lg = (rng.normal(0, 3, (700, 257)) * 65536).round().astype(np.int64)
    check_draw(torch, sampler, lg, words(rng, 700), top_p=np.full(700, 60000), top_k=np.full(700, 40))
    lg = (rng.normal(0, 3, (3, 262144)) * 65536).round().astype(np.int64)
    lg[1] = 77
    check_draw(torch, sampler, lg, words(rng, 3), top_p=np.full(3, 60000))
    check_draw(torch, sampler, lg, words(rng, 3), top_k=np.full(3, 100000))


@pytest.mark.parametrize("n,v,pad", [(90, 20501, 3), (80, 49152, 0), (5, 128003, 1)])
def test_sampling_long_rows(torch, sampler, n, v, pad):
    """Rows long enough for the searches that start from a sample (one block per row, and a cluster): every
    kind of row beside an ordinary one, small and large top-k, cuts within ties, too few logits for top-k,
    distances at the last octave's edge."""
    rng = np.random.default_rng(v)
    lg = (rng.normal(0, 2.6, (n, v)) * 65536).round().astype(np.int64)
    lg[rng.random((n, v)) < 0.01] = osv.MASKED
    kinds = [lambda r: np.zeros(v), lambda r: np.full(v, osv.MASKED), lambda r: np.where(rng.random(v) < 3 / v, r, osv.MASKED),
             lambda r: rng.integers(-4, 5, v) * 20000, lambda r: rng.integers(-(1 << 31) + 1, 1 << 31, v),
             lambda r: np.where(np.arange(v) < 40, 5 << 16, r), lambda r: r - (1 << 31) + (30 << 16),
             lambda r: -(rng.integers(30 << 16, 32 << 16, v) * 0.6931).astype(np.int64) * (np.arange(v) > 0),
             lambda r: np.sort(r), lambda r: np.where(np.arange(v) % 48 == 7, r + (9 << 16), r)]
    for i in range(n):
        if i % 2 == 0:
            lg[i] = np.maximum(kinds[i // 2 % len(kinds)](lg[i]), osv.MASKED)
    u = words(rng, n)
    t = np.where(np.arange(n) % 3 == 0, 65536, (65536 / rng.uniform(.05, 3, n)).round()).astype(np.int64)
    for k in (1, 2, 50, 300, 512, 513, 5000):
        check_draw(torch, sampler, lg, u, pad, inv_temp=t, top_k=np.full(n, k))
        check_draw(torch, sampler, lg, u, pad, top_k=np.full(n, k), top_p=rng.integers(0, 65537, n), min_p=rng.integers(0, 300, n))
    for p in (100, 30000, 60000, 65000, 65530):
        check_draw(torch, sampler, lg, u, pad, inv_temp=t, top_p=np.full(n, p))
    check_draw(torch, sampler, lg, u, pad, inv_temp=np.where(np.arange(n) % 2, 1, 1 << 22), top_p=np.full(n, 64000))


@pytest.mark.parametrize("n,v,near", [(2, 196609, 0), (1, 229377, 600), (40, 81925, 81925), (70, 49152, 24000), (20, 98304, 30000), (20, 98304, 77777)])
def test_sampling_uneven_blocks(torch, sampler, n, v, near):
    """Rows of several blocks of which some have hardly a logit: rows that end before the last block, and rows
    masked behind (every other one: before) their first `near` logits."""
    rng = np.random.default_rng(near + v)
    lg = (rng.normal(0, 2.6, (n, v)) * 65536).round().astype(np.int64)
    for i in range(n):
        if near and i % 2:
            lg[i, :v - near] = osv.MASKED
        elif near:
            lg[i, near:] = osv.MASKED
    u = words(rng, n)
    for k in (1, 50, 200, 500):
        check_draw(torch, sampler, lg, u, top_k=np.full(n, k))
        check_draw(torch, sampler, lg, u, 1, top_k=np.full(n, k), top_p=np.full(n, 60000))
    check_draw(torch, sampler, lg, u, top_p=np.full(n, 60000))


def test_sampling_refusals(torch, sampler):
    import _eii
    x = torch.zeros(2, 64, dtype=torch.int32, device="cuda")
    u = torch.zeros(2, dtype=torch.int32, device="cuda")
    tok = torch.zeros(2, dtype=torch.int64, device="cuda")
    call = lambda n=2, v=64, **kw: sampler.sample(x.data_ptr(), n, v, u.data_ptr(), tok.data_ptr(), stream=st(torch), **kw)
    for bad in (lambda: call(n=-1), lambda: call(v=0), lambda: call(v=262145), lambda: call(ld=63),
                lambda: sampler.sample(None, 2, 64, u.data_ptr(), tok.data_ptr()),
                lambda: sampler.sample(x.data_ptr(), 2, 64, None, tok.data_ptr()),
                lambda: sampler.sample(x.data_ptr(), 2, 64, u.data_ptr(), None),
                lambda: call(inv_temp_ptr=x.data_ptr() + 2), lambda: call(kept_ptr=x.data_ptr() + 1),
                lambda: sampler.sample(x.data_ptr() + 2, 2, 64, u.data_ptr(), tok.data_ptr())):
        with pytest.raises(_eii.EiiError) as e:
            bad()
        assert e.value.code == _eii.EII_ERR_ARG
    for name, value in (("inv_temp", 0), ("inv_temp", -5), ("inv_temp", (1 << 22) + 1), ("top_k", -1), ("top_p", -1),
                        ("top_p", 65537), ("min_p", -1), ("min_p", 65537)):
        ok = {"inv_temp": 65536, "top_k": 0, "top_p": 65536, "min_p": 0}[name]
        par = torch.tensor([ok, value], dtype=torch.int32, device="cuda")
        tok.fill_(-9)
        call(**{name + "_ptr": par.data_ptr()})
        with pytest.raises(_eii.EiiError, match="parameter"):
            sampler.sync(st(torch))
        assert tok.tolist() == [0, -1]
        sampler.sync(st(torch))
    call(n=0)
    sampler.sample(None, 0, 64, None, None, stream=st(torch))
    sampler.sync(st(torch))


# ------------------------------------------------------------------------- streams, graphs, a run
def test_streams_and_graphs(torch, sampler):
    """Two calls of one handle at once on two streams; a captured step replayed on new data."""
    rng = np.random.default_rng(12)
    lens = [900, 64, 333]
    c = Cache(torch, rng, 9, 3, 64, 16, 4, lens)
    c.fill(rng, lens)
    n = 3
    import _eii
    q = [rng.normal(0, 1500, (n, 9, 64)).round().astype(np.int64) for _ in range(2)]
    want = [np.empty((n, 9, 64), np.int64) for _ in range(2)]
    for a, b in zip(q, want):
        osv.attention(a, np.arange(n), lens, c.table, c.k, c.v, _eii.table_exp(), 17, 16, 16, 16, b)
    dq = [torch.from_numpy(a.astype(np.int16)).cuda() for a in q]
    out = [torch.zeros(n, 576, dtype=torch.int32, device="cuda") for _ in range(2)]
    dlen = torch.tensor(lens, dtype=torch.int32, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for i in range(2):
            c.p.attention(c.pages, dq[i].data_ptr(), n, dlen.data_ptr(), 900, 17, 16, 16, out[i].data_ptr(),
                          stream=streams[i].cuda_stream)
    for i in range(2):
        c.p.sync(streams[i].cuda_stream)
        assert np.array_equal(out[i].cpu().numpy().reshape(n, 9, 64), want[i])
    # capture append + attention + draw, replay with other inputs
    qkv = torch.zeros(n, 15 * 64, dtype=torch.int16, device="cuda")
    pos = torch.zeros(n, dtype=torch.int32, device="cuda")
    length = torch.zeros(n, dtype=torch.int32, device="cuda")
    qr, ctx = torch.zeros(n, 576, dtype=torch.int16, device="cuda"), torch.zeros(n, 576, dtype=torch.int32, device="cuda")
    u, tok = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int64, device="cuda")

    def step():
        c.p.append(c.pages, qkv.data_ptr() + 2 * 576, qkv.data_ptr() + 2 * 768, n, pos.data_ptr(), 30, q_ptr=qkv.data_ptr(),
                   q_out_ptr=qr.data_ptr(), shift_q=30, ldq=960, ldk=960, ldv=960, stream=st(torch))
        c.p.attention(c.pages, qr.data_ptr(), n, length.data_ptr(), 900, 17, 16, 16, ctx.data_ptr(), stream=st(torch))
        sampler.sample(ctx.data_ptr(), n, 576, u.data_ptr(), tok.data_ptr(), stream=st(torch))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for it in range(3):
        x = rng.normal(0, 1500, (n, 15, 64)).round().astype(np.int64)
        p = np.array([899 - it, 10 + it, 300], np.int32)
        w = rng.integers(0, 1 << 32, n, dtype=np.uint64)
        qkv.copy_(torch.from_numpy(x.reshape(n, -1).astype(np.int16)))
        pos.copy_(torch.from_numpy(np.minimum(p, 511)))
        length.copy_(torch.from_numpy(np.minimum(p, 511) + 1))
        u.copy_(torch.from_numpy(w.astype(np.uint32).view(np.int32)))
        g.replay()
        c.p.sync(st(torch))
        wq, wc = np.empty((n, 9, 64), np.int64), np.empty((n, 9, 64), np.int64)
        p = np.minimum(p, 511)
        osv.append(x[:, :9], x[:, 9:12], x[:, 12:], np.arange(n), p, c.table, c.k, c.v, c.rope, 30, 30, wq,
                   np.empty((n, 2, 3, 64), np.int64))
        osv.attention(wq, np.arange(n), p + 1, c.table, c.k, c.v, _eii.table_exp(), 17, 16, 16, 16, wc)
        assert np.array_equal(ctx.cpu().numpy().reshape(n, 9, 64), wc)
        assert tok.tolist() == [osv.draw(wc[r].reshape(-1), w[r])[0] for r in range(n)]
    sampler.sync(st(torch))


@pytest.mark.parametrize("n,v", [(1, 49152), (3, 20000), (30, 128003), (2, 262144)])
def test_sampling_small_top_k_over_blocks_repeated(torch, sampler, n, v):
    """Rows on several blocks with a small top-k whose list takes an odd or an even number of steps, many calls back
    to back: every call gives the first one's tokens, which are the oracle's."""
    rng = np.random.default_rng(v)
    lg = (rng.normal(0, 2.6, (n, v)) * 65536).round().astype(np.int64)
    u = words(rng, n)
    dl = torch.from_numpy(lg.astype(np.int32)).cuda()
    du = torch.from_numpy(u.astype(np.uint32).view(np.int32)).cuda()
    for k in (1, 40, 60, 90, 130, 200, 300, 400, 512):
        dk = torch.full((n,), k, dtype=torch.int32, device="cuda")
        tok = torch.full((200, n), -9, dtype=torch.int64, device="cuda")
        kept = torch.full((200, n), -9, dtype=torch.int32, device="cuda")
        for i in range(200):
            sampler.sample(dl.data_ptr(), n, v, du.data_ptr(), tok[i].data_ptr(), top_k_ptr=dk.data_ptr(),
                           kept_ptr=kept[i].data_ptr(), stream=st(torch))
        sampler.sync(st(torch))
        want = [osv.draw(lg[r], u[r], top_k=k) for r in range(n)]
        assert tok[0].tolist() == [w[0] for w in want] and kept[0].tolist() == [w[1] for w in want]
        assert (tok == tok[0]).all() and (kept == kept[0]).all()


def test_first_call_on_a_stream_of_its_own(torch):
    """New handles whose first call goes to a stream that does not wait for the default one: tables and error words
    are there when the handle is."""
    import _eii
    rng = np.random.default_rng(21)
    lens = [40, 9]
    side = torch.cuda.Stream()
    par = torch.tensor([65536, -1], dtype=torch.int32, device="cuda")
    x = torch.zeros(2, 64, dtype=torch.int32, device="cuda")
    u = torch.zeros(2, dtype=torch.int32, device="cuda")
    tok = torch.zeros(2, dtype=torch.int64, device="cuda")
    a = [rng.integers(-32768, 32768, (2, h, 64)) for h in (9, 3, 3)]
    for i in range(10):
        c = Cache(torch, rng, 9, 3, 64, 16, 16, lens, n_pos=20000)
        d = [torch.from_numpy(y.astype(np.int16)).cuda() for y in a]
        pos = np.array([39, 8], np.int32)
        dpos = torch.from_numpy(pos).cuda()
        torch.cuda.synchronize()
        c.p.close()
        c.p = _eii.Paged(9, 3, 64, 16, 16, rope=c.rope)
        c.p.append(c.pages, d[1].data_ptr(), d[2].data_ptr(), 2, dpos.data_ptr(), 30, q_ptr=d[0].data_ptr(),
                   q_out_ptr=d[0].data_ptr(), shift_q=30, stream=side.cuda_stream)
        s = _eii.Sampler(0)
        s.sample(x.data_ptr(), 2, 64, u.data_ptr(), tok.data_ptr(), top_p_ptr=par.data_ptr(), stream=side.cuda_stream)
        c.p.sync(side.cuda_stream)
        with pytest.raises(_eii.EiiError, match="parameter"):
            s.sync(side.cuda_stream)
        s.close()
        wq = np.zeros((2, 9, 64), np.int64)
        osv.append(*a, np.arange(2), pos, c.table, c.k, c.v, c.rope, 30, 30, wq, np.zeros((2, 2, 3, 64), np.int64))
        assert np.array_equal(d[0].cpu().numpy(), wq)
        c.check_pools()


@pytest.mark.parametrize("heads,kv,hd,bits,n", [(9, 3, 64, 16, 3), (9, 3, 64, 4, 3), (6, 2, 128, 4, 3), (9, 3, 64, 4, 9000), (6, 2, 128, 16, 9000)])
@pytest.mark.parametrize("what", ["seq", "pos", "page", "value"])
def test_append_leaves_what_it_refuses(torch, heads, kv, hd, bits, n, what):
    """A refused row leaves its q_out, its kv_out and the pools as they were; with a value outside int16 only the heads
    that hold one do.  The other rows are appended.  Few rows (warps share a row) and many."""
    import _eii
    rng = np.random.default_rng(n + hd)
    lens = [512] * (-(-n // 512) + 1)
    c = Cache(torch, rng, heads, kv, hd, 16, bits, lens)
    seq, pos = (np.arange(n) // 512).astype(np.int32), (np.arange(n) % 512).astype(np.int32)
    x = [rng.normal(0, 6000, (n, h, hd)).round().clip(-32768, 32767).astype(np.int64) for h in (heads, kv, kv)]
    bad = n // 2
    dseq, dpos, table = seq.copy(), pos.copy(), c.table.copy()
    heads_left = [range(heads), range(kv), range(kv)]
    if what == "seq":
        dseq[bad] = len(lens)
    elif what == "pos":
        dpos[bad] = 512
    elif what == "page":  # (a page of its own: the others' rows lie elsewhere)
        dseq[bad], dpos[bad] = len(lens) - 1, 40
        table[len(lens) - 1, 40 // 16] = c.n_pages
    else:
        heads_left = [[heads - 1], [0], [kv - 1]]
        for a, h, value in zip(x, (heads - 1, 0, kv - 1), (32768, -32769, 1 << 30)):
            a[bad, h, 5] = value
    c.dtable.copy_(torch.from_numpy(table))
    d = [torch.from_numpy(a.astype(np.int32)).cuda() for a in x]
    q_out = torch.full((n, heads, hd), 99, dtype=torch.int16, device="cuda")
    kv_out = torch.full((n, 2, kv, hd), 98, dtype=torch.int32, device="cuda")
    ds, dp = torch.from_numpy(dseq).cuda(), torch.from_numpy(dpos).cuda()
    before = [h.copy() for h in c.host]
    c.p.append(c.pages, d[1].data_ptr(), d[2].data_ptr(), n, dp.data_ptr(), 30, seq_ptr=ds.data_ptr(), q_ptr=d[0].data_ptr(),
               q_out_ptr=q_out.data_ptr(), shift_q=30, in_bits=32, kv_out_ptr=kv_out.data_ptr(), stream=st(torch))
    text = {"seq": "sequence", "pos": "position", "page": "page", "value": "int16"}[what]
    with pytest.raises(_eii.EiiError, match=text):
        c.p.sync(st(torch))
    c.p.sync(st(torch))
    wq, wkv = np.full((n, heads, hd), 99, np.int64), np.full((n, 2, kv, hd), 98, np.int64)
    x = [a.clip(-32768, 32767) for a in x]  # (what stands there instead is put back below)
    if what != "value":
        seq[bad] = -1
    osv.append(*x, seq, pos, c.table, c.k, c.v, c.rope, 30, 30, wq, wkv)
    if what == "value":
        wq[bad, heads - 1] = 99
        for i, (pool, old) in enumerate(((c.k, before[0]), (c.v, before[1]))):
            h = heads_left[1 + i][0]
            wkv[bad, i, h] = 98
            page, slot = int(c.table[seq[bad], pos[bad] // 16]), int(pos[bad] % 16)
            was = osv.Pool(old, kv, hd, 16, bits)
            for at, size in ((slot * pool.row, pool.row), (16 * pool.row + slot * hd // 16, hd // 16 if bits == 4 else 0)):
                pool.data[page, h, at:at + size] = was.data[page, h, at:at + size]
    assert np.array_equal(q_out.cpu().numpy(), wq)
    assert np.array_equal(kv_out.cpu().numpy(), wkv)
    c.check_pools()


@pytest.mark.parametrize("n", [(1 << 30) + 1, (1 << 31) - 1])
def test_sampling_refuses_rows_that_an_int_cannot_step_over(torch, sampler, n):
    import _eii
    x = torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises(_eii.EiiError, match="n_rows") as e:
        sampler.sample(x.data_ptr(), n, 1, x.data_ptr(), x.data_ptr(), stream=st(torch))
    assert e.value.code == _eii.EII_ERR_ARG
    sampler.sync(st(torch))


@pytest.mark.parametrize("heads,kv,hd,bits,inp", [(9, 3, 64, 16, 16), (9, 3, 64, 4, 32), (4, 4, 128, 4, 16), (16, 2, 128, 16, 32)])
@pytest.mark.parametrize("shift", [1, 2, 8, 15, 16, 17, 31, 32, 33, 40, 46, 47, 62])
def test_append_shifts_and_extremes(torch, heads, kv, hd, bits, inp, shift):
    """Every kind of shift, for q and k each with the other's neighbour; q, k and v over the whole int16 range, rows
    of one extreme and rows whose groups hold both (a 4-bit step of 4369); kv_out on a 4-byte boundary."""
    rng = np.random.default_rng(100 * shift + hd)
    n = 24
    c = Cache(torch, rng, heads, kv, hd, 32, bits, [n])
    x = [rng.integers(-32768, 32768, (n, h, hd)) for h in (heads, kv, kv)]
    for a in x:
        a[0], a[1] = -32768, 32767
        a[2], a[3] = rng.choice([-32768, 32767], a[2].shape), rng.integers(-3, 4, a[3].shape)
        a[4, :, ::64], a[4, :, 63::64] = -32768, 32767
    one, zero = np.full((2, hd // 2), 1 << 30, np.int64), np.zeros((2, hd // 2), np.int64)
    for rope in (c.rope, tuple(np.concatenate(t) for t in ((one, -one, zero, c.rope[0]), (zero, zero, one, c.rope[1])))):
        import _eii
        p = _eii.Paged(heads, kv, hd, 32, bits, rope=rope)
        d = [torch.from_numpy(a.astype(np.int16 if inp == 16 else np.int32)).cuda() for a in x]
        pos = rng.permutation(n).astype(np.int32)
        dpos, dseq = torch.from_numpy(pos).cuda(), torch.zeros(n, dtype=torch.int32, device="cuda")
        other = min(max(shift + rng.choice([-1, 1]), 1), 62)
        q_out = torch.full((n, heads, hd), 99, dtype=torch.int16, device="cuda")
        buf = torch.full((n * 2 * kv * hd + 1,), 98, dtype=torch.int32, device="cuda")
        p.append(c.pages, d[1].data_ptr(), d[2].data_ptr(), n, dpos.data_ptr(), shift, seq_ptr=dseq.data_ptr(), q_ptr=d[0].data_ptr(),
                 q_out_ptr=q_out.data_ptr(), shift_q=other, in_bits=inp, kv_out_ptr=buf.data_ptr() + 4, stream=st(torch))
        p.sync(st(torch))
        wq, wkv = np.zeros((n, heads, hd), np.int64), np.zeros((n, 2, kv, hd), np.int64)
        osv.append(*x, np.zeros(n, int), pos, c.table, c.k, c.v, rope, other, shift, wq, wkv)
        assert np.array_equal(q_out.cpu().numpy(), wq)
        got = buf.cpu().numpy()
        assert got[0] == 98 and np.array_equal(got[1:].reshape(wkv.shape), wkv)
        c.check_pools()


def test_calls_after_a_failed_allocation(torch, base_model_path):
    """A decoder whose pools do not fit is refused, and the calls that follow are not blamed for it."""
    import _eii
    rng = np.random.default_rng(14)
    lens = [40] * 500
    e = _eii.Engine(base_model_path, 0)
    try:
        c = Cache(torch, rng, 9, 3, 64, 16, 16, lens)
        c.fill(rng, lens[:0])
        x = [rng.integers(-32768, 32768, (2, h, 64)) for h in (9, 3, 3)]
        d = [torch.from_numpy(a.astype(np.int16)).cuda() for a in x]
        pos, seq = np.array([39, 8], np.int32), np.array([0, 1], np.int32)
        dpos = torch.from_numpy(pos).cuda()

        def refused():
            with pytest.raises(_eii.EiiError) as err:
                _eii.PagedDecoder(e, 1024, 16, (1 << 31) - 1)
            assert err.value.code == _eii.EII_ERR_CUDA
        refused()
        c.p.append(c.pages, d[1].data_ptr(), d[2].data_ptr(), 2, dpos.data_ptr(), 30, stream=st(torch))
        c.p.sync(st(torch))
        osv.append(None, x[1], x[2], seq, pos, c.table, c.k, c.v, c.rope, 30, 30, None, np.zeros((2, 2, 3, 64), np.int64))
        c.check_pools()
        refused()  # (500 short rows: one warp per item)
        check_attention(torch, c, rng, None, [1] * 500, 40)
        refused()
        check_attention(torch, c, rng, [0], [40], 40)
        a, W, one = rng.integers(-100, 100, (4, 32)), rng.integers(-100, 100, (16, 32)), np.ones(16, np.int64)
        refused()
        assert np.array_equal(e.linear(a, 16, W, one, one * 8, 0, 0, 32)[1], a @ W.T)
    finally:
        e.close()
