"""The model on a paged cache: ragged steps against the forward pass (16 bits), against the oracle's
compressed forward pass (4 bits), and a generation loop with the sampler."""
import numpy as np
import pytest

from oracle import serving as osv

pytestmark = pytest.mark.gpu

V = 49152


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.fixture(scope="module")
def eng(base_model_path):
    import _eii
    e = _eii.Engine(base_model_path, 0)
    yield e
    e.close()


class Run:
    """A paged decoder with a page table whose pages are handed out in shuffled order."""

    def __init__(self, torch, eng, page, bits, n_seq, max_T, seed=0):
        import _eii
        self.t, self.cols, self.n_seq = torch, -(-max_T // page), n_seq
        n_pages = n_seq * self.cols + 2
        self.table = np.random.default_rng(seed).permutation(n_pages)[:n_seq * self.cols].reshape(n_seq, -1).astype(np.int32)
        self.d_table = torch.from_numpy(self.table).cuda()
        self.d = _eii.PagedDecoder(eng, page, bits, n_pages)

    def step(self, ids, seq, pos, max_len=512, logits=True, sync=True):
        t = self.t
        n = len(seq)
        d_ids = ids if isinstance(ids, t.Tensor) else t.tensor(np.asarray(ids), dtype=t.int64, device="cuda")
        d_seq, d_pos = (t.tensor(np.asarray(x), dtype=t.int32, device="cuda") for x in (seq, pos))
        out = t.full((n, V), -7, dtype=t.int32, device="cuda") if logits else None
        st = t.cuda.current_stream().cuda_stream
        if st == 0:  # (a null stream is the engine's own, which does not wait for torch's)
            t.cuda.synchronize()
        self.d.step_device_async(d_ids.data_ptr(), d_seq.data_ptr(), d_pos.data_ptr(), n, self.d_table.data_ptr(), self.cols,
                                 self.n_seq, max_len, out.data_ptr() if logits else None, stream=st)
        if sync:
            self.d.sync(st)
        return out


@pytest.mark.parametrize("page,chunk", [(16, 0), (64, 0), (32, 7)])
def test_ragged_steps_equal_the_forward_pass(torch, eng, page, chunk, monkeypatch):
    """Prompts of different lengths in one step, a prompt in two parts, single tokens with padding between
    them, and a step in chunks of seven rows: every logits row equals the forward pass's."""
    if chunk:
        monkeypatch.setenv("EII_CHUNK_ROWS", str(chunk))
    rng = np.random.default_rng(page)
    lens = [5, 23, 70, 1]
    ids = [rng.integers(0, V, n) for n in lens]
    want = [eng.forward(x)["logits"][0] for x in ids]
    run = Run(torch, eng, page, 16, 4, 70)
    first = [3, 20, 66, 0]  # what the first step holds of each sequence
    rows = [(s, t) for s in range(4) for t in range(first[s])]
    order = np.argsort([t * 4 + s for s, t in rows], kind="stable")  # sequences interleaved, positions ascending
    rows = [rows[i] for i in order]
    got = run.step([ids[s][t] for s, t in rows], *zip(*rows)).cpu().numpy()
    for (s, t), row in zip(rows, got):
        assert np.array_equal(row, want[s][t]), (s, t)
    left = [[(s, t) for t in range(first[s], lens[s])] for s in range(4)]
    while any(left):
        rows = [r.pop(0) if r else (-1, 0) for r in left]
        got = run.step([ids[s][t] if s >= 0 else 0 for s, t in rows], *zip(*rows)).cpu().numpy()
        for (s, t), row in zip(rows, got):
            if s >= 0:
                assert np.array_equal(row, want[s][t]), (s, t)


def test_compressed_cache_equals_the_oracle(torch, eng, base_model):
    rng = np.random.default_rng(3)
    lens = [9, 18]
    ids = [rng.integers(0, V, n) for n in lens]
    want = [osv.forward_compressed(base_model, x) for x in ids]
    run = Run(torch, eng, 16, 4, 2, 18)
    rows = [(s, t) for s in range(2) for t in range(lens[s] - 1)]
    got = run.step([ids[s][t] for s, t in rows], *zip(*rows)).cpu().numpy()
    for (s, t), row in zip(rows, got):
        assert np.array_equal(row, want[s][t]), (s, t)
    got = run.step([x[-1] for x in ids], [0, 1], [n - 1 for n in lens]).cpu().numpy()
    for s in range(2):
        assert np.array_equal(got[s], want[s][-1])


@pytest.mark.parametrize("bits", [16, 4])
def test_generation_on_the_device(torch, eng, bits):
    """Prompt, then steps whose tokens the sampler draws on the device, with no host read between; the drawn
    tokens replayed through the forward pass (16 bits) give the same logits and the same draws."""
    import _eii
    rng = np.random.default_rng(11)
    lens, steps, n = [7, 30, 16], 6, 3
    ids = [rng.integers(0, V, m) for m in lens]
    run = Run(torch, eng, 16, bits, n, 40, seed=5)
    s = _eii.Sampler(0)
    side = torch.cuda.Stream()
    i32 = dict(dtype=torch.int32, device="cuda")
    u = torch.tensor(rng.integers(-(1 << 31), 1 << 31, (steps, n)), **i32)
    k, p, b = torch.tensor([40, 0, 1], **i32), torch.tensor([60000, 50000, 65536], **i32), torch.tensor([65536, 90000, 65536], **i32)
    tokens = torch.zeros(steps, n, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        rows = [(a, t) for a in range(n) for t in range(lens[a])]
        last = np.cumsum(lens) - 1
        logits = [run.step([ids[a][t] for a, t in rows], *zip(*rows), max_len=64, sync=False)[torch.tensor(last, device="cuda")]]
        for i in range(steps):
            lg = logits[-1]
            s.sample(lg.data_ptr(), n, V, u[i].data_ptr(), tokens[i].data_ptr(), inv_temp_ptr=b.data_ptr(), top_k_ptr=k.data_ptr(),
                     top_p_ptr=p.data_ptr(), stream=side.cuda_stream)
            logits.append(run.step(tokens[i], [0, 1, 2], [m + i for m in lens], max_len=64, sync=False))
        s.sync(side.cuda_stream)
        run.d.sync(side.cuda_stream)
    tok = tokens.cpu().numpy()
    for a in range(n):
        if bits == 16:
            want = eng.forward(np.concatenate([ids[a], tok[:, a]]))["logits"][0]
        for i in range(steps):
            row = logits[i][a].cpu().numpy()
            if bits == 16:
                assert np.array_equal(row, want[lens[a] - 1 + i])
            w = int(u[i, a].item()) & 0xFFFFFFFF
            assert tok[i, a] == osv.draw(row.astype(np.int64), w, inv_temp=int(b[a]), top_k=int(k[a]), top_p=int(p[a]))[0]


def test_paged_decoder_refusals(torch, eng):
    import _eii
    for args in ((16, 8, 4), (12, 16, 4), (16, 16, 0)):
        with pytest.raises(_eii.EiiError):
            _eii.PagedDecoder(eng, *args)
    run = Run(torch, eng, 16, 16, 2, 32)
    ids = [5, 6]
    for kw in (dict(max_len=0), dict(max_len=513)):
        with pytest.raises(_eii.EiiError):
            run.step(ids, [0, 1], [0, 0], **kw)
    for seq, pos, max_len in (([0, 2], [0, 0], 512), ([0, 1], [0, 32], 512), ([0, 1], [0, 512], 512), ([0, 1], [0, 4], 4)):
        with pytest.raises(_eii.EiiError) as e:
            run.step(ids, seq, pos, max_len=max_len)
        assert e.value.code == _eii.EII_ERR_ARG
    with pytest.raises(_eii.EiiError, match="token id"):
        run.step([5, V], [0, 1], [0, 0])
    want = eng.forward(np.array([[5], [6]]))["logits"][:, 0]
    assert np.array_equal(run.step(ids, [0, 1], [0, 0]).cpu().numpy(), want)
    run.d.step_device_async(None, None, None, 0, None, 1, 1, 1)
    run.d.sync()


def test_engine_closed_before_its_decoders(torch, base_model_path):
    """Decoders that are still open, a step on its way among them, when their engine is closed: they are closed with
    it, refuse further calls, and the next engine works."""
    import _eii
    for _ in range(2):
        e = _eii.Engine(base_model_path, 0)
        run, dense = Run(torch, e, 16, 4, 2, 32), _eii.Decoder(e, 2, 8)
        run.step([5, 6], [0, 1], [0, 0], sync=False)
        dense.prefill(np.array([[5], [6]]))
        e.close()
        assert not run.d.h and not dense.h
        for call in (lambda: run.d.sync(), lambda: dense.step([1, 2]), lambda: run.step([5, 6], [0, 1], [1, 1])):
            with pytest.raises(_eii.EiiError, match="decoder is null"):
                call()
        run.d.close()
        dense.close()


def test_sync_names_the_error_it_returns(torch, eng):
    """A step with a bad token id and a bad index reports the index, in its own words, and clears both; a bad token id
    alone is reported as such."""
    import _eii
    run = Run(torch, eng, 16, 16, 2, 32)
    for seq, pos, text in (([0, 2], [0, 0], "not below n_seq"), ([0, 1], [0, 32], "position lies outside"),
                           ([0, 1], [0, 0], "token id")):
        with pytest.raises(_eii.EiiError, match=text) as e:
            run.step([V, 6], seq, pos)
        assert e.value.code == _eii.EII_ERR_ARG
        run.d.sync()
    want = eng.forward(np.array([[5], [6]]))["logits"][:, 0]
    assert np.array_equal(run.step([5, 6], [0, 1], [0, 0]).cpu().numpy(), want)


def test_largest_position_is_refused(torch, eng):
    """A position of 2^31 - 1, whose length is no int, is refused like any other outside the table, and leaves the
    other rows alone."""
    import _eii
    run = Run(torch, eng, 16, 16, 2, 32)
    for pos in ((1 << 31) - 1, (1 << 31) - 2, 512):
        out = run.step([5, 6], [0, 1], [0, pos], sync=False)
        with pytest.raises(_eii.EiiError, match="position|length"):
            run.d.sync(0)
        run.d.sync(0)
        assert np.array_equal(out[0].cpu().numpy(), eng.forward(np.array([[5]]))["logits"][0, 0])


def paged_equals_forward(torch, e, ids, n_steps=3):
    """All but the last tokens of two sequences in one step without logits, the rest one by one: the forward pass's rows."""
    want = [e.forward(x)["logits"][0] for x in ids]
    run = Run(torch, e, 16, 16, len(ids), max(len(x) for x in ids), seed=2)
    rows = [(s, t) for s, x in enumerate(ids) for t in range(len(x) - n_steps)]
    assert run.step([ids[s][t] for s, t in rows], *zip(*rows), logits=False) is None
    for i in range(n_steps):
        at = [len(x) - n_steps + i for x in ids]
        got = run.step([x[t] for x, t in zip(ids, at)], list(range(len(ids))), at).cpu().numpy()
        for s, t in enumerate(at):
            assert np.array_equal(got[s], want[s][t]), (s, t)


@pytest.mark.parametrize("switch", ["EII_O_FEATURE_MAJOR", "EII_DOWN_ROW_MAJOR", "EII_LOGITS_FEATURE_MAJOR", "EII_NO_NORM_FUSION", "grid"])
def test_steps_with_the_engines_switches(torch, outlier_model_path, switch, monkeypatch):
    """The other layouts of the planes that the attention writes and of those behind it, and the narrow residual grid."""
    import _eii
    rng = np.random.default_rng(8)
    if switch != "grid":
        monkeypatch.setenv(switch, "1")
    e = _eii.Engine(outlier_model_path, 0)
    try:
        if switch == "grid":
            e.set_residual_grid(rng.integers(0, 4, 30), rng.integers(0, 4, 30))
        paged_equals_forward(torch, e, [rng.integers(0, V, n) for n in (37, 150)])
    finally:
        e.close()


def test_step_of_more_rows_than_a_chunk(torch, eng):
    """A prompt step of more rows than the engine's workspace takes at once."""
    rng = np.random.default_rng(9)
    ids = [rng.integers(0, V, 420) for _ in range(160)]
    run = Run(torch, eng, 64, 16, len(ids), 420)
    rows = [(s, t) for s in range(len(ids)) for t in range(419)]
    assert len(rows) > 65536
    run.step([ids[s][t] for s, t in rows], *zip(*rows), logits=False)
    got = run.step([x[419] for x in ids], list(range(len(ids))), [419] * len(ids)).cpu().numpy()
    for s in (0, 78, 79, 80, 159):
        assert np.array_equal(got[s], eng.forward(ids[s])["logits"][0][419]), s
