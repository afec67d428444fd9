"""GPU: penalties, biases and masks on logits against 64 bits.

Tolerance, before any run: a division or product, a product and a sum of the
penalties, their difference and the bias are at most five float32 roundings of
values no larger than the sum of the terms' magnitudes, 2^-24 each; 2^-21 of that
sum allows eight.  The output is rounded once.  What is masked is -infinity."""
import numpy as np
import pytest
import torch

from sili__new_amd import device as dev
from tests import block_ref, draft_ref as ref

pytestmark = pytest.mark.gpu


def gpu(a, dtype=None):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a if dtype is None else np.asarray(a).astype(dtype))).cuda()


def u64(a):
    return None if a is None else torch.from_numpy(np.array([int(m) for m in a], np.uint64).view(np.int64)).cuda()


def constrain(z, out=None, requests=None, stream=None, **kw):
    """kw as of draft_ref.logits; history_stride may be cut with `width`."""
    rows, vocab = z.shape
    k = lambda name: kw.get(name)  # noqa: E731
    t = dict(z=z, out=torch.full_like(z, 7.0) if out is None else out, start=gpu(k("q_start"), np.int32), history=gpu(k("history"), np.int32),
             lens=gpu(k("lens"), np.int32), since=gpu(k("since"), np.int32), tokens=gpu(k("tokens"), np.int32), masks=u64(k("masks")),
             rep=gpu(k("rep"), np.float32), freq=gpu(k("freq"), np.float32), pres=gpu(k("pres"), np.float32), bias=gpu(k("bias"), np.float32),
             allow=gpu(None if k("allow") is None else np.asarray(k("allow"), np.uint32).view(np.int32)), allow_row=gpu(k("allow_row"), np.int32))
    p = {name: None if v is None else v.data_ptr() for name, v in t.items()}
    n = requests if requests is not None else (len(k("q_start")) - 1 if k("q_start") is not None else rows)
    a = dev.LogitsConstrain(dtype=dev.DTYPES[str(z.dtype)[6:]], rows=rows, vocab=vocab, requests=n, logits=p["z"], logits_stride=z.stride(0),
                            out=p["out"], out_stride=t["out"].stride(0), q_start=p["start"], history=p["history"], history_lens=p["lens"],
                            history_stride=0 if t["history"] is None else t["history"].shape[1], counted_from=p["since"], tokens=p["tokens"],
                            ancestors=p["masks"], repetition=p["rep"], presence=p["pres"], frequency=p["freq"], bias=p["bias"],
                            bias_stride=t["bias"].shape[1] if t["bias"] is not None and t["bias"].dim() == 2 else 0, allow=p["allow"],
                            allow_row=p["allow_row"], allow_stride=0 if t["allow"] is None else t["allow"].shape[1],
                            n_allow=0 if t["allow"] is None else t["allow"].shape[0])
    torch.cuda.synchronize()
    dev.logits_constrain(a, stream)
    torch.cuda.synchronize()
    t["args"] = a
    return t


def check(t, z, requests=None, left=7.0, **kw):
    dtype = str(z.dtype)[6:]
    want, size, mine = ref.logits(z.double().cpu().numpy(), requests=requests, **kw)
    got = t["out"].double().cpu().numpy()
    if left is not None:
        assert (got[~mine] == left).all()
    got, want, size = got[mine], want[mine], size[mine]
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    fine = np.isfinite(want)
    assert np.isfinite(got[fine]).all()
    tol = 2.0 ** -21 * size[fine]
    err = np.abs(got[fine] - want[fine])
    tol = tol + block_ref.rounding(dtype, np.abs(want[fine]) + tol)
    assert np.all(err <= tol), np.max(err / tol)


def case(seed, new, vocab, longest, masks=3, bias="each", chained=True):
    """Everything at once: ragged histories, drafted paths, penalties, biases, masks."""
    rng = np.random.default_rng(seed)
    n, rows = len(new), int(np.sum(new))
    words = lambda *s: np.minimum(vocab * rng.random(s) ** 5, vocab - 1).astype(int)  # noqa: E731
    parents = np.concatenate([[int(rng.integers(-1, i)) if i else -1 for i in range(k)] for k in new] + [np.zeros(0, int)]).astype(int)
    start = np.concatenate([[0], np.cumsum(new)])
    lens = rng.integers(0, longest + 1, n)
    lens[0] = longest
    kw = dict(q_start=start, history=words(n, longest), lens=lens, since=(lens * rng.random(n)).astype(int), rep=1 + rng.random(n), freq=rng.random(n),
              pres=rng.random(n), tokens=words(rows), masks=ref.draft_tree(parents, start, [0] * n)[0])
    kw["bias"] = None if bias is None else rng.normal(size=(n, vocab) if bias == "each" else vocab)
    if masks:
        bits = rng.random((masks, -(-vocab // 32) * 32)) < np.array([0.9, 0.5, 0.02])[np.arange(masks) % 3, None]
        kw["allow"] = np.packbits(bits.reshape(masks, -1, 8), axis=-1, bitorder="little").reshape(masks, -1).view(np.uint32)
        kw["allow_row"] = rng.integers(-1, masks + 1, rows)
    return rng, kw


def logits(rng, rows, vocab, dtype):
    return torch.from_numpy((3 * rng.normal(size=(rows, vocab))).astype(np.float32)).cuda().to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [1, 7, 32, 33, 1000, 4095, 4096, 4097, 9001])
@pytest.mark.parametrize("new,longest", [([1], 1), ([1, 1, 1], 300), ([5, 0, 1, 12], 77), ([64, 3], 1500)])
def test_all_of_it(hip, new, longest, vocab, dtype):
    rng, kw = case(vocab + longest, new, vocab, longest, bias=["each", "one"][vocab % 2])
    z = logits(rng, int(np.sum(new)), vocab, dtype)
    check(constrain(z, **kw), z, **kw)


@pytest.mark.parametrize("drop", ["history", "path", "rep", "freq", "pres", "bias", "allow", "since", "allow_row", "all"])
def test_each_part_may_be_absent(hip, drop):
    rng, kw = case(3, [4, 1, 9], 5000, 200)
    names = dict(history=["history", "lens", "since"], path=["tokens", "masks"], allow=["allow", "allow_row"],
                 all=["history", "lens", "since", "tokens", "masks", "rep", "freq", "pres", "bias", "allow", "allow_row"]).get(drop, [drop])
    if drop == "allow_row":
        kw["allow"] = np.tile(kw["allow"], (5, 1))  # a mask a row, and one row past them
    for name in names:
        kw[name] = None
    z = logits(rng, 14, 5000, torch.float32)
    if drop == "allow_row":
        assert len(kw["allow"]) == 15
    t = constrain(z, **kw)
    check(t, z, **kw)
    if drop == "all":
        assert torch.equal(t["out"], z)


def test_a_row_a_request_without_starts(hip):
    rng, kw = case(5, [1] * 6, 3000, 90)
    kw["q_start"] = None
    z = logits(rng, 6, 3000, torch.bfloat16)
    check(constrain(z, **kw), z, **kw)
    short = dict(kw, tokens=kw["tokens"][:4], masks=kw["masks"][:4], allow_row=kw["allow_row"][:4])  # more requests than rows
    check(constrain(z[:4], requests=6, **short), z[:4], requests=4, **short)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_in_place_and_with_strides(hip, dtype):
    rng, kw = case(6, [3, 8], 1777, 64)
    z = logits(rng, 11, 1777, dtype)
    wide = torch.full((11 * 1801 + 1,), 3.0, device="cuda").to(dtype)
    view = wide[1:].view(11, 1801)[:, 5:1782]
    view.copy_(z)
    check(constrain(view, out=view, **kw), z, **kw)
    rest = torch.cat([wide[:1], wide[1:].view(11, 1801)[:, :5].flatten(), wide[1:].view(11, 1801)[:, 1782:].flatten()])
    assert float((rest.float() - 3).abs().max()) == 0
    out = torch.full((11, 1790), 3.0, device="cuda").to(dtype)
    check(constrain(z, out=out[:, 1:1778], **kw), z, **kw)
    assert float((out[:, 0].float() - 3).abs().max()) == 0 and float((out[:, 1778:].float() - 3).abs().max()) == 0


def test_masks_that_leave_nothing_and_values_that_are_not_finite(hip):
    vocab = 100
    z = torch.zeros(4, vocab, device="cuda")
    z[0] = float("nan")
    z[1] = float("inf")
    z[2, 3], z[2, 4], z[2, 5] = float("nan"), float("inf"), torch.finfo(torch.float32).min
    allow = np.zeros((2, 4), np.uint32)
    allow[1, 0] = 0b111000
    t = constrain(z, allow=allow, allow_row=[0, 0, 1, 1])
    out = t["out"].cpu().numpy()
    assert np.isneginf(out[:2]).all() and np.isneginf(np.delete(out[2], [3, 4, 5])).all()
    assert np.isnan(out[2, 3]) and np.isposinf(out[2, 4]) and out[2, 5] == torch.finfo(torch.float32).min and (out[3, 3:6] == 0).all()


def test_tokens_and_lengths_of_any_value(hip):
    """Tokens outside the vocabulary, lengths past the buffer and below 0, masks past the request, starts of any value."""
    rng, kw = case(7, [3, 2, 4], 500, 40)
    kw["history"][0, :6] = [-1, 500, 501, 2 ** 31 - 1, -2 ** 31, 499]
    kw["tokens"][[0, 4, 7]] = [-1, 500, 2 ** 31 - 1]
    kw["lens"][:] = [2 ** 31 - 1, -5, 30]
    kw["since"][:] = [-2 ** 31, 0, 2 ** 31 - 1]
    kw["masks"] = [2 ** 64 - 1] * 9
    z = logits(rng, 9, 500, torch.float32)
    check(constrain(z, **kw), z, **kw)
    for start in ([0, 3, 5, 30], [-1, 3, 5, 9], [4, 2, 5, 7], [0, 9, 9, 2 ** 31 - 1], [2 ** 31 - 1, 2 ** 31 - 1, 0, 4]):
        k = dict(kw, q_start=np.array(start), masks=[1] * 9)
        t = constrain(z, **k)
        if start[2] >= start[1] and start[3] >= start[2] or start[0] == 4:
            check(t, z, **k)


def test_a_token_that_is_often_repeated(hip):
    """Counts of one token from many threads, and a path that holds a token twice."""
    n = 5000
    kw = dict(q_start=[0, 4], history=np.full((1, n), 17), lens=[n], since=[100], tokens=[17, 17, 3, 3], masks=[1, 3, 0b101, 0b1101], rep=[1.5],
              freq=[0.001], pres=[0.25])
    rng = np.random.default_rng(1)
    z = logits(rng, 4, 50, torch.float32)
    check(constrain(z, **kw), z, **kw)


@pytest.mark.parametrize("vocab,requests,nodes", [(30000, 70, 8), (9000, 140, 5), (5000, 20, 12)])
def test_rows_with_and_without_a_path_in_a_chunk(hip, vocab, requests, nodes):
    """A path's tokens lie in few chunks, so a block's rows with barriers follow rows without; large and small chunks."""
    rng = np.random.default_rng(requests)
    for dtype in (torch.float32, torch.bfloat16):
        _, kw = case(int(rng.integers(1000)), [nodes] * requests, vocab, 40, bias="one")
        kw["tokens"] = rng.integers(0, vocab, requests * nodes)
        z = logits(rng, requests * nodes, vocab, dtype)
        t = constrain(z, **kw)
        check(t, z, **kw)
        for _ in range(3):
            assert torch.equal(t["out"], constrain(z, **kw)["out"])


def test_more_rows_of_a_request_than_a_wave_has_lanes(hip):
    """A block that goes over 150 rows, each with a mask of its own, beside a thousand requests of a row."""
    new = [150] + [1] * 600 + [0] * 423
    rng, kw = case(12, [1] * len(new), 37, 20)
    rows = int(np.sum(new))
    kw.update(q_start=np.concatenate([[0], np.cumsum(new)]), tokens=rng.integers(0, 37, rows), allow_row=rng.integers(-1, 4, rows),
              masks=[int(rng.integers(0, 2 ** 63)) for _ in range(150)] + [1] * 600)
    for dtype in (torch.float32, torch.bfloat16):
        z = logits(rng, rows, 37, dtype)
        check(constrain(z, **kw), z, **kw)


def test_a_large_vocabulary_and_a_long_history(hip):
    rng, kw = case(9, [2], 131071, 20000, masks=1, bias="one")
    z = logits(rng, 2, 131071, torch.bfloat16)
    s = constrain(z, **kw)
    check(s, z, **kw)
    assert torch.equal(s["out"], constrain(z, **kw)["out"])


def test_offsets_past_32_bits(hip):
    """Rows more than 4 GiB apart."""
    rng, kw = case(10, [3, 2], 700, 30)
    z = logits(rng, 5, 700, torch.float32)
    far = torch.zeros(5, 300 << 20, device="cuda")
    far[:, :700] = z
    t = constrain(far[:, :700], out=far[:, :700], **kw)
    check(t, z, **kw)


def test_replayed_with_longer_histories(hip):
    rng, kw = case(11, [6, 1, 9], 6000, 500)
    kw["lens"] = np.array([100, 0, 400])
    kw["since"] = np.array([50, 0, 400])
    z = logits(rng, 16, 6000, torch.bfloat16)
    st = torch.cuda.Stream()
    t = constrain(z, stream=st.cuda_stream, **kw)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        dev.logits_constrain(t["args"], st.cuda_stream)
    for step in range(3):
        t["lens"] += 20
        t["z"].mul_(0.5)
        t["out"].fill_(7)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        kw["lens"] = kw["lens"] + 20
        check(t, t["z"], **kw)
        assert torch.equal(t["out"], constrain(t["z"], **kw)["out"])
