"""q3s_process_logits through the Python binding against the 64-bit
restatement (oracle/step_oracle.py).

Bar: every entry within the sum of its f32 roundings (plus one bf16 rounding
for bf16 outputs), infinities and NaN in the same places, statuses exact.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - collected on CPU boxes
    pytest.skip("needs a CUDA device", allow_module_level=True)

import q3s  # noqa: E402
import step_oracle as so  # noqa: E402

DEV = torch.device("cuda:0")
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
IDS = {"u16": torch.int16, "u32": torch.int32, "i64": torch.int64}


class Case:
    """A batch on the device with its host form."""

    def __init__(self, seed, R, V, dtype="f32", out="f32", ids="u32", hist=40, bias=6, masks=3,
                 gap=0, shift=0, ends=False, prompts=True, keep=0.6):
        rng = np.random.default_rng(seed)
        x = rng.standard_normal((R, V)) * 2.5
        buf = torch.zeros(R * (V + gap) + shift, dtype=TYPES[dtype], device=DEV)
        rows = buf[shift:].view(R, V + gap)[:, :V]
        rows.copy_(torch.from_numpy(x).to(DEV))
        self.logits, self.R, self.V, self.out_dtype = rows, R, V, TYPES[out]
        self.x = rows.double().cpu().numpy()
        self.args = {"out_dtype": self.out_dtype}
        self.oracle = {}
        if hist:
            lens = rng.integers(0, hist + 1, R)
            lens[rng.integers(0, R)] = 0
            if R > 1:
                lens[-1] = hist
            # Repeats, and ids at and beyond the vocabulary.
            pool = np.concatenate([rng.integers(0, V, max(1, min(V, 12))),
                                   rng.integers(0, V + 3, 8)])
            hs = [rng.choice(pool, n) for n in lens]
            slot = hist + 3
            flat = np.full(R * slot if ends else int(lens.sum()) + 1, 1, np.int64)
            offs = np.arange(R + 1) * slot if ends else np.concatenate([[0], np.cumsum(lens)])
            for r in range(R):
                flat[offs[r]:offs[r] + lens[r]] = hs[r]
            self.args.update(history=torch.from_numpy(flat).to(IDS[ids]).to(DEV),
                             history_offsets=torch.from_numpy(offs).to(DEV))
            if ends:
                self.args["history_ends"] = torch.from_numpy(offs[:R] + lens).to(DEV)
            pen = np.stack([rng.uniform(0.7, 1.6, R), rng.uniform(-1, 1, R),
                            rng.uniform(-0.3, 0.6, R)], 1).astype(np.float32)
            pen[rng.random(R) < 0.2, 0] = 1.0
            pen[rng.random(R) < 0.2, 1:] = 0.0
            self.args["penalties"] = torch.from_numpy(pen).to(DEV)
            self.oracle.update(penalties=pen, histories=hs)
            if prompts:
                pl = rng.integers(0, hist + 2, R)
                self.args["prompt_lens"] = torch.from_numpy(pl).to(DEV)
                self.oracle["prompt_lens"] = pl
        if bias:
            counts = rng.integers(0, bias + 1, R)
            lists = []
            for n in counts:
                i = rng.integers(0, V + 2, n)
                v = (rng.standard_normal(n) * 5).astype(np.float32)
                v[rng.random(n) < 0.1] = -np.inf
                lists.append(list(zip(i.tolist(), v.tolist())))
            offs = np.concatenate([[0], np.cumsum(counts)])
            flat = [e for row in lists for e in row]
            self.args.update(
                bias_ids=torch.tensor([i for i, _ in flat], dtype=torch.int32, device=DEV),
                bias_values=torch.tensor([v for _, v in flat], dtype=torch.float32, device=DEV),
                bias_offsets=torch.from_numpy(offs).to(DEV))
            self.oracle["biases"] = lists
        if masks:
            allowed = rng.random((masks, V)) < keep
            allowed[0] = False  # a mask that leaves nothing
            which = rng.integers(-1, masks, R)
            self.args.update(masks=q3s.pack_mask(torch.from_numpy(allowed).to(DEV)),
                             mask_rows=torch.from_numpy(which).to(torch.int32).to(DEV))
            self.oracle["allowed"] = [None if m < 0 else allowed[m] for m in which]

    def check(self, out, status, rows=None):
        value, bound = so.process_logits(self.x, **self.oracle)
        bf16 = self.out_dtype == torch.bfloat16
        so.check(out.double().cpu().numpy(), value, so.rounded(bound, value, bf16))
        assert (status.cpu().numpy() == 0).all()


def run(case, **more):
    out, status = q3s.process_logits(case.logits, **{**case.args, **more})
    torch.cuda.synchronize()
    return out, status


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"),
                                       ("f32", "bf16")])
@pytest.mark.parametrize("V", [1, 2, 31, 33, 255, 2048, 3072, 4095, 4097, 9001])
def test_matches_the_definition(V, dtype, out):
    c = Case(V, 9, V, dtype, out, ids="i64" if V % 2 else "u16")
    c.check(*run(c))


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("gap,shift", [(1, 0), (8, 0), (3, 5), (0, 1), (16, 2)])
def test_strides_and_alignments(gap, shift, dtype, out):
    for V in (70, 2048, 5003):
        c = Case(V + gap, 6, V, dtype, out, gap=gap, shift=shift, ends=True)
        c.check(*run(c))
        # An output with a row stride and a start of its own.
        buf = torch.full((6 * (V + 3) + 3,), 7.0, dtype=TYPES[out], device=DEV)
        res = buf[1:1 + 6 * (V + 3)].view(6, V + 3)[:, :V]
        st = torch.empty(6, dtype=torch.uint8, device=DEV)
        c.check(*run(c, out=(res, st)))
        gaps = buf[1:1 + 6 * (V + 3)].view(6, V + 3)[:, V:]
        assert (gaps == 7).all() and buf[0] == 7 and (buf[-2:] == 7).all()


@pytest.mark.parametrize("R", [1, 2, 147, 1500])
@pytest.mark.parametrize("parts", [("hist",), ("bias",), ("masks",), ()])
def test_each_part_alone(R, parts):
    sizes = {k: (20 if k in parts else 0) for k in ("hist", "bias", "masks")}
    c = Case(R, R, 520, prompts=False, **sizes)
    c.check(*run(c))


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("R,V", [(300, 3072), (140, 14001), (200, 20003), (160, 30007), (400, 9000)])
def test_rows_shared_between_blocks(R, V, dtype, out):
    """Parts of one row from a third of 3072 entries to more than 5000."""
    c = Case(R + V, R, V, dtype, out, hist=40, bias=12, masks=3, ids="u32")
    c.check(*run(c))


@pytest.mark.parametrize("V", [700, 30000])
def test_long_histories_and_bias_lists(V):
    c = Case(5, 4, V, hist=20000, bias=900, ids="u32", ends=True)
    c.check(*run(c))


@pytest.mark.parametrize("ids", ["u16", "u32", "i64"])
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
def test_ids_that_no_vocabulary_has(ids, shift):
    """Negative ids, the largest, and those right behind the row, where rows
    start behind a vector's start: nothing changes, in the row or around it."""
    V, R = 50, 3
    top = {"u16": 2 ** 15 - 1, "u32": 2 ** 31 - 1, "i64": 2 ** 63 - 1}[ids]
    none = [-1, -2, -3, -4, -7, V, V + 1, V + 3, top, -top - 1, -2 ** 31 + 5 if ids != "u16" else 99]
    hist = torch.tensor(none * R, dtype=IDS[ids], device=DEV)
    offs = torch.arange(R + 1, device=DEV) * len(none)
    buf = torch.randn(R * (V + 4) + 8, device=DEV)
    res = torch.full_like(buf, 3.0)
    x, out = (t[shift:shift + R * (V + 4)].view(R, V + 4)[:, :V] for t in (buf, res))
    st = torch.empty(R, dtype=torch.uint8, device=DEV)
    bias = torch.tensor([-1, V, -2 ** 31], dtype=torch.int32, device=DEV)
    q3s.process_logits(x, penalties=torch.tensor([2.0, 1.0, 1.0], device=DEV), history=hist,
                       history_offsets=offs, bias_ids=bias, bias_values=torch.ones(3, device=DEV),
                       bias_offsets=torch.tensor([0, 3, 3, 3], device=DEV), out=(out, st))
    assert torch.equal(out, x) and (st == 0).all()
    res[shift:shift + R * (V + 4)].view(R, V + 4)[:, :V] = 3.0
    assert (res == 3.0).all()


def test_repeated_bias_ids_add_up_in_list_order():
    """Values whose f32 sum depends on the order, across groups of 32."""
    V, n = 100, 150
    rng = np.random.default_rng(3)
    ids = rng.choice([7, 9, 11], n)
    values = (rng.standard_normal(n) * 10.0 ** rng.integers(-4, 5, n)).astype(np.float32)
    x = torch.zeros((1, V), device=DEV)
    out, _ = q3s.process_logits(
        x, bias_ids=torch.from_numpy(ids).to(torch.int32).to(DEV),
        bias_values=torch.from_numpy(values).to(DEV),
        bias_offsets=torch.tensor([0, n], device=DEV))
    want = np.zeros(V, np.float32)
    for i in (7, 9, 11):
        s = None
        for v in values[ids == i]:
            s = v if s is None else np.float32(s + v)
        want[i] = s
    np.testing.assert_array_equal(out.cpu().numpy()[0], want)


def test_masked_row_leaves_nothing_and_the_sampler_says_so():
    V = 2048
    x = torch.randn((4, V), device=DEV)
    x[1, 5], x[2, 6] = float("nan"), float("inf")
    allowed = torch.zeros((2, V), dtype=torch.bool, device=DEV)
    allowed[1, 77] = True
    which = torch.tensor([0, 0, 0, 1], dtype=torch.int32, device=DEV)
    out, st = q3s.process_logits(x, masks=q3s.pack_mask(allowed), mask_rows=which)
    assert torch.isinf(out[:3]).all() and (out[:3] < 0).all() and (st == 0).all()
    assert out[3, 77] == x[3, 77] and int(torch.isfinite(out[3]).sum()) == 1
    seeds = torch.arange(4, device=DEV)
    tok, status = q3s.sample_batch(out, q3s.make_params(1, top_k=50), seeds, seeds)
    assert status.tolist() == [q3s.STATUS_NO_CANDIDATE] * 3 + [q3s.STATUS_OK]
    assert int(tok[3]) == 77


def test_lowest_values_infinities_and_nan():
    """The type's lowest value, infinities, NaN and signed zeros as logits."""
    special = [np.inf, -np.inf, np.nan, np.finfo(np.float32).min, np.finfo(np.float32).max, 0.0,
               -0.0, 1e-45, -1e-45]
    c = Case(17, 3, 64, hist=30, bias=0)
    x = c.x.copy()
    x[:, :len(special)] = special
    c.logits.copy_(torch.from_numpy(x).to(DEV))
    c.x = c.logits.double().cpu().numpy()
    hs = [list(range(12)) + list(h) for h in c.oracle["histories"]]
    flat = np.concatenate(hs).astype(np.int64)
    offs = np.concatenate([[0], np.cumsum([len(h) for h in hs])])
    pen = np.array([[1.3, 0.0, 0.0], [0.8, 0.5, 0.25], [1.0, -0.5, 0.1]], np.float32)
    c.oracle.update(histories=hs, penalties=pen, prompt_lens=[0, 3, 5])
    out, st = q3s.process_logits(
        c.logits, penalties=torch.from_numpy(pen).to(DEV),
        history=torch.from_numpy(flat).to(DEV), history_offsets=torch.from_numpy(offs).to(DEV),
        prompt_lens=torch.tensor([0, 3, 5], device=DEV), masks=c.args["masks"],
        mask_rows=c.args["mask_rows"])
    value, bound = so.process_logits(c.x, **c.oracle)
    # The largest magnitudes overflow f32 where 64 bits do not; subnormals
    # round to their own step.
    top = np.finfo(np.float32).max
    value = np.where(value >= top * (1 + 2.0 ** -25), np.inf, value)
    value = np.where(value <= -top * (1 + 2.0 ** -25), -np.inf, value)
    bound = bound + 2.0 ** -149
    so.check(out.double().cpu().numpy(), value, bound)
    # A row that nothing touches keeps its bits, the sign of zero included.
    same, _ = q3s.process_logits(c.logits)
    assert torch.equal(same.view(torch.int32), c.logits.contiguous().view(torch.int32))


def test_invalid_rows_fail_closed():
    R, V = 9, 300
    x = torch.randn((R, V), device=DEV)
    pen = torch.ones((R, 3), device=DEV) * torch.tensor([1.1, 0.1, 0.1], device=DEV)
    pen[0, 0], pen[1, 0], pen[2, 0] = 0.0, float("nan"), -1.0
    pen[3, 1], pen[4, 2], pen[5, 0] = float("inf"), float("nan"), float("inf")
    allowed = torch.ones((2, V), dtype=torch.bool, device=DEV)
    which = torch.tensor([0, 0, 0, 0, 0, 0, 2, 1, -5], dtype=torch.int32, device=DEV)
    out, st = q3s.process_logits(x, penalties=pen, masks=q3s.pack_mask(allowed), mask_rows=which)
    rp, pe = q3s.STATUS_INVALID_REPETITION_PENALTY, q3s.STATUS_INVALID_PENALTY
    assert st.tolist() == [rp, rp, rp, pe, pe, rp, q3s.STATUS_INVALID_MASK, 0, 0]
    assert (out[:7] == -float("inf")).all()
    assert torch.equal(out[7:], x[7:])


def test_rows_of_their_own_vocabulary():
    """row_offsets / row_vocab: rows of several lengths in one flat array; a
    length outside [0, vocab] is refused and the row is left alone."""
    vocabs = [3072, 2048, 1, 0, 2047, 4000, -1]
    offs = np.concatenate([[3], 3 + np.cumsum(np.maximum(vocabs, 0)[:-1] + 5)])
    rng = np.random.default_rng(4)
    flat = torch.from_numpy(rng.standard_normal(int(offs[-1]) + 10)).float().to(DEV)
    hist = torch.from_numpy(rng.integers(0, 3100, 7 * 64)).to(torch.int32).to(DEV)
    hoff = torch.arange(8, device=DEV) * 64
    pen = torch.tensor([1.25, 0.5, 0.125], device=DEV)
    res = torch.full_like(flat, 9.0)
    st = torch.empty(7, dtype=torch.uint8, device=DEV)
    q3s.process_logits(flat, row_offsets=torch.from_numpy(offs).to(DEV),
                       row_vocab=torch.tensor(vocabs, dtype=torch.int32, device=DEV), vocab=3072,
                       penalties=pen, history=hist, history_offsets=hoff, out=(res, st))
    un = q3s.STATUS_UNSUPPORTED
    assert st.tolist() == [0, 0, 0, 0, 0, un, un]
    touched = np.zeros(flat.numel(), bool)
    got, h = res.cpu().numpy(), hist.cpu().numpy().reshape(7, 64)
    for r, v in enumerate(vocabs[:5]):
        touched[offs[r]:offs[r] + v] = True
        x = flat.double().cpu().numpy()[None, offs[r]:offs[r] + v]
        value, bound = so.process_logits(x, [[1.25, 0.5, 0.125]], [h[r]])
        so.check(got[None, offs[r]:offs[r] + v], value, bound)
    assert (got[~touched] == 9.0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_in_place(dtype):
    c = Case(8, 33, 3072, dtype, dtype, gap=8)
    want, _ = run(c)
    st = torch.empty(33, dtype=torch.uint8, device=DEV)
    q3s.process_logits(c.logits, **c.args, out=(c.logits, st))
    assert torch.equal(c.logits, want)


def test_a_mask_for_each_row_and_strided_masks():
    V, R = 77, 5
    rng = np.random.default_rng(6)
    allowed = rng.random((R, V)) < 0.5
    words = q3s.pack_mask(torch.from_numpy(allowed).to(DEV))
    wide = torch.full((R, 9), -1, dtype=torch.int32, device=DEV)
    wide[:, :words.shape[1]] = words
    x = torch.randn((R, V), device=DEV)
    out, _ = q3s.process_logits(x, masks=wide)
    want = torch.where(torch.from_numpy(allowed).to(DEV), x, -float("inf"))
    assert torch.equal(out, want)


def test_empty_batches_and_ranges():
    out, st = q3s.process_logits(torch.empty((0, 50), device=DEV))
    assert out.shape == (0, 50) and st.shape == (0,)
    out, st = q3s.process_logits(torch.empty((3, 0), device=DEV))
    assert out.shape == (3, 0) and st.tolist() == [0, 0, 0]
    # A range that ends before it starts holds nothing.
    x = torch.ones((2, 8), device=DEV)
    out, _ = q3s.process_logits(
        x, penalties=torch.tensor([2.0, 1.0, 1.0], device=DEV),
        history=torch.arange(8, dtype=torch.int32, device=DEV),
        history_offsets=torch.tensor([4, 4], device=DEV),
        history_ends=torch.tensor([2, 5], device=DEV))
    assert torch.equal(out[0], x[0]) and out[1].tolist() == [1, 1, 1, 1, -1.5, 1, 1, 1]


def test_offsets_beyond_32_bits():
    """Two rows 2^31 + 16 elements apart."""
    V, far = 5000, 2 ** 31 + 16
    buf = torch.zeros(far + V, dtype=torch.bfloat16, device=DEV)
    rows = buf.as_strided((2, V), (far, 1))
    x = torch.randn((2, V), device=DEV).to(torch.bfloat16)
    rows.copy_(x)
    c = Case(11, 2, V, "bf16", "f32")
    want, _ = q3s.process_logits(x, **c.args)
    got, _ = q3s.process_logits(rows, **c.args)
    assert torch.equal(got, want)


def test_other_stream_and_prepared_call():
    c = Case(12, 64, 2048)
    want, _ = run(c)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got, st = q3s.process_logits(c.logits, **c.args, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(got, want) and (st == 0).all()
    plan = q3s.prepare_process_logits(c.logits, **c.args)
    for _ in range(3):
        plan.out.zero_()
        plan(torch.cuda.current_stream().cuda_stream)
        assert torch.equal(plan.out, want)


def test_captured_in_a_graph():
    c = Case(13, 16, 3072)
    want, _ = run(c)
    plan = q3s.prepare_process_logits(c.logits, **c.args)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        plan(s.cuda_stream)
        s.synchronize()
        with torch.cuda.graph(g, stream=s):
            plan(torch.cuda.current_stream().cuda_stream)
    plan.out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(plan.out, want)


def test_the_repetition_quotient_is_the_division():
    """Every bit of x / repetition, over random bit patterns of both: normal
    values, subnormal ones (whose quotients can be ties), and the largest; the
    few-row and the many-row kernel."""
    rng = np.random.default_rng(14)
    for R in (40, 1400):
        V = 2048
        bits = rng.integers(0, 2 ** 31, (R, V)).astype(np.uint32)
        bits[::4] %= 2 ** 24          # around the smallest normal values
        bits[1::4] |= 0x7E000000      # around the largest
        bits[2::8, ::2] = rng.integers(0, 2 ** 12, (len(bits[2::8]), V // 2))
        x = torch.from_numpy(bits.view(np.float32)).to(DEV)
        rho = rng.uniform(0.25, 4, R).astype(np.float32)
        rho[::5] = rng.choice([3.0, 1.5, 0.75, 1.1, 1.0 + 2.0 ** -23, 2.0, 1e-3, 1e3], len(rho[::5]))
        rho[7::50] = 1e-40
        rho = torch.from_numpy(rho).to(DEV)
        pen = torch.zeros((R, 3), device=DEV)
        pen[:, 0] = rho
        hist = torch.arange(V, device=DEV).to(torch.int16)
        off = torch.zeros(R + 1, dtype=torch.int64, device=DEV)
        out, _ = q3s.process_logits(x, penalties=pen, history=hist, history_offsets=off,
                                    history_ends=off[:R] + V)
        want = x / rho[:, None]
        nan = torch.isnan(want)
        assert torch.equal(torch.isnan(out), nan)
        assert torch.equal(out.view(torch.int32)[~nan], want.view(torch.int32)[~nan])


def test_the_repetition_rule_is_the_samplers():
    """With the repetition penalty alone, sampling the processed row gives
    what the sampler gives with its own penalty."""
    R, V = 64, 2048
    x = torch.randn((R, V), device=DEV) * 2.5
    hist = torch.randint(0, V, (R * 50,), device=DEV).to(torch.int16)
    offs = torch.arange(R + 1, device=DEV) * 50
    seeds = torch.arange(R, device=DEV)
    pen = np.float32(1.3)
    own = q3s.make_params(1, top_k=50, temperature=0.9, repetition_penalty=float(pen))
    want = q3s.sample_batch(x, own, seeds, seeds, history=hist, history_offsets=offs)
    y, _ = q3s.process_logits(x, penalties=torch.tensor([float(pen), 0, 0], device=DEV), history=hist,
                              history_offsets=offs)
    got = q3s.sample_batch(y, q3s.make_params(1, top_k=50, temperature=0.9), seeds, seeds)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"),
                                       ("f32", "bf16")])
@pytest.mark.parametrize("V", [8, 520, 2048, 3072, 4096])
def test_many_rows(V, dtype, out):
    """More rows than the device holds at once, of lengths that travel as one
    copy: histories of no, a few and more ids than a block counts at a time."""
    R = 148 * 33 + 5
    c = Case(V, R, V, dtype, out, hist=300, bias=40 if V == 520 else 3, ids="u16", ends=True,
             masks=5)
    out_, st = run(c)
    rows = np.unique(np.concatenate([np.arange(40), np.arange(R - 40, R),
                                     np.random.default_rng(1).integers(0, R, 60)]))
    # The oracle walks rows in Python: a sample of them, and all against the
    # same rows in small calls.
    sub = dict(c.oracle)
    for k in ("histories", "biases", "allowed"):
        if k in sub:
            sub[k] = [sub[k][r] for r in rows]
    for k in ("penalties", "prompt_lens"):
        if k in sub:
            sub[k] = sub[k][rows]
    value, bound = so.process_logits(c.x[rows], **sub)
    so.check(out_[torch.from_numpy(rows).to(DEV)].double().cpu().numpy(), value,
             so.rounded(bound, value, out == "bf16"))
    assert (st == 0).all()
    for lo in range(0, R, 1000):
        hi = min(R, lo + 1000)
        a = dict(c.args)
        for k in ("penalties", "history_ends", "prompt_lens", "mask_rows"):
            if k in a:
                a[k] = a[k][lo:hi].contiguous()
        for k in ("history_offsets", "bias_offsets"):
            if k in a:
                a[k] = a[k][lo:hi + 1].contiguous()
        small, _ = q3s.process_logits(c.logits[lo:hi], **a)
        assert torch.equal(small.float(), out_[lo:hi].float())


def test_many_rows_with_invalid_ones_and_strides():
    R, V = 2000, 1024
    x = torch.randn((R, V + 8), device=DEV)[:, 4:V + 4]
    pen = torch.tensor([1.2, 0.5, 0.25], device=DEV).repeat(R, 1)
    pen[::7, 0] = -1.0
    hist = torch.randint(0, V, (R, 40), device=DEV).to(torch.int64)
    offs = torch.arange(R + 1, device=DEV) * 40
    res = torch.full((R, V + 12), 5.0, device=DEV)
    st = torch.empty(R, dtype=torch.uint8, device=DEV)
    q3s.process_logits(x, penalties=pen, history=hist, history_offsets=offs, out=(res[:, 8:V + 8], st))
    bad = torch.arange(R, device=DEV) % 7 == 0
    assert torch.equal(st == q3s.STATUS_INVALID_REPETITION_PENALTY, bad)
    assert (res[bad][:, 8:V + 8] == -float("inf")).all()
    assert (res[:, :8] == 5).all() and (res[:, V + 8:] == 5).all()
    good = torch.nonzero(~bad)[:, 0]
    for part in good.split(500):
        want, _ = q3s.process_logits(x[part].contiguous(), penalties=pen[part].contiguous(),
                                     history=hist[part].contiguous(),
                                     history_offsets=torch.arange(len(part) + 1, device=DEV) * 40)
        assert torch.equal(res[part][:, 8:V + 8], want)


def test_bounded_wait_gives_up_and_the_context_stays_usable():
    """The testing hook stops the refills: the rows after each block's first
    ones are never asked for, their waits run out, and the call returns."""
    R, V = 20000, 3072
    x = torch.randn((R, V), device=DEV)
    ctx = q3s.Context(0)
    ctx.set_test_hooks(stage_wait_ns=2_000_000, hold_refill=True)
    out, st = q3s.process_logits(x, ctx=ctx)
    torch.cuda.synchronize()
    late = st == 255
    assert 0 < int(late.sum()) < R and int((st == 0).sum()) == R - int(late.sum())
    assert torch.equal(out[~late], x[~late])
    ctx.set_test_hooks()
    out, st = q3s.process_logits(x, ctx=ctx)
    assert (st == 0).all() and torch.equal(out, x)
    ctx.close()


def test_refusals():
    x = torch.zeros((2, 64), device=DEV)
    i64 = lambda *v: torch.tensor(v, device=DEV)  # noqa: E731
    ids = torch.zeros(4, dtype=torch.int32, device=DEV)
    words = torch.zeros((2, 2), dtype=torch.int32, device=DEV)
    for error, bad in [
        (TypeError, dict(logits=x.double())),
        (TypeError, dict(out_dtype=torch.float16)),
        (ValueError, dict(logits=x.cpu())),
        (ValueError, dict(logits=x[0])),
        (ValueError, dict(logits=x.t())),
        (ValueError, dict(vocab=65)),
        (ValueError, dict(penalties=torch.ones((3, 3), device=DEV))),
        (ValueError, dict(penalties=torch.ones((2, 3)))),
        (ValueError, dict(penalties=torch.ones((2, 3), device=DEV).double())),
        (ValueError, dict(history=ids)),
        (ValueError, dict(history_offsets=i64(0, 0, 0))),
        (TypeError, dict(history=ids.float(), history_offsets=i64(0, 0, 0))),
        (ValueError, dict(history=ids, history_offsets=i64(0, 0))),
        (TypeError, dict(history=ids, history_offsets=i64(0, 0, 0).int())),
        (ValueError, dict(history=ids, history_offsets=i64(0, 0, 0), history_ends=i64(0))),
        (ValueError, dict(bias_ids=ids)),
        (ValueError, dict(bias_ids=ids, bias_values=torch.zeros(3, device=DEV),
                          bias_offsets=i64(0, 0, 4))),
        (TypeError, dict(bias_ids=ids.long(), bias_values=torch.zeros(4, device=DEV),
                         bias_offsets=i64(0, 0, 4))),
        (ValueError, dict(masks=words[:, :1])),
        (ValueError, dict(masks=words[:1])),
        (ValueError, dict(masks=words.long())),
        (ValueError, dict(mask_rows=ids[:2])),
        (ValueError, dict(masks=words, mask_rows=ids)),
        (ValueError, dict(out=(torch.empty((2, 63), device=DEV),
                               torch.empty(2, dtype=torch.uint8, device=DEV)))),
        (ValueError, dict(out=(torch.empty((2, 64), device=DEV),
                               torch.empty(3, dtype=torch.uint8, device=DEV)))),
        (TypeError, dict(out=(torch.empty((2, 64), device=DEV), torch.empty(2, device=DEV)))),
        (ValueError, dict(logits=x.view(-1), row_offsets=i64(0, 64))),
    ]:
        args = dict(bad)
        with pytest.raises(error):
            q3s.process_logits(args.pop("logits", x), **args)


def test_the_c_entry_refuses():
    import ctypes
    ctx = q3s.default_context(0)
    x = torch.zeros((2, 64), device=DEV)
    plan = q3s.prepare_process_logits(x)
    lib = q3s.load()
    ok = bytes(plan._b)

    def call(**fields):
        b = q3s._LogitsBatch.from_buffer_copy(ok)
        for k, v in fields.items():
            setattr(b, k, v)
        return lib.q3s_process_logits(ctx.handle, ctypes.byref(b), None)

    assert call() == q3s.OK
    for fields in [dict(num_rows=-1), dict(vocab=-1), dict(dtype=2), dict(out_dtype=-1),
                   dict(logits=None), dict(out=None), dict(status=None), dict(row_stride=-1),
                   dict(out_stride=63), dict(params_stride=2), dict(history_type=3),
                   dict(history_offsets=x.data_ptr()), dict(bias_offsets=x.data_ptr()),
                   dict(masks=x.data_ptr(), mask_stride=1, num_masks=2),
                   dict(masks=x.data_ptr(), mask_stride=2, num_masks=1),
                   dict(out=x.data_ptr(), out_dtype=q3s.DTYPE_BF16),
                   dict(out=x.data_ptr(), out_stride=65)]:
        assert call(**fields) == q3s.E_INVALID_ARGUMENT, fields
        assert "q3s_process_logits" in q3s.last_error()
    assert lib.q3s_process_logits(None, None, None) == q3s.E_INVALID_ARGUMENT
    torch.cuda.synchronize()


@pytest.mark.parametrize("R", [20, 2000])
def test_ranges_too_long_are_refused(R):
    """A history or a bias list of 2^30 entries or more: UNSUPPORTED, the row
    is left alone, and the rows around it are processed; the few-row and the
    many-row kernel.  Every range starts on real entries; a refused row reads
    none of them."""
    V, n = 1024, 512
    x = torch.randn((R, V), device=DEV)
    hist = torch.randint(0, V, (n,), dtype=torch.int32, device=DEV)
    offs = torch.zeros(R, dtype=torch.int64, device=DEV)
    ends = offs + 40
    ends[3::10] = 2 ** 30 + 8
    ends[4::10] = 2 ** 62
    bias_ids = torch.randint(0, V, (n,), dtype=torch.int32, device=DEV)
    # A row whose list begins where the row before ended and ends far behind it.
    boffs = torch.zeros(R + 1, dtype=torch.int64, device=DEV)
    boffs[6::10] = 2 ** 31  # rows 5, 15, ... are too long; rows 6, 16, ... empty
    pen = torch.tensor([1.3, 0.5, 0.25], device=DEV)
    res = torch.full((R, V), 9.0, device=DEV)
    st = torch.empty(R, dtype=torch.uint8, device=DEV)
    q3s.process_logits(x, penalties=pen, history=hist, history_offsets=offs, history_ends=ends,
                       bias_ids=bias_ids, bias_values=torch.ones(n, device=DEV), bias_offsets=boffs,
                       out=(res, st))
    bad = torch.zeros(R, dtype=torch.bool, device=DEV)
    for k in (3, 4, 5):
        bad[k::10] = True
    assert torch.equal(st == q3s.STATUS_UNSUPPORTED, bad) and (st[~bad] == 0).all()
    assert (res[bad] == 9.0).all()
    good = x[~bad]
    want, _ = q3s.process_logits(good, penalties=pen, history=hist,
                                 history_offsets=offs[:len(good)], history_ends=ends[:1].repeat(len(good)))
    assert torch.equal(res[~bad], want)


def _bias_args(lists):
    """Lists of (ids, values) as the arguments of process_logits."""
    offs = np.concatenate([[0], np.cumsum([len(i) for i, _ in lists])])
    return dict(
        bias_ids=torch.from_numpy(np.concatenate([i for i, _ in lists])).to(torch.int32).to(DEV),
        bias_values=torch.from_numpy(np.concatenate([v for _, v in lists]).astype(np.float32)).to(DEV),
        bias_offsets=torch.from_numpy(offs).to(DEV))


def _list_sums(V, ids, values):
    """(sums, which ids have one): every id's values added in f32, in list order."""
    want, has = np.zeros(V, np.float32), np.zeros(V, bool)
    for i, v in zip(ids, values.astype(np.float32)):
        want[i] = want[i] + v if has[i] else v
        has[i] = True
    return want, has


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("R,V,bias", [(3, 700, 300), (5, 9001, 3000), (1500, 520, 90),
                                      (1300, 3072, 400)])
def test_more_biases_than_a_block_keeps_at_hand(R, V, bias, dtype, out):
    """Lists that overflow a block's own, with histories and masks, in the
    few-row and the many-row kernel; out of place and in place."""
    c = Case(R + V + bias, R, V, dtype, out, hist=60, bias=bias, masks=3)
    got, st = run(c)
    rows = np.unique(np.concatenate([np.arange(min(R, 12)), np.arange(max(0, R - 12), R)]))
    sub = dict(c.oracle)
    for k in ("histories", "biases", "allowed"):
        sub[k] = [sub[k][r] for r in rows]
    for k in ("penalties", "prompt_lens"):
        sub[k] = sub[k][rows]
    value, bound = so.process_logits(c.x[rows], **sub)
    so.check(got[torch.from_numpy(rows).to(DEV)].double().cpu().numpy(), value,
             so.rounded(bound, value, out == "bf16"))
    assert (st == 0).all()
    if dtype == out:  # in place runs in the few-row kernel
        q3s.process_logits(c.logits, **c.args, out=(c.logits, st))
        assert torch.equal(c.logits, got) and (st == 0).all()


@pytest.mark.parametrize("R,V,n", [(1, 100, 150), (2, 3000, 5000), (1200, 64, 200), (1200, 2048, 1000)])
def test_long_bias_lists_add_up_in_list_order(R, V, n):
    """Bit for bit, with values whose f32 sum depends on the order: ids that
    repeat side by side, within 32 entries and far apart."""
    rng = np.random.default_rng(n)
    lists = []
    for r in range(R):
        ids = rng.integers(0, V, n)
        ids[: n // 3] = rng.integers(0, 5, n // 3)
        ids[n // 2: n // 2 + 40] = V - 1
        values = rng.standard_normal(n) * 10.0 ** rng.integers(-4, 5, n)
        lists.append((ids, values.astype(np.float32)))
    x = torch.zeros((R, V), device=DEV)
    out, st = q3s.process_logits(x, **_bias_args(lists))
    out = out.cpu().numpy()
    for r in {0, R // 2, R - 1}:
        np.testing.assert_array_equal(out[r], _list_sums(V, *lists[r])[0])
    assert (st == 0).all()


@pytest.mark.parametrize("R", [2, 1200])
def test_special_values_in_long_bias_lists(R):
    """Infinities that cancel, NaN of any payload and a NaN before a number:
    NaN in those entries, and only there."""
    V, n = 256, 200
    ids = np.arange(n) % 150
    bits = np.float32(1.0).view(np.uint32) + np.zeros(n, np.uint32)
    values = bits.view(np.float32)
    bits[7], bits[9], bits[160] = 0xFFFFFFFF, 0x7FC00001, 0xFFFFFFFF  # id 10 comes at 10 and 160
    values[3], values[153] = np.inf, -np.inf                          # id 3 twice
    values[20] = -np.inf
    x = torch.zeros((R, V), device=DEV)
    out, _ = q3s.process_logits(x, **_bias_args([(ids, values)] * R))
    want = np.zeros(V, np.float32)
    with np.errstate(invalid="ignore"):
        np.add.at(want, ids, values)
    assert np.isnan(want).nonzero()[0].tolist() == [3, 7, 9, 10]
    for r in (0, R - 1):
        np.testing.assert_array_equal(out[r].cpu().numpy(), want)


def test_the_longest_bias_list():
    """2^20 entries are added up; one more is refused, and the row left alone."""
    V, n = 700, 2 ** 20
    ids = torch.randint(0, V, (n + 1,), device=DEV).to(torch.int32)
    one = torch.ones(n + 1, device=DEV)
    x = torch.zeros((2, V), device=DEV)
    res, st = torch.full((2, V), 9.0, device=DEV), torch.empty(2, dtype=torch.uint8, device=DEV)
    q3s.process_logits(x, bias_ids=ids, bias_values=one, out=(res, st),
                       bias_offsets=torch.tensor([0, n, n], device=DEV))
    want = torch.bincount(ids[:n].long(), minlength=V).float()
    assert torch.equal(res[0], want) and torch.equal(res[1], x[1]) and st.tolist() == [0, 0]
    res.fill_(9.0)
    q3s.process_logits(x, bias_ids=ids, bias_values=one, out=(res, st),
                       bias_offsets=torch.tensor([0, n + 1, n + 1], device=DEV))
    assert st.tolist() == [q3s.STATUS_UNSUPPORTED, 0]
    assert (res[0] == 9.0).all() and torch.equal(res[1], x[1])
