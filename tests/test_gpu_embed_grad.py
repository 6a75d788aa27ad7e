"""q3s_embed_grad through the Python binding against the 64-bit restatement
(oracle/step_oracle.py), against differences of the forward pass, and
against itself (equal calls give equal bits).

Bar: for a sum of n values, 2 (n - 1) f32 roundings of the sum of their
magnitudes plus one of the product (and one bf16 rounding for bf16
gradients); codes that do not occur exactly zero.
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


def _grad(rng, R, H, dtype, gap=0, shift=0):
    buf = torch.zeros(R * (H + gap) + shift, dtype=TYPES[dtype], device=DEV)
    g = buf[shift:].view(R, H + gap)[:, :H]
    g.copy_(torch.from_numpy(rng.standard_normal((R, H))).to(DEV))
    return g


def _codes(rng, R, vocabs, skew=1.0):
    return np.stack([(v * rng.random(R) ** skew).astype(np.int64).clip(0, v - 1)
                     for v in vocabs], 1)


def _check(tables, codes, grad, vocabs, scale=1.0, padding_id=None):
    want, _ = so.embed_grad(codes, grad.double().cpu().numpy(), vocabs, scale, padding_id)
    for g, (value, bound) in enumerate(want):
        bf16 = tables[g].dtype == torch.bfloat16
        got = tables[g].double().cpu().numpy()
        so.check(got, value, so.rounded(bound, value, bf16), f"group {g}")
        used = np.zeros(vocabs[g], bool)
        used[codes[:, g][(codes[:, g] >= 0) & (codes[:, g] < vocabs[g])]] = True
        assert (got[~used] == 0).all()


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"),
                                       ("f32", "bf16")])
@pytest.mark.parametrize("H", [1, 5, 64, 130, 1000, 1024])
@pytest.mark.parametrize("R,V", [(1, 1), (1, 2048), (33, 7), (700, 300), (700, 4097)])
def test_one_table(R, V, H, dtype, out):
    rng = np.random.default_rng(R + V + H)
    kind = ["u16", "u32", "i64"][(R + H) % 3]
    codes = _codes(rng, R, [V], 2.0)
    if R > 30:
        codes[3] = V if V < 32768 else -1
    grad = _grad(rng, R, H, dtype)
    ids = torch.from_numpy(codes[:, 0]).to(IDS[kind]).to(DEV)
    got = q3s.embed_grad(ids, grad, V, 0.3, padding_id=2, out_dtype=TYPES[out])
    _check([got], codes, grad, [V], 0.3, 2)


@pytest.mark.parametrize("R", [0, 1, 31, 1025, 3000, 9000])
@pytest.mark.parametrize("vocabs", [[40, 30, 30], [1, 1], [3072] + [2048] * 15, [5000, 3, 4096]])
def test_codebooks(R, vocabs):
    """Vocabularies of one and several sort passes, more rows than one block."""
    rng = np.random.default_rng(R + len(vocabs))
    H = 24
    codes = _codes(rng, R, vocabs, 1.5)
    if R > 30:
        codes[7, -1], codes[8, 0], codes[9, 0] = vocabs[-1], -1, vocabs[0]
    grad = _grad(rng, R, H, "f32")
    dev = torch.from_numpy(codes).to(torch.int32).to(DEV)
    got = q3s.embed_sum_grad(dev, grad, vocabs)
    _check(got, codes, grad, vocabs)


@pytest.mark.parametrize("V", [1, 50, 20000])
@pytest.mark.parametrize("hot", [0.5, 1.0])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_long_runs_of_one_id(V, hot, dtype):
    """Most rows, or all, share one id: its sum is as exact as the others'."""
    rng = np.random.default_rng(V)
    R, H = 6001, 72
    codes = rng.integers(0, V, (R, 1))
    codes[rng.random(R) < hot] = V - 1
    grad = _grad(rng, R, H, dtype)
    got = q3s.embed_grad(torch.from_numpy(codes[:, 0]).to(DEV), grad, V, out_dtype=torch.float32)
    _check([got], codes, grad, [V])


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("gap,shift", [(1, 0), (8, 0), (24, 8), (0, 3), (16, 2)])
def test_strides_and_alignments(gap, shift, dtype, out):
    rng = np.random.default_rng(gap * 10 + shift)
    for H in (72, 512, 1001):
        grad = _grad(rng, 300, H, dtype, gap, shift)
        wide = torch.zeros((300, 7), dtype=torch.int64, device=DEV)
        codes = _codes(rng, 300, [50, 60])
        wide[:, 2:4] = torch.from_numpy(codes).to(DEV)
        bufs = [torch.full((v * H + 5,), 7.0, dtype=TYPES[out], device=DEV) for v in (50, 60)]
        tables = [b[3:3 + v * H].view(v, H) for b, v in zip(bufs, (50, 60))]
        q3s.embed_sum_grad(wide[:, 2:4], grad, [50, 60], scale=2.0, out=tables)
        _check(tables, codes, grad, [50, 60], 2.0)
        for b in bufs:
            assert (b[:3] == 7).all() and (b[-2:] == 7).all()


@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_accumulate(out):
    rng = np.random.default_rng(5)
    R, H, V = 500, 136, 100
    codes = _codes(rng, R, [V], 3.0)
    grad = _grad(rng, R, H, "f32")
    ids = torch.from_numpy(codes[:, 0]).to(DEV)
    before = torch.randn((V, H), device=DEV).to(TYPES[out])
    got = before.clone()
    res = q3s.embed_grad(ids, grad, V, 0.5, out=got, accumulate=True)
    assert res.data_ptr() == got.data_ptr()
    (value, bound), = so.embed_grad(codes, grad.double().cpu().numpy(), [V], 0.5)[0]
    value = value + before.double().cpu().numpy()
    bound = bound + so.U * (np.abs(value) + bound)
    so.check(got.double().cpu().numpy(), value, so.rounded(bound, value, out == "bf16"))


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("R", [1, 40, 2500])
def test_text_gradients(R, dtype, out):
    rng = np.random.default_rng(R)
    H, vocabs = 200, [40, 30]
    codes = _codes(rng, R, vocabs)
    if R > 30:
        codes[[4, 20], [0, 1]] = [40, 30]
    grad = _grad(rng, R, H, dtype)
    dev = torch.from_numpy(codes).to(torch.int32).to(DEV)
    host = grad.double().cpu().numpy()
    _, valid = so.embed_grad(codes, host, vocabs)
    tables, rows = q3s.embed_sum_grad(dev, grad, vocabs, out_dtype=TYPES[out], text="rows")
    _check(tables, codes, grad, vocabs)
    want = np.where(valid[:, None], host, 0.0)
    so.check(rows.double().cpu().numpy(), want,
             so.rounded(np.zeros_like(want), want, out == "bf16"))
    tables, one = q3s.embed_sum_grad(dev, grad, vocabs, out_dtype=TYPES[out], text="broadcast")
    _check(tables, codes, grad, vocabs)
    value = want.sum(0)
    bound = 2 * so.U * max(0, valid.sum() - 1) * np.abs(want).sum(0) + so.U * np.abs(value)
    so.check(one.double().cpu().numpy(), value, so.rounded(bound, value, out == "bf16"))


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"),
                                       ("f32", "bf16")])
@pytest.mark.parametrize("H,gap", [(1, 0), (513, 0), (1024, 0), (1024, 1), (2056, 8)])
def test_text_gradients_of_wide_and_strided_rows(H, gap, dtype, out):
    """Whole vectors and single columns; a row of text_grad may start anywhere."""
    import ctypes
    rng = np.random.default_rng(H + gap)
    R, vocabs = 77, [19, 23, 5]
    codes = _codes(rng, R, vocabs)
    codes[[4, 76], [0, 2]] = [19, 5]
    grad = _grad(rng, R, H, dtype)
    dev = torch.from_numpy(codes).to(torch.int32).to(DEV)
    tables = [torch.empty((v, H), dtype=TYPES[out], device=DEV) for v in vocabs]
    text = torch.full((R, H + gap), 3.0, dtype=TYPES[out], device=DEV)
    ptrs = (ctypes.c_void_p * 3)(*[t.data_ptr() for t in tables])
    sizes = (ctypes.c_int32 * 3)(*vocabs)
    b = q3s._EmbedGradBatch(dtype=int(dtype == "bf16"), grads_dtype=int(out == "bf16"), ids_type=1,
                            groups=3, hidden=H, num_rows=R, codes=dev.data_ptr(), codes_stride=3,
                            grad_out=grad.data_ptr(), grad_stride=H, grads=ctypes.addressof(ptrs),
                            vocab=ctypes.addressof(sizes), padding_id=-1, scale=1.0,
                            text_grad=text.data_ptr(), text_stride=H + gap)
    assert q3s.load().q3s_embed_grad(q3s.default_context(0).handle, ctypes.byref(b), None) == q3s.OK
    torch.cuda.synchronize()
    host = grad.double().cpu().numpy()
    _, valid = so.embed_grad(codes, host, vocabs)
    want = np.where(valid[:, None], host, 0.0)
    so.check(text[:, :H].double().cpu().numpy(), want,
             so.rounded(np.zeros_like(want), want, out == "bf16"))
    assert (text[:, H:] == 3).all()
    _check(tables, codes, grad, vocabs)


def test_equal_calls_give_equal_bits():
    """On two streams, with other work between, and with the rows elsewhere in
    memory."""
    rng = np.random.default_rng(6)
    R, H, vocabs = 20000, 256, [3072, 2048, 2048]
    dev = torch.from_numpy(_codes(rng, R, vocabs, 6.0)).to(DEV)
    grad = _grad(rng, R, H, "bf16")
    want = q3s.embed_sum_grad(dev, grad, vocabs, out_dtype=torch.float32)
    q3s.embed_grad(dev[:100, 0].contiguous(), grad[:100], 3072)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for kw in ({}, {}, {"stream": s.cuda_stream}):
        got = q3s.embed_sum_grad(dev, grad.clone(), vocabs, out_dtype=torch.float32, **kw)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_special_values():
    """Infinities and NaN reach the rows of their id and no other."""
    grad = torch.ones((6, 8), device=DEV)
    grad[1, 0], grad[2, 1], grad[4, 2] = float("inf"), float("nan"), -float("inf")
    grad[5] = float("nan")
    ids = torch.tensor([0, 0, 1, 1, 3, 9], device=DEV)
    got = q3s.embed_grad(ids, grad, 4)
    want = torch.zeros((4, 8), device=DEV)
    want[0], want[1], want[3] = 2, 2, 1
    want[0, 0], want[1, 1], want[3, 2] = float("inf"), float("nan"), -float("inf")
    assert torch.equal(got.nan_to_num(7, 8, 9), want.nan_to_num(7, 8, 9))


def test_broadcast_gradient_rows():
    """The gradient of a sum is one value for every row (stride 0)."""
    ids = torch.tensor([0, 2, 2, 1, 2], device=DEV)
    row = torch.randn(33, device=DEV)
    got = q3s.embed_grad(ids, row.expand(5, 33), 3)
    assert torch.equal(got[0], row) and torch.equal(got[1], row)
    assert torch.equal(got[2], row + row + row)


def test_offsets_beyond_32_bits():
    far = 2 ** 30 + 8
    buf = torch.zeros(2 * far + 64, dtype=torch.bfloat16, device=DEV)
    grad = buf.as_strided((3, 64), (far, 1))
    grad.copy_(torch.randn((3, 64), device=DEV))
    got = q3s.embed_grad(torch.tensor([1, 0, 1], device=DEV), grad, 2, out_dtype=torch.float32)
    assert torch.equal(got[0], grad[1].float())
    assert torch.equal(got[1], grad[0].float() + grad[2].float())


def test_autograd_against_differences():
    """d/dT of sum(w * embedding) by central differences of the forward pass:
    the pass is linear in the table, so the difference quotient is exact up to
    the forward pass's own roundings."""
    rng = np.random.default_rng(7)
    V, H, scale = 11, 9, 1.5
    table = torch.from_numpy(rng.standard_normal((V, H))).float().to(DEV).requires_grad_()
    ids = torch.tensor([[3, 3, 0], [10, 2, 11]], device=DEV)
    w = torch.from_numpy(rng.standard_normal((2, 3, H))).to(DEV)
    (q3s.embedding(ids, table, scale, padding_id=0).double() * w).sum().backward()
    h = 2.0 ** -6

    def f(t):
        return float((q3s.embedding(ids, t, scale, padding_id=0).double() * w).sum())

    for v in range(V):
        for k in range(H):
            e = torch.zeros_like(table)
            e[v, k] = h
            with torch.no_grad():
                d = (f(table + e) - f(table - e)) / (2 * h)
            # roundings of t +- h and of the product, over every use of the id
            uses = float((w[ids == v][:, k].abs()).sum())
            bound = 2 * scale * uses * 2 * so.U * (abs(float(table.detach()[v, k])) + h) / h + 1e-9
            got = float(table.grad[v, k])
            assert abs(got - d) <= bound + 4 * so.U * scale * uses, (v, k, got, d)


def test_codebook_autograd():
    """Tables, a text per row and a broadcast text, against torch's own
    autograd of the same sum in 64 bits."""
    rng = np.random.default_rng(8)
    R, H, vocabs = 50, 16, [20, 10, 10]
    codes = _codes(rng, R, vocabs)
    codes[5, 1] = 10  # an invalid row
    dev = torch.from_numpy(codes).to(torch.int32).to(DEV)
    w = torch.from_numpy(rng.standard_normal((R, H))).to(DEV)
    for shape in ((R, H), (H,), None):
        tables = [torch.from_numpy(rng.standard_normal((v, H))).float().to(DEV).requires_grad_()
                  for v in vocabs]
        text = None if shape is None else torch.randn(shape, device=DEV, requires_grad=True)
        (q3s.codebook_embedding(dev, tables, text).double() * w).sum().backward()
        ok = torch.ones(R, 1, dtype=torch.float64, device=DEV)
        ok[5] = 0
        want = [t.detach().double().requires_grad_() for t in tables]
        wtext = None if text is None else text.detach().double().requires_grad_()
        idx = torch.from_numpy(codes).to(DEV).clamp(max=9)
        idx[:, 0] = torch.from_numpy(codes[:, 0]).to(DEV)
        s = sum(t[idx[:, g]] for g, t in enumerate(want))
        s = s if wtext is None else s + wtext
        (s * ok * w).sum().backward()
        size = float(w.abs().sum(0).max())
        for a, b in zip(tables + ([text] if text is not None else []),
                        want + ([wtext] if wtext is not None else [])):
            assert float((a.grad.double() - b.grad).abs().max()) <= 2 * R * so.U * size


def test_captured_in_a_graph():
    rng = np.random.default_rng(9)
    codes = torch.from_numpy(_codes(rng, 300, [90])[:, 0]).to(DEV)
    grad = _grad(rng, 300, 64, "f32")
    out = torch.empty((90, 64), device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        q3s.embed_grad(codes, grad, 90, out=out)  # the workspace
        s.synchronize()
        with torch.cuda.graph(g, stream=s):
            q3s.embed_grad(codes, grad, 90, out=out)
        # A larger call outgrows the workspace that the graph uses.
        q3s.embed_grad(codes.repeat(100), grad.repeat(100, 1), 90)
    s.synchronize()
    want = out.clone()
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_refusals():
    ids = torch.zeros(3, dtype=torch.int64, device=DEV)
    codes = torch.zeros((3, 2), dtype=torch.int32, device=DEV)
    grad = torch.zeros((3, 8), device=DEV)
    out = torch.zeros((4, 8), device=DEV)
    for error, f in [
        (TypeError, lambda: q3s.embed_grad(ids.float(), grad, 4)),
        (TypeError, lambda: q3s.embed_grad(ids, grad.double(), 4)),
        (TypeError, lambda: q3s.embed_grad(ids, grad, 4, out_dtype=torch.float16)),
        (ValueError, lambda: q3s.embed_grad(ids.cpu(), grad, 4)),
        (ValueError, lambda: q3s.embed_grad(ids, grad.cpu(), 4)),
        (ValueError, lambda: q3s.embed_grad(ids, grad[:2], 4)),
        (ValueError, lambda: q3s.embed_grad(ids, grad, 0)),
        (ValueError, lambda: q3s.embed_grad(ids, grad, 4, accumulate=True)),
        (ValueError, lambda: q3s.embed_grad(ids, grad, 5, out=out)),
        (ValueError, lambda: q3s.embed_grad(ids, grad, 4, out=out.t())),
        (ValueError, lambda: q3s.embed_grad(ids, grad, 4, out=out.cpu())),
        (ValueError, lambda: q3s.embed_grad(codes[:, 0], grad, 4)),
        (ValueError, lambda: q3s.embed_sum_grad(ids, grad, [4])),
        (ValueError, lambda: q3s.embed_sum_grad(codes, grad, [4])),
        (ValueError, lambda: q3s.embed_sum_grad(codes, grad, [4, 0])),
        (ValueError, lambda: q3s.embed_sum_grad(codes, grad, [4, 4], text="row")),
        (ValueError, lambda: q3s.embed_sum_grad(codes, grad, [4, 4], out=[out])),
        (ValueError, lambda: q3s.embed_sum_grad(codes, grad, [4, 4], out=[out, out.bfloat16()])),
        (ValueError, lambda: q3s.embed_sum_grad(codes.t().contiguous().t(), grad, [4, 4])),
        (ValueError, lambda: q3s.embed_sum_grad(codes.repeat(1, 17), grad, [4] * 34)),
        (ValueError, lambda: q3s.embed_grad(ids, torch.zeros((8, 3), device=DEV).t(), 4)),
    ]:
        with pytest.raises(error):
            f()


def test_the_c_entry_refuses():
    import ctypes
    ctx = q3s.default_context(0)
    lib = q3s.load()
    codes = torch.zeros((3, 2), dtype=torch.int32, device=DEV)
    grad = torch.zeros((3, 8), device=DEV)
    out = [torch.zeros((4, 8), device=DEV) for _ in range(2)]
    ptrs = (ctypes.c_void_p * 2)(*[t.data_ptr() for t in out])
    vocab = (ctypes.c_int32 * 2)(4, 4)

    def call(**fields):
        b = q3s._EmbedGradBatch(dtype=0, grads_dtype=0, ids_type=1, groups=2, hidden=8, num_rows=3,
                                codes=codes.data_ptr(), codes_stride=2, grad_out=grad.data_ptr(),
                                grad_stride=8, grads=ctypes.addressof(ptrs),
                                vocab=ctypes.addressof(vocab), padding_id=-1, scale=1.0)
        for k, v in fields.items():
            setattr(b, k, v)
        return lib.q3s_embed_grad(ctx.handle, ctypes.byref(b), None)

    assert call() == q3s.OK
    none = (ctypes.c_void_p * 2)(out[0].data_ptr(), None)
    zero = (ctypes.c_int32 * 2)(4, 0)
    skew = (ctypes.c_void_p * 2)(out[0].data_ptr() + 2, out[1].data_ptr())
    for fields in [dict(num_rows=-1), dict(num_rows=2 ** 31), dict(dtype=2), dict(grads_dtype=3),
                   dict(ids_type=-1), dict(groups=0), dict(groups=33), dict(hidden=0),
                   dict(codes=None), dict(grad_out=None), dict(grads=None), dict(vocab=None),
                   dict(codes_stride=1), dict(grad_stride=7),
                   dict(grads=ctypes.addressof(none)), dict(vocab=ctypes.addressof(zero)),
                   dict(text_grad=grad.data_ptr(), text_stride=7),
                   dict(codes=codes.data_ptr() + 2), dict(grad_out=grad.data_ptr() + 2),
                   dict(text_grad=grad.data_ptr() + 1), dict(grads=ctypes.addressof(skew))]:
        assert call(**fields) == q3s.E_INVALID_ARGUMENT, fields
        assert "q3s_embed_grad" in q3s.last_error()
    assert lib.q3s_embed_grad(None, None, None) == q3s.E_INVALID_ARGUMENT
    torch.cuda.synchronize()


def test_threads_on_one_stream():
    """Calls of several host threads on one stream, through the context they
    share: the launches of a call stay together, so each gets its own sums."""
    import threading
    rng = np.random.default_rng(10)
    jobs = []
    for R, vocabs, H in ((3000, [700, 300, 40], 64), (257, [50, 60], 32), (9000, [900], 16),
                         (1200, [40] * 9, 128)):
        codes = torch.from_numpy(_codes(rng, R, vocabs, 2.0)).to(DEV)
        grad = _grad(rng, R, H, "f32")
        jobs.append((codes, grad, vocabs, q3s.embed_sum_grad(codes, grad, vocabs)))
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    start, wrong = threading.Barrier(len(jobs)), []

    def work(codes, grad, vocabs, want):
        start.wait()
        for _ in range(100):
            with torch.cuda.stream(stream):
                got = q3s.embed_sum_grad(codes, grad, vocabs)
                if not all(torch.equal(a, b) for a, b in zip(got, want)):
                    wrong.append(len(codes))

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_threads_get_one_default_context():
    import threading
    from unittest import mock
    got = []
    with mock.patch.dict(q3s._default_ctx, clear=True):
        threads = [threading.Thread(target=lambda: got.append(q3s.default_context(0)))
                   for _ in range(8)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert len(got) == 8 and all(c is got[0] for c in got)


def _captured(codes, grad, vocabs, stream, ctx=None):
    """(the graph of one call captured on `stream`, its outputs)."""
    out = [torch.empty((v, grad.shape[1]), device=DEV) for v in vocabs]
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=stream):
        q3s.embed_sum_grad(codes, grad, vocabs, out=out, ctx=ctx)
    return g, out


def test_graphs_and_direct_calls_run_side_by_side():
    """Two graphs captured on one stream, replayed on two others while direct
    calls run on the capture stream: each has a workspace of its own."""
    rng = np.random.default_rng(11)
    capture, streams = torch.cuda.Stream(), [torch.cuda.Stream() for _ in range(2)]
    jobs = []
    for R, vocabs, H in ((9000, [900, 30], 64), (1500, [700, 300, 40], 128), (4000, [50, 60], 32)):
        codes = torch.from_numpy(_codes(rng, R, vocabs, 2.0)).to(DEV)
        grad = _grad(rng, R, H, "f32")
        jobs.append((codes, grad, vocabs, q3s.embed_sum_grad(codes, grad, vocabs)))
    graphs = [_captured(*j[:3], capture) for j in jobs[:2]]
    wrong = []
    for _ in range(30):
        for s, (g, out) in zip(streams, graphs):
            with torch.cuda.stream(s):
                for t in out:
                    t.zero_()
                for _ in range(5):
                    g.replay()
        with torch.cuda.stream(capture):
            got = [q3s.embed_sum_grad(*jobs[2][:3]) for _ in range(5)]
        torch.cuda.synchronize()
        for (_, out), job in zip(graphs, jobs):
            wrong += [not torch.equal(a, b) for a, b in zip(out, job[3])]
        for tables in got:
            wrong += [not torch.equal(a, b) for a, b in zip(tables, jobs[2][3])]
    assert not any(wrong)


def test_two_calls_in_one_graph_and_the_first_call_of_a_context():
    """A capture needs no call before it; a larger call in the same capture
    does not take the first one's workspace away."""
    rng = np.random.default_rng(12)
    ctx = q3s.Context(0)
    sizes = [(300, [90, 20], 16), (20000, [500, 300], 64), (300, [90, 20], 16)]
    jobs = []
    for R, vocabs, H in sizes:
        codes = torch.from_numpy(_codes(rng, R, vocabs)).to(DEV)
        jobs.append((codes, _grad(rng, R, H, "f32"), vocabs))
    outs = [[torch.empty((v, j[1].shape[1]), device=DEV) for v in j[2]] for j in jobs]
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        for j, out in zip(jobs, outs):
            q3s.embed_sum_grad(*j, out=out, ctx=ctx)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    for j, out in zip(jobs, outs):
        for a, b in zip(out, q3s.embed_sum_grad(*j)):
            assert torch.equal(a, b)
    del g
    torch.cuda.synchronize()
    ctx.close()


def test_workspaces_of_destroyed_graphs_are_used_again():
    import gc
    import time
    rng = np.random.default_rng(13)
    ctx = q3s.Context(0)
    vocabs = [3000, 2000]
    codes = torch.from_numpy(_codes(rng, 60000, vocabs)).to(torch.int32).to(DEV)
    grad = _grad(rng, 60000, 512, "f32")
    want = q3s.embed_sum_grad(codes, grad, vocabs)
    stream, free = torch.cuda.Stream(), []
    for _ in range(6):
        g, out = _captured(codes, grad, vocabs, stream, ctx)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        free.append(torch.cuda.mem_get_info(DEV)[0])
        del g, out
        gc.collect()
        torch.cuda.synchronize()
        time.sleep(0.1)  # what a graph holds may be let go on a thread of CUDA's
    # One workspace is tens of MB; six graphs one after another have one between them.
    assert free[1] - free[-1] < 8 << 20
    ctx.close()


def test_a_workspace_that_cannot_be_had_leaves_no_error_behind():
    """32 codebooks of 2^31 - 1 ids need a workspace of some 550 GB: refused
    before any launch, and the next call works."""
    import ctypes
    lib, ctx = q3s.load(), q3s.Context(0)
    codes = torch.zeros((3, 32), dtype=torch.int32, device=DEV)
    grad = torch.ones((3, 1), device=DEV)
    # Addresses of tables that do not exist: nothing is launched.
    ptrs = (ctypes.c_void_p * 32)(*[(1 << 44) + (k << 34) for k in range(32)])
    sizes = (ctypes.c_int32 * 32)(*[2 ** 31 - 1] * 32)
    b = q3s._EmbedGradBatch(dtype=0, grads_dtype=0, ids_type=1, groups=32, hidden=1, num_rows=3,
                            codes=codes.data_ptr(), codes_stride=32, grad_out=grad.data_ptr(),
                            grad_stride=1, grads=ctypes.addressof(ptrs),
                            vocab=ctypes.addressof(sizes), padding_id=-1, scale=1.0)
    torch.cuda.synchronize()
    for _ in range(2):
        assert lib.q3s_embed_grad(ctx.handle, ctypes.byref(b), None) == q3s.E_OUT_OF_MEMORY
        assert "cudaMalloc" in q3s.last_error()
        got = q3s.embed_grad(codes[:, 0].contiguous(), grad, 2, ctx=ctx)
        assert got.tolist() == [[3.0], [0.0]]
        out, st = q3s.embed_lookup(codes[:, 0].contiguous(), grad, ctx=ctx)
        assert out.tolist() == [[1.0]] * 3 and st.tolist() == [0, 0, 0]
    ctx.close()


def test_gradients_that_overlap_are_refused():
    """Two groups that write one table, wholly or in part, or the text's
    gradient inside a table; tables that touch are fine, in any order."""
    import ctypes
    lib, ctx = q3s.load(), q3s.default_context(0)
    R, H, sizes = 5, 8, (4, 6, 5)
    codes = torch.randint(0, 4, (R, 3), dtype=torch.int32, device=DEV)
    grad = torch.randn((R, H), device=DEV)
    want = q3s.embed_sum_grad(codes, grad, sizes)
    flat = torch.zeros((60, H), device=DEV)
    vocab = (ctypes.c_int32 * 3)(*sizes)

    def call(rows, accumulate=0, **fields):
        flat.zero_()
        ptrs = (ctypes.c_void_p * 3)(*[flat[r].data_ptr() for r in rows])
        b = q3s._EmbedGradBatch(dtype=0, grads_dtype=0, ids_type=1, groups=3, hidden=H, num_rows=R,
                                accumulate=accumulate, codes=codes.data_ptr(), codes_stride=3,
                                grad_out=grad.data_ptr(), grad_stride=H,
                                grads=ctypes.addressof(ptrs), vocab=ctypes.addressof(vocab),
                                padding_id=-1, scale=1.0, **fields)
        return lib.q3s_embed_grad(ctx.handle, ctypes.byref(b), None)

    for rows in ((0, 4, 10), (11, 5, 0), (20, 0, 6)):
        assert call(rows) == q3s.OK
        for r, t in zip(rows, want):
            assert torch.equal(flat[r:r + len(t)], t)
    text = dict(text_grad=flat[40].data_ptr(), text_stride=H)
    assert call((0, 4, 10), **text) == q3s.OK and call((35, 45, 30), **text) == q3s.OK
    for rows in ((0, 0, 10), (0, 3, 10), (10, 4, 0), (9, 0, 5), (0, 20, 4 + 20)):
        for accumulate in (0, 1):
            assert call(rows, accumulate) == q3s.E_INVALID_ARGUMENT, rows
            assert "overlap" in q3s.last_error()
    for rows in ((0, 35, 10), (44, 4, 10)):  # rows 40..44 are the text's
        assert call(rows, **text) == q3s.E_INVALID_ARGUMENT, rows
    assert call((0, 38, 10), text_grad=flat[40].data_ptr(), text_stride=0) == q3s.E_INVALID_ARGUMENT
    torch.cuda.synchronize()
    one = torch.zeros((4, H), device=DEV)
    with pytest.raises(ValueError, match="table of its own"):
        q3s.embed_sum_grad(codes[:, :2], grad, [4, 4], out=[one, one], accumulate=True)


def test_the_largest_table():
    """2^31 - 1 ids: the counts of buckets and blocks pass 31 bits."""
    V = 2 ** 31 - 1
    ids = torch.tensor([0, V - 1, 5, V - 1, 2 ** 30, V - 1025, V - 1024, 5], device=DEV)
    grad = torch.arange(1, 9, device=DEV, dtype=torch.float32)[:, None].bfloat16()
    ctx = q3s.Context(0)  # its workspace holds a range for each id: 17 GB
    got = q3s.embed_grad(ids.to(torch.int32), grad, V, ctx=ctx)[:, 0]
    want = {0: 1, V - 1: 6, 5: 11, 2 ** 30: 5, V - 1025: 6, V - 1024: 7}
    assert {k: float(got[k]) for k in want} == want
    assert sum(int(torch.count_nonzero(p)) for p in got.split(1 << 28)) == len(want)
    ctx.close()
    del got
    torch.cuda.empty_cache()


def test_the_longest_rows():
    """hidden beyond 2^30 is refused (num_rows 0: nothing would be read)."""
    import ctypes
    out = torch.zeros((1, 8), device=DEV)
    ptrs, sizes = (ctypes.c_void_p * 1)(out.data_ptr()), (ctypes.c_int32 * 1)(1)
    b = q3s._EmbedGradBatch(dtype=0, grads_dtype=0, ids_type=1, groups=1, hidden=2 ** 30 + 1,
                            num_rows=0, accumulate=1, grads=ctypes.addressof(ptrs),
                            vocab=ctypes.addressof(sizes), padding_id=-1, scale=1.0)
    lib, ctx = q3s.load(), q3s.default_context(0)
    assert lib.q3s_embed_grad(ctx.handle, ctypes.byref(b), None) == q3s.E_INVALID_ARGUMENT
    assert "hidden" in q3s.last_error()


def _loss_with_its_own_gradient(rows, tensors):
    """sum rows^3, plus the squares of its own gradient, plus the cubes of that
    gradient's: derivatives up to the third.  Small whole numbers, so every
    product and sum is exact in f32."""
    loss = (rows ** 3).sum()
    first = torch.autograd.grad(loss, tensors, create_graph=True)
    assert all(g.requires_grad for g in first)
    second = torch.autograd.grad(sum((g ** 2).sum() for g in first), tensors, create_graph=True)
    return loss + sum((g * w).sum() for g, w in zip(second, tensors))


def test_second_and_third_derivatives_of_the_lookup():
    """Against torch's own embedding in 64 bits; a padding id and an id that
    the table does not have."""
    rng = np.random.default_rng(14)
    V, H, pad = 6, 5, 2
    ids = torch.tensor([[0, 1, 1], [2, 5, 6]], device=DEV)
    table = torch.from_numpy(rng.integers(-1, 2, (V, H))).float().to(DEV).requires_grad_()
    x = q3s.embedding(ids, table, 2.0, padding_id=pad)
    _loss_with_its_own_gradient(x, [table]).backward()
    want = table.detach().double().requires_grad_()
    live = ((ids != pad) & (ids < V)).double()[..., None]
    y = torch.nn.functional.embedding(ids.clamp(max=V - 1), want) * 2.0 * live
    _loss_with_its_own_gradient(y, [want]).backward()
    assert torch.equal(table.grad.double(), want.grad)
    assert float(want.grad.abs().max()) < 2 ** 24


@pytest.mark.parametrize("shape", [None, (12, 4), (4,)])
def test_second_and_third_derivatives_of_the_codebook_sum(shape):
    """With no text, one per row and one for all; a row with a code that its
    codebook does not have."""
    rng = np.random.default_rng(15)
    vocabs, R, H = [3, 5], 12, 4
    codes = _codes(rng, R, vocabs)
    codes[7, 1] = 5
    dev = torch.from_numpy(codes).to(torch.int32).to(DEV)
    tensors = [torch.from_numpy(rng.integers(-1, 2, (v, H))).float().to(DEV).requires_grad_()
               for v in vocabs]
    if shape is not None:
        tensors.append(torch.from_numpy(rng.integers(-1, 2, shape)).float().to(DEV).requires_grad_())
    x = q3s.codebook_embedding(dev, tensors[:2], tensors[2] if shape else None)
    _loss_with_its_own_gradient(x, tensors).backward()
    want = [t.detach().double().requires_grad_() for t in tensors]
    live = torch.ones((R, 1), dtype=torch.float64, device=DEV)
    live[7] = 0
    y = sum(want[g][torch.from_numpy(codes[:, g].clip(0, v - 1)).to(DEV)] for g, v in enumerate(vocabs))
    y = (y + want[2] if shape else y) * live
    _loss_with_its_own_gradient(y, want).backward()
    for a, b in zip(tensors, want):
        assert float(b.grad.abs().max()) < 2 ** 24
        assert torch.equal(a.grad.double(), b.grad)


def test_a_penalty_on_the_gradient_reaches_only_what_trains():
    """One frozen table and a text that does not train, with create_graph."""
    codes = torch.tensor([[0, 1], [1, 1]], dtype=torch.int32, device=DEV)
    a = torch.ones((2, 3), device=DEV, requires_grad=True)
    b, text = torch.ones((2, 3), device=DEV), torch.ones(3, device=DEV)
    x = q3s.codebook_embedding(codes, [a, b], text)
    (g,) = torch.autograd.grad((x ** 2).sum(), [a], create_graph=True)
    (g ** 2).sum().backward()
    # g = 2 (a + b + text) a row, its square's derivative 2 g 2
    assert torch.equal(a.grad, torch.full((2, 3), 24.0, device=DEV)) and b.grad is None


def test_vocabularies_beyond_31_bits_are_refused():
    """2^32 + 5 must not pass for 5."""
    ids = torch.zeros(3, dtype=torch.int64, device=DEV)
    grad = torch.zeros((3, 1), device=DEV)
    codes = torch.zeros((3, 2), dtype=torch.int32, device=DEV)
    for vocab in (2 ** 31, 2 ** 32 + 5):
        with pytest.raises(ValueError, match="vocabulary"):
            q3s.embed_grad(ids, grad, vocab)
        with pytest.raises(ValueError, match="vocabulary"):
            q3s.embed_sum_grad(codes, grad, [4, vocab])


def _check_large(tables, codes, grad, vocabs):
    """_check for many rows: the same sums and the same bound, on the device."""
    dev = torch.from_numpy(codes).to(DEV)
    g64 = grad.double()
    for g, v in enumerate(vocabs):
        value, size = (torch.zeros((v, grad.shape[1]), dtype=torch.float64, device=DEV).index_add_(
            0, dev[:, g], x) for x in (g64, g64.abs()))
        count = torch.bincount(dev[:, g], minlength=v).double()
        bound = 1.01 * (2 * so.U * (count - 1).clamp(min=0)[:, None] * size + so.U * value.abs())
        bf16 = tables[g].dtype == torch.bfloat16
        so.check(tables[g].double().cpu().numpy(), value.cpu().numpy(),
                 so.rounded(bound.cpu().numpy(), value.cpu().numpy(), bf16), f"group {g}")
        assert (tables[g][count == 0] == 0).all()


@pytest.mark.parametrize("R,vocabs,hot", [
    (70000, [100003], 0.5),       # one block a bucket; warps that find more keys than they keep
    (70000, [100003], 0.0),
    (140000, [500], 0.97),        # clusters of eight, the same
    (140000, [500, 40], 0.97),    # several groups
    (140000, [500, 40], 0.0),
    (33000, [2000], 0.3),         # clusters of eight, lists that suffice
    (2000, [152000], 0.1),        # more buckets than multiprocessors
])
def test_sorts_of_many_rows(R, vocabs, hot):
    """Each way the sort goes with many rows, and pieces of more than 32
    rows (above 65536)."""
    rng = np.random.default_rng(R + len(vocabs))
    codes = _codes(rng, R, vocabs, 2.0)
    codes[rng.random(R) < hot] = np.array(vocabs) - 1
    grad = _grad(rng, R, 4, "f32")
    dev = torch.from_numpy(codes).to(torch.int32).to(DEV)
    got = [q3s.embed_grad(dev[:, 0].contiguous(), grad, vocabs[0])] if len(vocabs) == 1 else \
        q3s.embed_sum_grad(dev, grad, vocabs)
    _check_large(got, codes, grad, vocabs)


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("H", [256, 512, 1024, 1280])
def test_long_runs_of_wide_bf16_rows(H, out):
    """A code with most of 6001 rows: pieces joined in two steps, in tiles of
    one, two and four 16-byte vectors a lane."""
    rng = np.random.default_rng(H)
    R, vocabs = 6001, [300, 50]
    codes = _codes(rng, R, vocabs)
    codes[rng.random(R) < 0.8] = [299, 17]
    grad = _grad(rng, R, H, "bf16")
    dev = torch.from_numpy(codes).to(torch.int32).to(DEV)
    got = q3s.embed_sum_grad(dev, grad, vocabs, out_dtype=TYPES[out])
    _check_large(got, codes, grad, vocabs)
    one = q3s.embed_grad(dev[:, 0].contiguous(), grad, 300, out_dtype=TYPES[out])
    assert torch.equal(one, got[0])


def test_calls_that_would_take_minutes_are_refused():
    """The sort's time goes by rows times ids: beyond 2^48 the call is refused
    on the host.  (32 tables of 2^31 - 1 ids: their workspace could not be had
    either, so nothing is launched in any case.)"""
    import ctypes
    lib, ctx = q3s.load(), q3s.Context(0)
    codes = torch.zeros((3, 32), dtype=torch.int32, device=DEV)
    grad = torch.ones((3, 1), device=DEV)
    ptrs = (ctypes.c_void_p * 32)(*[(1 << 44) + (k << 34) for k in range(32)])
    sizes = (ctypes.c_int32 * 32)(*[2 ** 31 - 1] * 32)
    b = q3s._EmbedGradBatch(dtype=0, grads_dtype=0, ids_type=1, groups=32, hidden=1,
                            num_rows=2 ** 31 - 1, codes=codes.data_ptr(), codes_stride=32,
                            grad_out=grad.data_ptr(), grad_stride=1,
                            grads=ctypes.addressof(ptrs), vocab=ctypes.addressof(sizes),
                            padding_id=-1, scale=1.0)
    for rows, want in ((2 ** 31 - 1, q3s.E_INVALID_ARGUMENT), (4097, q3s.E_INVALID_ARGUMENT),
                       (4096, q3s.E_OUT_OF_MEMORY)):
        b.num_rows = rows
        assert lib.q3s_embed_grad(ctx.handle, ctypes.byref(b), None) == want, rows
        assert ("2^48" in q3s.last_error()) == (want == q3s.E_INVALID_ARGUMENT)
    ctx.close()
