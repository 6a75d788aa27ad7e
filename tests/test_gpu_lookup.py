"""q3s_embed_lookup through the Python binding against the 64-bit restatement
(oracle/step_oracle.py).

Bar: one f32 rounding of the product (and one bf16 rounding for bf16
outputs), statuses exact, padding and invalid rows exactly zero.
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


def _table(rng, V, H, dtype, gap=0, shift=0):
    buf = torch.zeros(V * (H + gap) + shift, dtype=TYPES[dtype], device=DEV)
    t = buf[shift:].view(V, H + gap)[:, :H]
    t.copy_(torch.from_numpy(rng.standard_normal((V, H))).to(DEV))
    return t


def _check(out, status, ids, table, scale, padding_id, V=None):
    value, bound, st = so.embed_lookup(ids, table.double().cpu().numpy(), scale, padding_id)
    bf16 = out.dtype == torch.bfloat16
    so.check(out.double().cpu().numpy().reshape(value.shape), value,
             so.rounded(bound, value, bf16))
    np.testing.assert_array_equal(status.cpu().numpy().reshape(-1), st)


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"),
                                       ("f32", "bf16")])
@pytest.mark.parametrize("H", [1, 2, 7, 64, 1000, 1024, 1003, 2048, 5000])
@pytest.mark.parametrize("N", [1, 3, 600])
def test_matches_the_definition(N, H, dtype, out):
    rng = np.random.default_rng(N * H)
    V = 97
    kind = ["u16", "u32", "i64"][(N + H) % 3]
    t = _table(rng, V, H, dtype)
    ids = rng.integers(0, V, N)
    ids[rng.random(N) < 0.1] = 5
    if N > 3:
        ids[1], ids[2] = V, 32767 if kind == "u16" else 2 ** 31 - 1
    dev = torch.from_numpy(ids).to(IDS[kind]).to(DEV)
    got, st = q3s.embed_lookup(dev, t, 0.37, padding_id=5, out_dtype=TYPES[out])
    _check(got, st, ids, t, 0.37, 5)


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("gap,shift", [(1, 0), (8, 0), (24, 8), (0, 3), (16, 2)])
def test_strides_and_alignments(gap, shift, dtype, out):
    rng = np.random.default_rng(gap * 10 + shift)
    for H in (72, 512, 1001):
        t = _table(rng, 50, H, dtype, gap, shift)
        ids = rng.integers(0, 50, 130)
        buf = torch.full((130 * H + 5,), 7.0, dtype=TYPES[out], device=DEV)
        res = buf[3:3 + 130 * H].view(130, H)
        st = torch.empty(130, dtype=torch.uint8, device=DEV)
        q3s.embed_lookup(torch.from_numpy(ids).to(DEV), t, 2.5, out=(res, st))
        _check(res, st, ids, t, 2.5, None)
        assert (buf[:3] == 7).all() and (buf[-2:] == 7).all()


def test_shapes_of_ids_and_negative_ids():
    rng = np.random.default_rng(1)
    t = _table(rng, 20, 40, "f32")
    ids = torch.tensor([[0, -1, 19], [20, -2 ** 31, 7]], dtype=torch.int32, device=DEV)
    out, st = q3s.embed_lookup(ids, t, 3.0)
    assert out.shape == (2, 3, 40) and st.tolist() == [[0, 8, 0], [8, 8, 0]]
    _check(out, st, ids.cpu().numpy().reshape(-1), t, 3.0, None)
    out, st = q3s.embed_lookup(ids.long(), t, 3.0, padding_id=7)
    _check(out, st, ids.cpu().numpy().reshape(-1), t, 3.0, 7)
    out, st = q3s.embed_lookup(ids[0, 0], t)
    assert out.shape == (40,) and st.shape == () and torch.equal(out, t[0])


def test_empty():
    t = torch.ones((3, 8), device=DEV)
    out, st = q3s.embed_lookup(torch.empty((2, 0), dtype=torch.int64, device=DEV), t)
    assert out.shape == (2, 0, 8) and st.shape == (2, 0)


def test_special_values_pass_through():
    """Infinities, NaN and the lowest value; padding's own row is not read."""
    lowest = torch.finfo(torch.float32).min
    t = torch.tensor([[float("nan")] * 8, [float("inf"), -float("inf"), lowest, 0.0, -0.0, 1e-45,
                                           float("nan"), 1.0]], device=DEV)
    out, _ = q3s.embed_lookup(torch.tensor([0, 1], device=DEV), t, 1.0, padding_id=0)
    assert (out[0] == 0).all()
    nan = torch.isnan(t[1])  # a product's NaN has no payload of its own
    assert torch.equal(torch.isnan(out[1]), nan)
    assert torch.equal(out[1].view(torch.int32)[~nan], t[1].view(torch.int32)[~nan])


def test_many_ids():
    rng = np.random.default_rng(2)
    t = _table(rng, 300, 48, "bf16")
    ids = rng.integers(0, 300, 200_003)
    out, st = q3s.embed_lookup(torch.from_numpy(ids).to(DEV), t, 1.5, out_dtype=torch.float32)
    want = t.float()[torch.from_numpy(ids).to(DEV)] * 1.5
    assert torch.equal(out, want) and (st == 0).all()


def test_table_offsets_beyond_32_bits():
    """A table of 2^31 + elements: rows far apart."""
    far = 2 ** 30 + 8
    buf = torch.zeros(2 * far + 64, dtype=torch.bfloat16, device=DEV)
    t = buf.as_strided((3, 64), (far, 1))
    t.copy_(torch.randn((3, 64), device=DEV))
    out, _ = q3s.embed_lookup(torch.tensor([2, 0, 1, 2], device=DEV), t, 2.0)
    assert torch.equal(out, t[[2, 0, 1, 2]] * 2)


def test_other_stream_prepared_call_and_graph():
    rng = np.random.default_rng(3)
    t = _table(rng, 100, 256, "bf16")
    ids = torch.from_numpy(rng.integers(0, 100, 40)).to(torch.int32).to(DEV)
    want, _ = q3s.embed_lookup(ids, t, 16.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got, _ = q3s.embed_lookup(ids, t, 16.0, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(got, want)
    plan = q3s.prepare_embed_lookup(ids, t, scale=16.0)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        plan(s.cuda_stream)
        s.synchronize()
        with torch.cuda.graph(g, stream=s):
            plan(torch.cuda.current_stream().cuda_stream)
    ids.copy_(ids.flip(0))  # the plan reads the buffer as it is at the launch
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(plan.out, want.flip(0))


def test_agrees_with_the_codebook_sum():
    """One codebook without text is a lookup with scale 1."""
    rng = np.random.default_rng(4)
    t = _table(rng, 3072, 1024, "bf16")
    codes = torch.from_numpy(rng.integers(0, 3073, (500, 1))).to(torch.int32).to(DEV)
    a, sa = q3s.embed_sum(codes, [t])
    b, sb = q3s.embed_lookup(codes[:, 0].contiguous(), t)
    assert torch.equal(a, b) and torch.equal(sa, sb)


def test_refusals():
    t = torch.zeros((4, 8), device=DEV)
    ids = torch.zeros(3, dtype=torch.int64, device=DEV)
    st = torch.empty(3, dtype=torch.uint8, device=DEV)
    for error, bad in [
        (TypeError, dict(ids=ids.float())),
        (TypeError, dict(table=t.double())),
        (TypeError, dict(out_dtype=torch.float16)),
        (ValueError, dict(ids=ids.cpu())),
        (ValueError, dict(table=t.cpu())),
        (ValueError, dict(table=t.t())),
        (ValueError, dict(table=t[0])),
        (ValueError, dict(table=t[:0])),
        (ValueError, dict(ids=torch.zeros((3, 2), dtype=torch.int64, device=DEV)[:, 0])),
        (ValueError, dict(out=(torch.empty((3, 9), device=DEV), st))),
        (ValueError, dict(out=(torch.empty((3, 8)), st))),
        (ValueError, dict(out=(torch.empty((3, 8), device=DEV), st[:2]))),
        (ValueError, dict(out=(torch.empty((3, 8), device=DEV), st.int()))),
    ]:
        args = dict(bad)
        with pytest.raises(error):
            q3s.embed_lookup(args.pop("ids", ids), args.pop("table", t), **args)


def test_the_c_entry_refuses():
    import ctypes
    ctx = q3s.default_context(0)
    plan = q3s.prepare_embed_lookup(torch.zeros(3, dtype=torch.int64, device=DEV),
                                    torch.zeros((4, 8), device=DEV))
    lib = q3s.load()
    ok = bytes(plan._b)

    def call(**fields):
        b = q3s._LookupBatch.from_buffer_copy(ok)
        for k, v in fields.items():
            setattr(b, k, v)
        return lib.q3s_embed_lookup(ctx.handle, ctypes.byref(b), None)

    assert call() == q3s.OK
    for fields in [dict(num_ids=-1), dict(hidden=0), dict(vocab=0), dict(dtype=2),
                   dict(out_dtype=5), dict(ids_type=3), dict(ids=None), dict(table=None),
                   dict(ids=plan._b.ids + 4),
                   dict(out=None), dict(status=None), dict(table_stride=7), dict(out_stride=7)]:
        assert call(**fields) == q3s.E_INVALID_ARGUMENT, fields
        assert "q3s_embed_lookup" in q3s.last_error()
    assert lib.q3s_embed_lookup(None, None, None) == q3s.E_INVALID_ARGUMENT
    torch.cuda.synchronize()


@pytest.mark.parametrize("H", [2 ** 29 + 8, 2 ** 29 + 9])
def test_rows_longer_than_2_gib(H):
    """Offsets inside one row pass 31 bits: f32 rows of 2 GiB and a little,
    in vectors and in single elements."""
    table = torch.empty((2, H), device=DEV)
    table[:, :1024], table[:, 1024:-1024], table[:, -1024:] = 1.0, 2.0, 3.0
    table[1, -1] = 5.0
    out, st = q3s.embed_lookup(torch.tensor([1, 0], device=DEV), table, 0.5)
    assert st.tolist() == [0, 0]
    for k in (0, 1):
        for part in (slice(0, 1024), slice(1024, H - 1024), slice(H - 1024, H)):
            a, b = out[k, part], table[1 - k, part]
            for lo in range(0, len(a), 1 << 27):
                assert torch.equal(a[lo:lo + (1 << 27)], b[lo:lo + (1 << 27)] * 0.5)
    del table, out
    torch.cuda.empty_cache()


def test_the_longest_rows():
    ids = torch.zeros(1, dtype=torch.int64, device=DEV)
    x = torch.zeros((1, 8), device=DEV)
    st = torch.zeros(1, dtype=torch.uint8, device=DEV)
    b = q3s._LookupBatch(dtype=0, out_dtype=0, ids_type=2, hidden=2 ** 30 + 1, vocab=1, num_ids=0,
                         ids=ids.data_ptr(), table=x.data_ptr(), table_stride=2 ** 31,
                         out=x.data_ptr(), out_stride=2 ** 31, scale=1.0, status=st.data_ptr())
    import ctypes
    call = lambda: q3s.load().q3s_embed_lookup(q3s.default_context(0).handle,  # noqa: E731
                                               ctypes.byref(b), None)
    assert call() == q3s.E_INVALID_ARGUMENT and "hidden" in q3s.last_error()
    b.hidden = 2 ** 30
    assert call() == q3s.OK  # no ids: nothing is launched
