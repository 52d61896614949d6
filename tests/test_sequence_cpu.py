"""CPU-side checks of the sequence operators: what the Python wrappers and the C entry points refuse, without a
launch; shapes of the fake kernels."""
import ctypes as C

import pytest
import torch


@pytest.fixture
def ops(monkeypatch):
    """hv_amd.ops without its device check: every refusal below comes before a launch."""
    from hv_amd import ops
    monkeypatch.setattr(ops, "_cuda", lambda *t: None)
    return ops


def attn(ops, **kw):
    a = dict(q=torch.zeros(6, 4, 32), k=torch.zeros(6, 2, 32), v=torch.zeros(6, 2, 32),
             cu_q=torch.tensor([0, 6], dtype=torch.int32), cu_k=torch.tensor([0, 6], dtype=torch.int32))
    extra = {n: kw.pop(n) for n in ("causal", "scale") if n in kw}
    a.update(kw)
    return ops.attn_packed_args(*a.values(), extra.get("causal", False), extra.get("scale"))


def test_packed_attention_arguments(ops):
    d = attn(ops, causal=True)
    assert (d.hq, d.hkv, d.d, d.nseq, d.causal, d.total_q) == (4, 2, 32, 1, 1, 6)
    assert abs(d.scale - 32 ** -0.5) < 1e-7
    z = torch.zeros
    bad = [dict(k=z(6, 3, 32), v=z(6, 3, 32)), dict(k=z(6, 2, 64)), dict(q=z(6, 128)), dict(k=z(6, 0, 32), v=z(6, 0, 32)),
           dict(q=z(6, 4, 12), k=z(6, 2, 12), v=z(6, 2, 12)), dict(q=z(6, 4, 136), k=z(6, 2, 136), v=z(6, 2, 136)),
           dict(k=z(6, 2, 32, dtype=torch.bfloat16)), dict(cu_q=torch.tensor([0, 6])),
           dict(cu_k=torch.tensor([0, 3, 6], dtype=torch.int32)), dict(cu_q=z(0, dtype=torch.int32), cu_k=z(0, dtype=torch.int32)),
           dict(q=z(6, 4, 33)[:, :, 1:]), dict(q=z(6, 4, 64)[:, :, ::2]), dict(scale=0.0), dict(scale=-1.0),
           dict(scale=float("nan")), dict(scale=float("inf"))]
    for kw in bad:
        with pytest.raises(ValueError):
            attn(ops, **kw)
    with pytest.raises(TypeError):
        attn(ops, q=z(6, 4, 32).double(), k=z(6, 2, 32).double(), v=z(6, 2, 32).double())


def test_norm_and_linear_arguments(ops):
    z, w = torch.zeros(4, 32), torch.ones(32)
    for args in ((z, torch.zeros(4, 16), w), (z, torch.zeros(32), w), (z, z, torch.ones(16)), (z.t(), z.t(), torch.ones(4)),
                 (torch.zeros(2, 0), torch.zeros(2, 0), torch.ones(0)), (torch.zeros(1, 32776), torch.zeros(1, 32776), torch.ones(32776))):
        with pytest.raises(ValueError):
            ops.add_rmsnorm(*args)
        with pytest.raises(ValueError):
            ops.add_rmsnorm_fp8(*args)
    with pytest.raises(TypeError):
        ops.add_rmsnorm(z, z, w.bfloat16())
    with pytest.raises(ValueError):
        ops.quantize_rows_fp8(torch.zeros(4))
    with pytest.raises(ValueError):
        ops.quantize_rows_fp8(torch.zeros(4, 8).t())
    f8 = torch.float8_e4m3fn
    a, b, s4, s3 = torch.zeros(4, 32).to(f8), torch.zeros(3, 32).to(f8), torch.ones(4), torch.ones(3)
    for args, kw in (((z, s4, b, s3), {}), ((a, s3, b, s3), {}), ((a, s4, b, s4), {}), ((a, s4, b, s3), dict(bias=s4)),
                     ((a, s4, b, s3), dict(act="tanh")), ((a[:, :24], s4, b[:, :24], s3), {}),
                     ((torch.zeros(4, 48).to(f8)[:, 8:40], s4, b, s3), {}), ((a, s4.double(), b, s3), {}),
                     ((torch.zeros(4, 16).to(f8), s4, b, s3), {})):
        with pytest.raises(ValueError):
            ops.linear_fp8(*args, **kw)
    with pytest.raises(TypeError):
        ops.linear_fp8(a, s4, b, s3, out_dtype=torch.float16)


def test_product_path_refuses_cpu_tensors():
    from hv_amd import ops
    z = torch.zeros(4, 4, 32)
    with pytest.raises(RuntimeError):
        ops.attention_packed(z, z, z, torch.tensor([0, 4], dtype=torch.int32))
    with pytest.raises(RuntimeError):
        ops.add_rmsnorm(z, z, torch.ones(32))


def test_c_entries_refuse():
    """Argument errors of the C ABI come back as codes, nothing is launched."""
    from hv_amd import _lib as L
    lib = L.lib()
    buf = torch.zeros(4096, dtype=torch.uint8)
    p = (buf.data_ptr() + 63) // 64 * 64

    def args(**kw):
        a = L.AttnPackedArgs()
        base = dict(dtype=1, hq=4, hkv=2, d=32, nseq=1, scale=0.5, total_q=4, total_k=4, cu_q=p, cu_k=p, q=p, k=p, v=p,
                    q_row=128, q_head=32, k_row=64, k_head=32, v_row=64, v_head=32, out=p, lse=p, work=p, dout=p, do_row=128,
                    do_head=32, dq=p, dk=p, dv=p)
        base.update(kw)
        for n, v in base.items():
            setattr(a, n, v)
        return C.byref(a)

    inval = [dict(dtype=2), dict(hq=3), dict(hkv=0), dict(nseq=-1), dict(total_q=-1), dict(scale=0.0), dict(scale=-1.0),
             dict(scale=float("nan")), dict(cu_q=None), dict(q=None), dict(k=p + 2), dict(v_row=61), dict(q_head=3)]
    for kw in inval:
        assert lib.hv_attn_packed(args(**kw), None) == -1, kw
        assert lib.hv_attn_packed_backward(args(**kw), None) == -1, kw
    for kw in (dict(d=12), dict(d=136), dict(d=0), dict(total_q=1 << 30), dict(total_k=1 << 30)):
        assert lib.hv_attn_packed(args(**kw), None) == -2, kw
    assert lib.hv_attn_packed(args(out=None), None) == -1
    assert lib.hv_attn_packed(None, None) == -1
    for kw in (dict(dout=None), dict(lse=None), dict(work=None), dict(dk=None), dict(dv=p + 8), dict(dq=p + 8)):
        assert lib.hv_attn_packed_backward(args(**kw), None) == -1, kw
    assert lib.hv_attn_packed(args(total_q=0), None) == 0                   # nothing to do
    assert lib.hv_add_rmsnorm(0, p, 0, p, 0, 32, 1e-8, p, p, 0, p, None, None, None) == 0
    for bad in ((5, p, 0, p, 2, 32, 1e-8, p, p, 0, p, None, None), (0, p, 0, p, 2, 0, 1e-8, p, p, 0, p, None, None),
                (0, p, 0, p, 2, 32, -1.0, p, p, 0, p, None, None), (0, None, 0, p, 2, 32, 1e-8, p, p, 0, p, None, None),
                (0, p, 0, p, 2, 32, 1e-8, p, None, 0, p, None, None), (0, p, 0, p, 2, 32, 1e-8, p, p, 3, p, None, None),
                (0, p, 0, p, 2, 32, 1e-8, p, p, 2, p, None, None)):
        assert lib.hv_add_rmsnorm(*bad, None) == -1, bad
    assert lib.hv_add_rmsnorm(0, p, 0, p, 2, 32769, 1e-8, p, p, 0, p, None, None, None) == -2
    assert lib.hv_add_rmsnorm_backward(0, p, 0, p, p, p, 0, None, p, 2, 32, 0, p, p, p, p, None) == -1
    assert lib.hv_add_rmsnorm_backward(0, p, 2, p, p, p, 0, p, p, 2, 32, 0, p, p, p, p, None) == -1
    assert lib.hv_quantize_rows_fp8(0, p, 16, 2, 32, p, p, None) == -1
    for bad, rc in (((p, 32, p, p, 32, p, None, 9, 4, 4, 32, 1, p, 4, None), -1), ((p, 32, p, p, 32, p, None, 0, 4, 4, 32, 2, p, 4, None), -1),
                    ((p, 16, p, p, 32, p, None, 0, 4, 4, 32, 1, p, 4, None), -1), ((p, 32, p, p, 32, p, None, 0, 4, 4, 24, 1, p, 4, None), -2),
                    ((p + 1, 32, p, p, 32, p, None, 0, 4, 4, 32, 1, p, 4, None), -1), ((p, 32, None, p, 32, p, None, 0, 4, 4, 32, 1, p, 4, None), -1)):
        assert lib.hv_linear_fp8(*bad, None) == rc, bad
    # more outputs than a grid has blocks for
    assert lib.hv_linear_fp8(p, 16, p, p, 16, p, None, 0, 1 << 30, 1 << 28, 16, 1, p, 1 << 28, None, None) == -2
    # a description whose parts would pass 32 bits (every head reads one: stride 0): the workspace stays bounded
    assert 0 < lib.hv_attn_packed_work_bytes(args(hq=1024, hkv=1024, d=64, nseq=1, total_q=1, total_k=(1 << 30) - 1)) <= 256 << 20


def test_fake_kernels():
    import hv_amd  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        d = "cuda"
        q, k = torch.empty(10, 4, 64, device=d, dtype=torch.bfloat16), torch.empty(12, 2, 64, device=d, dtype=torch.bfloat16)
        cu = torch.empty(3, device=d, dtype=torch.int32)
        out, lse = torch.ops.hv.attention_packed(q, k, k, cu, cu, True)
        assert out.shape == q.shape and lse.shape == (10, 4) and lse.dtype == torch.float32
        x, r, w = torch.empty(5, 64, device=d, dtype=torch.bfloat16), torch.empty(5, 64, device=d), torch.empty(64, device=d)
        y, s = torch.ops.hv.add_rmsnorm(x, r, w)
        assert y.dtype == torch.bfloat16 and s.dtype == torch.float32
        c, sc, s = torch.ops.hv.add_rmsnorm_fp8(x, r, w)
        assert c.dtype == torch.float8_e4m3fn and sc.shape == (5,)
        w8, ws = torch.ops.hv.quantize_rows_fp8(torch.empty(7, 64, device=d))
        assert torch.ops.hv.linear_fp8(c, sc, w8, ws).shape == (5, 7)


# ------------------------------------------------------------------------------------------- strides and alignment of operands
def in_place(a, name):
    """Whether the C entry takes the operand of this description."""
    head = getattr(a, name + "_head"), getattr(a, name + "_row")
    return getattr(a, {"do": "dout"}.get(name, name)) % 16 == 0 and all(s * 2 % 16 == 0 for s in head)


def test_single_rows_and_heads_have_no_stride(ops):
    """The stride of a dimension of one element is never used: such operands are read in place."""
    cu = torch.tensor([0, 1], dtype=torch.int32)
    q = torch.zeros(5, 4 * 32 + 1, dtype=torch.bfloat16).as_strided((1, 4, 32), (129, 32, 1))
    k = torch.zeros(5, 2 * 32 + 1, dtype=torch.bfloat16).as_strided((1, 2, 32), (65, 32, 1))
    a = ops.attn_packed_args(q, k, k, cu, cu, False, None)
    assert all(in_place(a, n) for n in ("q", "k", "v")) and a.q_head == 32 and a.k == k.data_ptr()
    one = torch.zeros(6, 48, dtype=torch.bfloat16).as_strided((6, 1, 32), (48, 5, 1))
    a = ops.attn_packed_args(one, one, one, torch.tensor([0, 6], dtype=torch.int32), torch.tensor([0, 6], dtype=torch.int32), False, None)
    assert in_place(a, "q") and a.q_row == 48


def odd_views(rows, heads, d, dtype=torch.bfloat16):
    """Contiguous views off a 16-byte boundary, and single rows / heads whose strides mean nothing."""
    flat = torch.arange(rows * heads * d + 8, dtype=torch.float32).to(dtype)
    yield flat[1:1 + rows * heads * d].view(rows, heads, d)
    yield flat[3:3 + heads * d].view(1, heads, d)
    yield torch.ones(rows, heads * d + 1, dtype=dtype)[:1, :heads * d].view(1, heads, d)
    yield torch.ones(rows, heads * d + 3, dtype=dtype)[:, :d].view(rows, 1, d)

def test_operands_off_the_boundary_are_copied(ops, monkeypatch):
    """The differentiable form hands on operands that the kernels can read, with the same values: .contiguous() alone
    returns a contiguous view off the boundary as it is."""
    from hv_amd import train_fn
    got = []
    monkeypatch.setattr(train_fn.PackedAttentionFn, "apply", lambda *a: got.append(a) or (None, None))
    cu = torch.tensor([0, 6], dtype=torch.int32)
    for t in odd_views(6, 4, 32):
        train_fn.attention_packed(t, t, t, cu)
        for x in got.pop()[:3]:
            assert torch.equal(x, t)
            a = ops.attn_packed_args(x, x, x, cu, cu, False, None)
            assert in_place(a, "q")


def test_backward_copies_what_it_cannot_read(ops, monkeypatch):
    """Gradients that arrive as contiguous views off the boundary, far strides of a single row, and operands that saved-tensor
    hooks returned in another layout."""
    import contextlib
    from hv_amd import ops_train as T
    seen = []

    class Lib:
        def hv_attn_packed_backward_work_bytes(self, a):
            return 64

        def hv_attn_packed_backward(self, a, stream):
            seen.append(T.L.AttnPackedArgs.from_buffer_copy(a._obj))
            return 0

    monkeypatch.setattr(T.L, "lib", Lib)
    monkeypatch.setattr(T, "on_device", contextlib.nullcontext)
    for dout in odd_views(6, 4, 32):
        n, hq = dout.shape[:2]
        q = torch.zeros(n, hq, 32, dtype=torch.bfloat16)
        k = torch.zeros(n, hq * 32 + 1, dtype=torch.bfloat16)[:, :hq * 32].view(n, hq, 32)
        cu = torch.tensor([0, n], dtype=torch.int32)
        call = ops.attn_packed_args(q, q, q, cu, cu, False, None)
        out = torch.zeros(n * hq * 32 + 1, dtype=torch.bfloat16)[1:].view(n, hq, 32)
        lse = torch.zeros(hq, n).t()
        T.attention_packed_backward(q, k, k, cu, cu, call, out, torch.zeros_like(q), lse, dout)
        a = seen.pop()
        assert all(in_place(a, x) for x in ("q", "k", "v", "do")) and a.out % 16 == 0 and a.out_low % 16 == 0
        assert a.lse != lse.data_ptr() or lse.is_contiguous()


def test_dispatcher_gradient_carries_the_log_sum_exp(ops, monkeypatch):
    """A gradient of the second output reaches the backward kernel: it is an output like the first."""
    import contextlib
    import types
    from hv_amd import library, ops_train as T
    seen = []

    class Lib:
        def hv_attn_packed_work_bytes(self, a):
            return 0

        def hv_attn_packed(self, a, stream):
            return 0

        def hv_attn_packed_backward_work_bytes(self, a):
            return 64

        def hv_attn_packed_backward(self, a, stream):
            a = a._obj
            seen.append((C.c_float * 24).from_address(a.dlse)[:] if a.dlse else None)
            return 0

    monkeypatch.setattr(T.L, "lib", Lib)
    monkeypatch.setattr(T, "on_device", contextlib.nullcontext)
    q, cu = torch.zeros(6, 4, 32, dtype=torch.bfloat16), torch.tensor([0, 6], dtype=torch.int32)
    ctx = types.SimpleNamespace(saved_tensors=(q, q, q, cu, cu), meta=(True, None))
    dlse = torch.arange(24, dtype=torch.float32).view(6, 4)
    library._attn_packed_bwd(ctx, torch.zeros_like(q), dlse)
    assert seen.pop() == dlse.flatten().tolist()
    library._attn_packed_bwd(ctx, torch.zeros_like(q), dlse.t().contiguous().t())
    assert seen.pop() == dlse.flatten().tolist()
    library._attn_packed_bwd(ctx, torch.zeros_like(q), None)
    assert seen.pop() is None
    library._attn_packed_bwd(ctx, None, dlse)                       # the log-sum-exp alone
    assert seen.pop() == dlse.flatten().tolist()


def test_few_rows_form_only_where_its_grid_fits():
    """The join has a wave per (token, head): 2^26 of them and more are past a grid's 2^32 threads, the tile form takes them
    (no workspace)."""
    from hv_amd import _lib as L

    def work(total_q):
        a = L.AttnPackedArgs()
        for n, v in dict(dtype=1, hq=64, hkv=4, d=8, nseq=(1 << 20) - 1, scale=0.5, total_q=total_q, total_k=(1 << 30) - 1).items():
            setattr(a, n, v)
        return L.lib().hv_attn_packed_work_bytes(C.byref(a))

    assert work((1 << 19) - 1) > 0
    assert work((1 << 20) - 1) > 0 and work(1 << 20) == 0
