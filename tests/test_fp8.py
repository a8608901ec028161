"""Host side of the 8-bit floating point operators, the row norm and gradient clipping: the oracle's own format against
torch's e4m3 type, refusals of the C ABI before any launch, refusals of the wrappers (no GPU)."""
import numpy as np
import pytest
import torch

from oracle import fp8 as F8


def test_oracle_codes_are_those_of_torch():
    c = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn)
    assert np.array_equal(F8.VALUES, c.double().numpy(), equal_nan=True)
    rs = np.random.RandomState(0)
    mids = (F8._POS[1:] + F8._POS[:-1]) / 2
    x = np.concatenate([mids, np.nextafter(mids, 0), np.nextafter(mids, 1e3), F8._POS, rs.uniform(0, 448, 5000), 2.0 ** rs.uniform(-12, 8.8, 5000)])
    x = np.concatenate([x, -x]).astype(np.float32)
    x = x[np.abs(x) <= 448]
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(F8.encode(x), want)


def test_oracle_scale_exponent_borders():
    for e in (-120, -3, 0, 5, 100):
        top = 448.0 * 2.0 ** e
        assert F8.scale_exponent(top) == e and F8.scale_exponent(np.nextafter(top, np.inf)) == e + 1
    assert F8.scale_exponent(0.0) == 0 and F8.scale_exponent(1e-45) == -126


def _rc(name, *args):
    import quantized_cnn_amd._lib as L
    rc = getattr(L.lib(), name)(*args)
    return rc, L.lib().aq_last_error().decode()


P = 4096  # an address that no call below reads


@pytest.mark.parametrize("args,word", [
    ((P, 7, 4, 128, 128, P, 128, P, 1, None, 0, None, 0, 1, 0, None, None, 0, None), "element type"),
    ((P, 0, 4, 128, 128, P, 128, P, 1, None, 0, None, 0, 1, 5, None, None, 0, None), "scale type"),
    ((P, 0, 4, 128, 128, P, 128, P, 1, None, 0, None, 0, 2, 0, None, None, 0, None), "blocks of 2 rows"),
    ((P, 0, -1, 128, 128, P, 128, P, 1, None, 0, None, 0, 1, 0, None, None, 0, None), "bad sizes"),
    ((P, 0, 4, 128, 128, None, 0, None, 0, None, 0, None, 0, 1, 0, None, None, 0, None), "no output"),
    ((P, 0, 4, 128, 100, P, 128, P, 1, None, 0, None, 0, 1, 0, None, None, 0, None), "pitch"),
    ((P, 0, 4, 128, 128, P, 128, None, 1, None, 0, None, 0, 1, 0, None, None, 0, None), "NULL"),
    ((P, 0, 4, 128, 128, P, 128, P, 1, None, 0, None, 0, 1, 0, P, None, 0, None), "column sums"),
    ((P, 0, 4, 128, 128, None, 0, None, 0, P, 4, P, 1, 1, 0, P, None, 0, None), "workspace"),
    ((P, 0, 1 << 40, 128, 128, P, 128, P, 1, None, 0, None, 0, 1, 0, None, None, 0, None), "too large"),
])
def test_quantize_refusals(args, word):
    rc, err = _rc("aq_fp8_quantize", *args)
    assert rc < 0 and word in err, err


@pytest.mark.parametrize("change,word", [
    ({"a_br": 3}, "blocks of 3"), ({"st": 9}, "scale type"), ({"K": 0}, "bad sizes"), ({"M": -2}, "bad sizes"), ({"lda": 24}, "pitch"),
    ({"lda": 136}, "multiples of 16"), ({"a": P + 8}, "multiples of 16"), ({"yt": 3}, "element type"), ({"ldy": 2}, "pitch"), ({"a": None}, "NULL"),
    ({"M": 1 << 40}, "too large")])
def test_matmul_refusals(change, word):
    v = dict(a=P, lda=128, a_br=1, st=0, M=4, K=128, yt=1, ldy=8)
    v.update(change)
    rc, err = _rc("aq_fp8_matmul", v["a"], v["lda"], P, 1, v["a_br"], P, 128, P, 1, 128, v["M"], 8, v["K"], v["st"], None, P, v["yt"], v["ldy"], None, 0, None)
    assert rc < 0 and word in err, err


def test_norm_and_clip_refusals():
    import ctypes as C
    rc, err = _rc("aq_rms_norm_fwd", P, 64, None, 0, 3, P, 4, 64, 1e-6, P, 64, None, 0, None, 0, 0, None, 0, P, None)
    assert rc < 0 and "element type" in err
    rc, err = _rc("aq_rms_norm_fwd", P, 64, None, 0, 0, P, 4, 0, 1e-6, P, 64, None, 0, None, 0, 0, None, 0, P, None)
    assert rc < 0 and "bad sizes" in err
    rc, err = _rc("aq_rms_norm_fwd", P, 64, None, 0, 0, P, 4, 64, -1.0, P, 64, None, 0, None, 0, 0, None, 0, P, None)
    assert rc < 0 and "eps" in err
    rc, err = _rc("aq_rms_norm_fwd", P, 63, None, 0, 0, P, 4, 64, 1e-6, P, 64, None, 0, None, 0, 0, None, 0, P, None)
    assert rc < 0 and "pitch" in err
    rc, err = _rc("aq_rms_norm_bwd", P, 64, None, 0, P, 64, 0, P, P, 4, 64, None, 0, None, None, 0, None)
    assert rc < 0 and "no output" in err
    rc, err = _rc("aq_rms_norm_bwd", P, 64, None, 0, P, 64, 0, P, P, 2000, 64, P, 64, P, None, 0, None)  # (few rows need none)
    assert rc < 0 and "workspace" in err
    one = lambda t, v: (t * 1)(v)  # noqa: E731
    p, n, t = one(C.c_void_p, P), one(C.c_longlong, 10), one(C.c_int, 0)
    rc, err = _rc("aq_clip_grad_norm", p, p, n, t, 1, -1.0, P, P, 64, None)
    assert rc < 0 and "max_norm" in err
    rc, err = _rc("aq_clip_grad_norm", p, p, n, one(C.c_int, 9), 1, 1.0, P, P, 64, None)
    assert rc < 0 and "element type" in err
    rc, err = _rc("aq_clip_grad_norm", p, p, n, t, 1, 1.0, P, P, 8, None)
    assert rc < 0 and "workspace" in err


def test_cpu_tensors_are_refused_loudly():
    from quantized_cnn_amd import ops
    x = torch.randn(4, 256)
    with pytest.raises(RuntimeError, match="HIP device only"):
        ops.fp8_quantize(x)
    with pytest.raises(RuntimeError, match="HIP device only"):
        ops.Fp8Blocks(x.to(torch.float8_e4m3fn), torch.ones(4, 2))
    with pytest.raises(RuntimeError, match="HIP device only"):
        ops.rms_norm_forward(x, torch.ones(256))
    with pytest.raises(RuntimeError, match="HIP device only"):
        ops.clip_grad_norm([x], 1.0)
    with pytest.raises(ValueError, match="empty"):
        ops.clip_grad_norm([], 1.0)
    with pytest.raises(ValueError):
        ops.fp8_matmul(x, x)


def test_training_steps_check_max_norm():
    from quantized_cnn_amd import train
    m = torch.nn.Linear(2, 2)
    for bad in (0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            train.CapturedStep(m, torch.optim.SGD(m.parameters(), 0.1), torch.nn.functional.mse_loss, max_norm=bad)


def test_a_residual_of_another_shape_is_refused():
    from quantized_cnn_amd import fp8
    x, w = torch.randn(4, 6, 128), torch.ones(128)
    for r in (torch.randn(6, 4, 128), torch.randn(24, 128), torch.randn(128)):  # as many elements, or fewer
        with pytest.raises(ValueError, match="residual"):
            fp8.rms_norm(x, w, residual=r)
        with pytest.raises(ValueError, match="residual"):
            fp8.norm_linear(x, w, torch.randn(128, 8), residual=r)


@pytest.mark.parametrize("ldas,ldbs", [(1 << 24, 1), (1, 1 << 30)])
def test_matmul_refuses_scales_too_far_apart(ldas, ldbs):
    """(the offsets of a tile's scales have 32 bits)"""
    rc, err = _rc("aq_fp8_matmul", P, 128, P, ldas, 1, P, 128, P, ldbs, 1, 256, 256, 128, 0, None, P, 1, 256, None, 0, None)
    assert rc < 0 and "pitch" in err and "scales" in err


@pytest.mark.parametrize("args,word", [
    ((P, 100, -1, 100, P, 112, None), "bad sizes"), ((P, 99, 4, 100, P, 112, None), "pitch"), ((P, 100, 4, 100, P, 100, None), "pitch"),
    ((P, 100, 4, 100, P + 8, 112, None), "multiples of 16"), ((P, 100, 4, 100, P, 120, None), "multiples of 16"), ((None, 100, 4, 100, P, 112, None), "NULL"),
    ((P, 100, 1 << 40, 100, P, 112, None), "too large")])
def test_repitch_refusals(args, word):
    rc, err = _rc("aq_fp8_repitch", *args)
    assert rc < 0 and word in err, err


def test_leaves_behind_operands_are_found():
    """(the check before a capture looks at them)"""
    from quantized_cnn_amd import fp8

    class Product(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w, b):
            return x @ w.float() + (0 if b is None else b)

        @staticmethod
        def backward(ctx, g):
            return g, g, g
    leaf = lambda *s, t=torch.float32: torch.randn(*s).to(t).requires_grad_(True)  # noqa: E731

    def names(out, weights):
        return sorted(id(n.variable) for n in fp8._leaf_nodes(out.grad_fn, weights))
    ids = lambda *ts: sorted(map(id, ts))  # noqa: E731
    x, w, b = leaf(2, 3, 4), leaf(5, 4, t=torch.bfloat16), leaf(5)
    y = Product.apply(x.view(6, 4), w.t(), b)
    assert names(y, (1, 2)) == ids(x, w, b)
    lo, hi = leaf(4, 2), leaf(2, 5)
    y = Product.apply(x.view(6, 4).relu(), torch.randn(4, 5) + lo @ hi, None)  # a weight of several leaves
    assert names(y, (1, 2)) == ids(x, lo, hi)
    z = Product.apply(y.relu(), torch.randn(5, 5), None)
    assert names(z, (1, 2)) == []  # (several operands: theirs are not this call's)
    z = Product.apply(Product.apply(x.view(6, 4), torch.randn(4, 5), None).relu(), torch.randn(5, 5), b)
    assert names(z, (1, 2)) == ids(x, b)
    z.grad_fn.next_functions[0][0].next_functions[0][0].metadata["fp8_checked"] = True  # a node of the module: its own call has looked
    assert names(z, (1, 2)) == ids(b)
    u, v = leaf(6, 4), leaf(6, 4)
    assert names(Product.apply(u + v, w.float().t(), None), (1, 2)) == ids(w)  # (what other operators join is theirs)


def test_dense_gradients_in_memory_order():
    from quantized_cnn_amd import ops
    for t in (torch.randn(4, 6).t(), torch.randn(2, 3, 4, 5).to(memory_format=torch.channels_last), torch.randn(3, 1, 5).permute(2, 1, 0), torch.randn(7),
              torch.tensor(2.0), torch.empty(0, 3).t(), torch.randn(1, 5).t(), torch.randn(2, 3, 4).permute(1, 2, 0)):
        v = ops.in_memory_order(t)
        assert v.is_contiguous() and v.data_ptr() == t.data_ptr() and v.numel() == t.numel()
        assert torch.equal(v.flatten().sort()[0], t.flatten().sort()[0])
    for t in (torch.randn(4, 6)[:, :5], torch.randn(1, 5).expand(3, 5), torch.randn(9).as_strided((3, 3), (2, 1)), torch.randn(6, 4)[::2].t()):
        with pytest.raises(ValueError, match="gaps or overlap"):
            ops.in_memory_order(t)


def test_package_imports_on_a_torch_without_a_gpu_back_end():
    import os
    import subprocess
    import sys
    code = ("import torch\n"
            "for name in [n for n in dir(torch._C) if n.startswith('_cuda')]: delattr(torch._C, name)\n"
            "import quantized_cnn_amd.layers, quantized_cnn_amd.checkpoint, quantized_cnn_amd.fp8, quantized_cnn_amd.train\n"
            "from quantized_cnn_amd import ops\n"
            "try: ops.fp8_quantize(torch.zeros(2, 2))\n"
            "except RuntimeError as e: print('refused:', e)\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "HIP device only" in r.stdout, r.stderr[-2000:]


def test_inline_assembly_names_what_it_writes():
    """m0 is the compiler's too: assembly that writes it has to say so."""
    import os
    import re
    src = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "quantized-cnn_amd", "csrc")
    for name in sorted(os.listdir(src)):
        if name.endswith((".hip", ".h")):
            with open(os.path.join(src, name)) as f:
                for stmt in re.findall(r"asm volatile\(.*?\);", f.read(), re.S):
                    assert "m0," not in stmt or '"m0"' in stmt, (name, stmt)
