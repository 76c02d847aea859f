"""GPU tests of the operators around a block's projections beyond one call's agreement with its
definition: codes against the library's other quantisers' rule, calls that meet other calls."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def _randn(seed, *shape):
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda")


# --------------------------------------------------------------------------------------
# residual_norm: codes
# --------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,width", [(4096, 2048), (4096, 520), (512, 1001), (64, 16384)])
def test_codes_are_the_rounded_quotient(cuda_device, rows, width):
    """A code is round(h / scale) with the correctly rounded quotient, as the library's other
    quantisers give it: h in fp32 is stored as it is before the quantiser, so the codes follow
    from it bit for bit (torch divides fp32 correctly rounded and rounds ties to even)."""
    from h3tp import ops
    x, b = _randn(width, rows, width), _randn(width + 1, rows, width)
    pre = ops.NormSpec("rms", _randn(2, width))
    shift, scale = _randn(3, 1, width) * 0.3, _randn(4, 1, width) * 0.3
    kw = dict(pre=pre, shift=shift, scale=scale)
    y, h, _ = ops.residual_norm(x, b, out=torch.empty_like(x), **kw)
    z, q, s = ops.residual_norm(x, b, out=torch.empty_like(x), quantize=True, convrot=False, **kw)
    assert torch.equal(y, z)
    want_s = h.abs().amax(1, keepdim=True) * torch.tensor(1 / 127, device="cuda")
    assert torch.equal(s, want_s)
    want = torch.round(h / s).clamp(-128, 127).to(torch.int8)
    wrong = int((q != want).sum())
    assert wrong == 0, (wrong, q.numel())


# --------------------------------------------------------------------------------------
# two sizes of one kernel at once: they ask for different amounts of shared memory
# --------------------------------------------------------------------------------------
def _int4_entry(k):
    """A call of h3_int4_linear on a stream of its own, as a thread makes it: without Python's
    own work around the entry point, two threads are inside it most of the time."""
    from h3tp import _native as N
    x = _randn(k, 8, k).half()
    w = torch.randint(0, 256, (16, k // 2), device="cuda", dtype=torch.uint8)
    s, out, st = torch.ones(16, k // 64, device="cuda"), torch.empty(8, 16, device="cuda"), torch.cuda.Stream()
    args = (x.data_ptr(), N.TYPE_F16, k, 8, k, w.data_ptr(), 16, s.data_ptr(), N.TYPE_F32, None, 64, None,
            out.data_ptr(), N.TYPE_F32, st.cuda_stream)
    entry = N.load().h3_int4_linear
    return lambda: entry(*args), (x, w, s, out, st)


def _norm_entry(width):
    from h3tp import _native as N
    x, b = _randn(width, 8, width), _randn(width + 1, 8, width)
    out, h, st = torch.empty_like(x), torch.empty_like(x), torch.cuda.Stream()
    args = (x.data_ptr(), N.TYPE_F32, b.data_ptr(), N.TYPE_F32, 8, width, 1.0, None, 0, None, 0, None, 0, 1, None,
            N.NORM_NONE, None, None, 0.0, N.NORM_RMS, None, None, 1e-6, out.data_ptr(), h.data_ptr(), 0, None, None,
            st.cuda_stream)
    entry = N.load().h3_residual_norm
    return lambda: entry(*args), (x, b, out, h, st)


@pytest.mark.parametrize("entry,big,small", [(_int4_entry, 8192, 256), (_norm_entry, 2944, 1536)],
                         ids=["int4_linear", "residual_norm"])
def test_two_threads_with_two_sizes(cuda_device, entry, big, small):
    """Neither thread's launches are refused because of the other's size."""
    calls = [entry(size) for size in (big, small)]
    torch.cuda.synchronize()
    refused = [0, 0]

    def work(i):
        for _ in range(20000):
            refused[i] += calls[i][0]() != 0

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert refused == [0, 0]


def test_graph_of_two_sizes(cuda_device):
    """One graph with the larger size of a kernel before the smaller one, replayed."""
    from h3tp import ops

    def calls():
        out = []
        for k in (8192, 256):
            x = _randn(k, 8, k).half()
            w = torch.full((16, k // 2), 0x3A, device="cuda", dtype=torch.uint8)
            s = torch.ones(16, k // 64, device="cuda")
            out.append(([x], lambda x=x, w=w, s=s: ops.int4_linear(x, w, s, group=64)))
        for width in (2944, 1536):
            x, b = _randn(width, 8, width), _randn(width + 1, 8, width)
            out.append(([x, b], lambda x=x, b=b: ops.residual_norm(x, b, pre=ops.NormSpec(), out=torch.empty_like(x))[1]))
        return out

    made = calls()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = [c() for _, c in made]
    for _ in range(2):
        for inputs, _ in made:
            for t in inputs:
                t.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(h, c()) for h, (_, c) in zip(held, made))


# --------------------------------------------------------------------------------------
# int4_linear: the smallest scales
# --------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,low", [(torch.float16, 2.0 ** -24), (torch.bfloat16, 2.0 ** -126)])
def test_scales_below_the_normal_numbers(cuda_device, dtype, low):
    """fp16 scales down to the smallest subnormal, bf16 ones down to the smallest normal number:
    x, codes and scales are small integers times a power of two here, so every sum is exact."""
    from h3tp import ops
    k, n = 128, 32
    x = torch.randint(-8, 9, (3, k), device="cuda").to(torch.bfloat16)
    codes = torch.randint(0, 16, (n, k), device="cuda")
    w = (codes[:, 0::2] | (codes[:, 1::2] << 4)).to(torch.uint8)
    steps = torch.randint(1, 8, (n, k // 64), device="cuda")
    s = (steps.double() * low).to(dtype)
    want = x.double() @ ((codes - 8).double() * steps.repeat_interleave(64, 1).double()).T * low
    y = ops.int4_linear(x, w, s, group=64, out_dtype=torch.float32)
    assert torch.equal(y.double(), want)


# --------------------------------------------------------------------------------------
# outputs over tables, weights and positions
# --------------------------------------------------------------------------------------
def test_outputs_may_not_overlap_what_is_read(cuda_device):
    """Every row reads the tables and weights, so an output over one of them is refused; between
    the rows of a table there is room for one."""
    from h3tp import ops
    from h3tp.rms_rope import RotaryAxes, qk_norm_rope
    pre = ops.NormSpec()
    buf = _randn(1, 6, 64)
    x, b = buf[2:5], torch.ones(3, 64, device="cuda")
    lab = torch.zeros(3, dtype=torch.int32, device="cuda")
    one, keep = torch.zeros(1, 64, device="cuda"), buf.clone()
    for bad in (dict(gate=buf[2:3]), dict(gate=buf[1:3], labels=lab), dict(pre=pre, shift=buf[4:5]),
                dict(pre=pre, scale=buf[4:], labels=lab), dict(pre=ops.NormSpec("rms", buf[3])),
                dict(pre=ops.NormSpec("rms", None, buf[3])), dict(post=ops.NormSpec("rms", buf[4])),
                dict(post=ops.NormSpec("layer", None, buf[2])),
                dict(gate=one, labels=buf.view(torch.int32).view(-1)[130:133])):
        with pytest.raises(ValueError):
            ops.residual_norm(x, b, **bad)
        with pytest.raises(ValueError):
            ops.residual_norm(x.clone(), b, out=x, **bad)
    assert torch.equal(buf, keep)
    ops.residual_norm(x, b, gate=buf[1:2], pre=ops.NormSpec("rms", buf[5]), shift=buf[:1])
    wide = _randn(2, 2, 128)
    ops.residual_norm(wide[:1, 64:], b[:1], gate=wide[:, :64], labels=lab[:1])  # x between the gate's rows

    axes = RotaryAxes(64, (64,))
    packed = _randn(3, 4, 3, 64)
    q, pos = packed[:, :1], torch.zeros(4, dtype=torch.int32, device="cuda")
    whole = packed[:, :2]
    with pytest.raises(ValueError):
        qk_norm_rope(q, None, pos, axes, q_weight=packed[1, 0], out_q=q)
    with pytest.raises(ValueError):
        qk_norm_rope(q, whole[:, 1:], pos, axes, k_weight=packed[2, 1], out_k=whole[:, 1:])
    with pytest.raises(ValueError):
        qk_norm_rope(q, None, packed.view(torch.int32).view(-1)[:4], axes, out_q=q)
    w = packed[1, 2]  # between the heads of two tokens
    want, _ = qk_norm_rope(q.clone(), None, pos, axes, q_weight=w.clone())
    qk_norm_rope(q, None, pos, axes, q_weight=w, out_q=q)
    assert torch.equal(q, want)


# --------------------------------------------------------------------------------------
# arguments that are no tensors
# --------------------------------------------------------------------------------------
def test_arguments_that_are_no_tensors(cuda_device):
    from h3tp import ops
    from h3tp.rms_rope import RotaryAxes, packed_qk_norm_rope, qk_norm_rope
    x = torch.zeros(2, 64, dtype=torch.float16, device="cuda")
    w = torch.zeros(16, 32, dtype=torch.uint8, device="cuda")
    s, z = torch.zeros(16, 2, device="cuda"), torch.zeros(16, 2, dtype=torch.uint8, device="cuda")
    axes, pos = RotaryAxes(64, (64,)), torch.zeros(2, dtype=torch.int32, device="cuda")
    q = x.view(2, 1, 64)
    for bad in (3, [1.0], "x"):
        for call in (lambda: ops.residual_norm(bad), lambda: ops.residual_norm(x, bad),
                     lambda: ops.residual_norm(x, x.clone(), bad), lambda: ops.residual_norm(x, x.clone(), out=bad),
                     lambda: ops.residual_norm(x, x.clone(), labels=bad),
                     lambda: ops.residual_norm(x, pre=ops.NormSpec("rms", bad)),
                     lambda: ops.residual_norm(x, pre=ops.NormSpec(), shift=bad),
                     lambda: ops.int4_linear(bad, w, s, group=32), lambda: ops.int4_linear(x, bad, s, group=32),
                     lambda: ops.int4_linear(x, w, bad, group=32), lambda: ops.int4_linear(x, w, s, bad, group=32),
                     lambda: ops.int4_linear(x, w, s, z, group=32, bias=bad),
                     lambda: qk_norm_rope(bad, None, pos, axes), lambda: qk_norm_rope(q, bad, pos, axes),
                     lambda: qk_norm_rope(q, None, bad, axes), lambda: qk_norm_rope(q, None, pos, bad),
                     lambda: qk_norm_rope(q, None, pos, axes, q_weight=bad),
                     lambda: qk_norm_rope(q, None, pos, axes, out_q=bad),
                     lambda: packed_qk_norm_rope(bad, 1, 1, pos, axes)):
            with pytest.raises(ValueError):
                call()
    for call in (lambda: ops.int4_linear(x, None, s, group=32), lambda: ops.int4_linear(x, w, None, group=32),
                 lambda: qk_norm_rope(q, None, pos, None), lambda: qk_norm_rope(q, None, None, axes)):
        with pytest.raises(ValueError):
            call()


# --------------------------------------------------------------------------------------
# in place through another view of the same heads
# --------------------------------------------------------------------------------------
def test_in_place_through_another_view(cuda_device):
    """The stride of a dimension of one does not make an output another tensor than its input."""
    from h3tp.rms_rope import RotaryAxes, qk_norm_rope
    axes, pos = RotaryAxes(64, (64,)), torch.arange(5, device="cuda")
    x = _randn(1, 5, 64).half()
    for q, out in ((x.view(5, 1, 64), x.as_strided((5, 1, 64), (64, 7, 1))),
                   (x.view(1, 5, 64), x.as_strided((1, 5, 64), (9999, 64, 1)))):
        keep = x.clone()
        at = pos[:q.shape[0]]
        want, _ = qk_norm_rope(q.clone(), None, at, axes)
        got, _ = qk_norm_rope(q, None, at, axes, out_q=out)
        assert got is out and torch.equal(q, want)
        x.copy_(keep)


# --------------------------------------------------------------------------------------
# the block
# --------------------------------------------------------------------------------------
def _block():
    from h3tp.rms_rope import RotaryAxes
    from h3tp.tp_dit import TPDiTModulatedBlockINT8
    block = TPDiTModulatedBlockINT8(256, 256, 4, RotaryAxes(64, (64,)), 64, device="cuda", group=32)
    for m in (block.qkv_proj, block.out_proj, block.fc1, block.fc2):
        m.weight.data.random_(-100, 101)
        m.weight_scale.data.fill_(1e-4)
    block.modulation.load_from_full(_randn(1, 6 * 256, 64) * 0.05, _randn(2, 6 * 256))
    return block


class _Adapter:
    def add_to(self, source, out, **kw):
        return out


@pytest.mark.parametrize("which", ["qkv_proj", "fc1"])
def test_block_refuses_an_adapter_before_it_changes_the_residual(cuda_device, which):
    block = _block()
    getattr(block, which).lora_adapter = _Adapter()
    x, pos = _randn(3, 40, 256).half(), torch.arange(40, device="cuda")
    keep = x.clone()
    with pytest.raises(ValueError):
        block(x, _randn(4, 1, 64).half(), pos)
    assert torch.equal(x, keep)


def test_captured_block_keeps_its_labels(cuda_device):
    """The labels of captured calls stay as they are, however many other segment layouts come
    between captures and replays."""
    from h3tp.dit_fusion import labels_for
    block = _block()
    x0, cond, pos = _randn(5, 640, 256).half(), _randn(6, 2, 64).half(), torch.arange(640, device="cuda")
    segments = [(0, 77, 0), (77, 640, 1)]
    want = x0.clone()
    block(want, cond, pos, segments=segments)

    def other_layouts():
        for i in range(16):
            labels_for(x0, [(0, 100 + i, 1), (100 + i, 640, 0)], 2)
        torch.cuda.synchronize()
        return [torch.zeros(640, dtype=torch.int32, device="cuda") for _ in range(64)]

    runs, others = [], []
    for _ in range(2):
        x = x0.clone()
        block(x, cond, pos, segments=segments)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            block(x, cond, pos, segments=segments)
        runs.append((x, graph))
        others += other_layouts()
    for x, graph in runs:
        x.copy_(x0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, want)
    assert all(int(t.sum()) == 0 for t in others)


# --------------------------------------------------------------------------------------
# offsets past 32 bits
# --------------------------------------------------------------------------------------
def test_offsets_past_32_bits(cuda_device):
    """The last rows, tokens and columns of tensors of more than 2^31 elements (of int4_linear's
    weight: bytes) come out as in small calls."""
    from h3tp import ops
    from h3tp.rms_rope import RotaryAxes, qk_norm_rope
    rows, width = 690003, 3200
    x = torch.ones(rows, width, dtype=torch.float16, device="cuda")
    b = torch.ones_like(x)
    x[-9:], b[-9:] = _randn(1, 9, width), _randn(2, 9, width)
    kw = dict(pre=ops.NormSpec(), quantize=True, convrot=False)
    want = ops.residual_norm(x[-9:].clone(), b[-9:].clone(), **kw)
    got = ops.residual_norm(x, b, **kw)
    assert all(torch.equal(g[-9:], w) for g, w in zip(got, want))
    del x, b, got

    tokens, stride = 54001, 40000
    packed = torch.empty(tokens, stride, dtype=torch.float16, device="cuda")
    packed[:, -256:] = _randn(3, tokens, 256)
    q, k = (packed[:, a:a + 128 or None].unflatten(1, (2, 64)) for a in (-256, -128))
    axes, pos = RotaryAxes(64, (32, 32)), torch.randint(0, 9999, (tokens, 2), device="cuda")
    want = qk_norm_rope(q.contiguous(), k.contiguous(), pos, axes)
    got = qk_norm_rope(q, k, pos, axes, out_q=q, out_k=k)
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    del packed, q, k, got, want

    # x, codes and scales are small integers: every sum is exact, in any order
    n, k = 270000, 16384
    w = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda")
    s = torch.randint(1, 4, (n, k // 128), device="cuda").float()
    x = torch.randint(-2, 3, (3, k), device="cuda").half()
    y = ops.int4_linear(x, w, s, out_dtype=torch.float32)
    assert torch.equal(y[:, -40:], ops.int4_linear(x, w[-40:].contiguous(), s[-40:], out_dtype=torch.float32))
    del w, s, y
    m, n = 40000, 54000
    w = torch.randint(0, 256, (n, 16), dtype=torch.uint8, device="cuda")
    s, x = torch.ones(n, 1, device="cuda"), torch.randint(-2, 3, (m, 32), device="cuda").half()
    y = ops.int4_linear(x, w, s, group=32)
    assert torch.equal(y[-17:], ops.int4_linear(x[-17:], w, s, group=32))


def test_int4_linear_most_rows(cuda_device):
    from h3tp import ops
    w = torch.randint(0, 256, (16, 16), dtype=torch.uint8, device="cuda")
    s, x = torch.ones(16, 1, device="cuda"), torch.randint(-2, 3, (16 * 65535 + 1, 32), device="cuda").half()
    y = ops.int4_linear(x[:-1], w, s, group=32)
    assert torch.equal(y[-21:], ops.int4_linear(x[-22:-1], w, s, group=32))
    with pytest.raises(ValueError):
        ops.int4_linear(x, w, s, group=32)


def test_labels_on_several_threads(cuda_device):
    """More layouts than the table holds, from threads that evict each other's."""
    from h3tp.dit_fusion import labels_for
    x = torch.empty(64, 8, device="cuda")
    wrong = []

    def work(i):
        try:
            for k in range(400):
                cut = 1 + (7 * k + 3 * i) % 62
                got = labels_for(x, [(0, cut, 1), (cut, 64, 0)], 2)
                if int(got.sum()) != cut:
                    wrong.append((i, k))
        except Exception as e:  # noqa: BLE001 - told below
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == []


def test_first_calls_in_a_capture(cuda_device):
    """A process whose first calls, of sizes that raise the shared-memory limit, are captured."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import sys, torch
sys.path.insert(0, sys.argv[1])
from h3tp import ops
from h3tp.rms_rope import RotaryAxes, qk_norm_rope
x, b = torch.randn(5, 2944, device="cuda"), torch.randn(5, 2944, device="cuda")
a, w = torch.randn(3, 256, device="cuda").half(), torch.randint(0, 256, (32, 128), device="cuda", dtype=torch.uint8)
s, q, pos = torch.ones(32, 2, device="cuda"), torch.randn(4, 2, 64, device="cuda"), torch.arange(4, device="cuda")
def calls():
    return (ops.residual_norm(x, b, pre=ops.NormSpec(), out=torch.empty_like(x))[1], ops.int4_linear(a, w, s),
            qk_norm_rope(q, None, pos, RotaryAxes(64, (64,)))[0])
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    held = calls()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(h, c) for h, c in zip(held, calls()))
"""
    pkg = Path(__file__).resolve().parents[1] / "minimax-h3-2xt4_b200"
    r = subprocess.run([sys.executable, "-c", code, str(pkg)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
