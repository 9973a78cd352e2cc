"""What the documentation of expert layers, routers and adapter sets promises beside their values: padding, strides, streams, graphs, handles,
refusals, and all of them in turn as a layer uses them.

Where two calls have to give the same bits, no tolerance is involved.  Where values are compared, the bounds are those that
test_gpu_moe.py, test_gpu_adapters.py and test_gpu_router.py derive."""
import struct

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import magnitude_b200 as mb  # noqa: E402
from magnitude_b200 import _binding as B  # noqa: E402
from magnitude_b200 import ggml_quant as gq  # noqa: E402
from test_gpu_adapters import Set  # noqa: E402
from test_gpu_adapters import _check as check_adapters  # noqa: E402
from test_gpu_moe import Case  # noqa: E402
from test_gpu_moe import _check as check_moe  # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32
ROWS = [1, 2, 7, 16, 32, 33, 40]      # every launch plan of an expert layer: one row, a few, more


@pytest.fixture(scope="module")
def layer(backend, orc):
    return Case(backend, orc, 8, 3, 512, 768, mb.TYPE_Q4_K, mb.TYPE_Q6_K, 64, clamped=True, seed=3)


def _same(a, b):
    return torch.equal(a.view(torch.int16 if a.element_size() == 2 else torch.int32), b.view(torch.int16 if b.element_size() == 2 else torch.int32))


def _refused(backend, text, call):
    with pytest.raises(mb.B200QError) as e:
        call()
    assert e.value.status == B.ERR_INVALID_CONFIG and text in str(e.value), str(e.value)


# ---- expert layers ---------------------------------------------------------------------------------

@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_moe_rows_and_choices(backend, layer, m, dtype):
    x, ids, w = layer.inputs(m, dtype, 11)
    plain = backend.run_moe(layer.layer, x, ids, w, out_dtype=dtype)
    check_moe(plain, layer.want(x, ids, w), dtype == BF16)
    for _ in range(3):
        assert _same(plain, backend.run_moe(layer.layer, x, ids, w, out_dtype=dtype))
    # the result added to what is there: one more rounding-free term
    y0 = torch.randn_like(plain)
    got = backend.run_moe(layer.layer, x, ids, w, out=y0.clone(), accumulate=True)
    check_moe(got, layer.want(x, ids, w) + y0.double().cpu().numpy(), dtype == BF16)
    # no row has an expert: zeros, or what was there
    for none in (torch.full_like(ids, -1), torch.full_like(ids, 8), torch.full_like(ids, -2 ** 31)):
        assert not backend.run_moe(layer.layer, x, none, w, out=torch.full_like(plain, 7.0)).any()
        assert _same(y0, backend.run_moe(layer.layer, x, none, w, out=y0.clone(), accumulate=True))
    # the same expert twice, a choice that is none, a row without any
    ids[0, 1] = ids[0, 0]
    ids[m - 1, 2] = -1
    if m > 2:
        ids[1] = 99
    check_moe(backend.run_moe(layer.layer, x, ids, w, out_dtype=dtype), layer.want(x, ids, w), dtype == BF16)


@pytest.mark.parametrize("m", [2, 7, 17, 40])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_moe_a_bad_row_spoils_no_other(backend, layer, m, dtype):
    x, ids, w = layer.inputs(m, dtype, 12)
    ids[:] = ids[0]                      # all rows in the same groups
    clean = backend.run_moe(layer.layer, x, ids, w, out_dtype=dtype)
    for bad in (float("nan"), float("inf"), float("-inf")):
        y = x.clone()
        y[1, 300] = bad
        got = backend.run_moe(layer.layer, y, ids, w, out_dtype=dtype)
        assert got[1].isnan().all()
        keep = [r for r in range(m) if r != 1]
        assert _same(got[keep], clean[keep])


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_moe_strides_and_in_place(backend, layer, m, dtype):
    x, ids, w = layer.inputs(m, dtype, 13)
    plain = backend.run_moe(layer.layer, x, ids, w, out_dtype=dtype)
    # nothing aligned, everything a part of something wider
    wide = lambda t, pad, at: torch.full((m, t.shape[1] + pad), 5, dtype=t.dtype, device="cuda")[:, at:at + t.shape[1]].copy_(t)  # noqa: E731
    out = torch.full((m, 512 + 9), 3.0, dtype=dtype, device="cuda")
    got = backend.run_moe(layer.layer, wide(x, 5, 1), wide(ids, 2, 1), wide(w, 3, 2), out=out[:, 3:515])
    assert _same(got.contiguous(), plain)
    assert bool((out[:, :3] == 3).all() and (out[:, 515:] == 3).all())
    assert _same(backend.run_moe(layer.layer, x, ids, w, out=x), plain)


@pytest.mark.parametrize("m", [31, 130, 512])
def test_moe_every_row_the_same_experts(backend, orc, m):
    c = Case(backend, orc, 5, 2, 256, 288, mb.TYPE_Q8_0, mb.TYPE_Q8_0, 512, seed=4)
    x, ids, w = c.inputs(m, BF16, 14, spread=False)
    check_moe(backend.run_moe(c.layer, x, ids, w, out_dtype=F32), c.want(x, ids, w), False)


@pytest.mark.parametrize("experts,top_k,n_embd,n_ff,gu,dn,clamped", [
    (3, 2, 96, 32, mb.TYPE_Q8_0, mb.TYPE_Q8_0, True),            # less than one record, fewer tiles than blocks
    (16, 16, 1056, 544, mb.TYPE_MXFP4, mb.TYPE_Q4_0, True),      # every expert, a last record that is not full
    (300, 8, 2304, 512, mb.TYPE_Q5_K, mb.TYPE_Q5_K, False),
    (4, 2, 2048, 4096, mb.TYPE_Q6_K, mb.TYPE_Q6_K, False),       # fits beside the rings
    (4, 4, 1024, 7168, mb.TYPE_Q4_K, mb.TYPE_Q4_K, False),       # does not: lists and images
])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_moe_one_row(backend, orc, experts, top_k, n_embd, n_ff, gu, dn, clamped, dtype):
    c = Case(backend, orc, experts, top_k, n_embd, n_ff, gu, dn, 2, clamped, seed=n_ff)
    x, ids, w = c.inputs(1, dtype, 15)
    check_moe(backend.run_moe(c.layer, x, ids, w, out_dtype=dtype), c.want(x, ids, w), dtype == BF16)
    ids[0, top_k // 2] = -1
    check_moe(backend.run_moe(c.layer, x, ids, w, out_dtype=dtype), c.want(x, ids, w), dtype == BF16)


# ---- routers -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("m", [1, 8, 9, 40])
def test_router_ties_and_bad_numbers(backend, sigmoid, m):
    # expert e's logit is x[0] * (e // 2): pairs of equal ones; the lower index first
    w = torch.zeros(12, 64)
    w[:, 0] = torch.arange(12) // 2
    r = backend.router(w, 4, scoring=mb.SCORING_SIGMOID if sigmoid else mb.SCORING_SOFTMAX, max_rows=m)
    x = torch.zeros(m, 64, device="cuda")
    x[:, 0] = 1.0
    ids, weights = backend.route(r, x)
    assert ids.tolist() == [[10, 11, 8, 9]] * m
    x[:, 0] = 0.0
    ids, weights = backend.route(r, x)
    assert ids.tolist() == [[0, 1, 2, 3]] * m and torch.allclose(weights, torch.full_like(weights, 0.25), rtol=1e-6)
    # an infinity: 0 * inf is NaN, the lowest; of the others all are equally large
    x[m - 1, 0] = float("inf")
    ids, weights = backend.route(r, x)
    assert ids[m - 1].tolist() == [2, 3, 4, 5] and weights.isfinite().all()
    assert ids[:m - 1].tolist() == [[0, 1, 2, 3]] * (m - 1)
    # NaN everywhere: all are the lowest
    x[m - 1, 0] = float("nan")
    ids, weights = backend.route(r, x)
    assert ids[m - 1].tolist() == [0, 1, 2, 3] and weights.isfinite().all()
    assert ids[:m - 1].tolist() == [[0, 1, 2, 3]] * (m - 1)


def test_router_batches_strides_and_outputs(backend):
    g = torch.Generator().manual_seed(5)
    w, x = torch.randn((130, 1100), generator=g), torch.randn((300, 1100), generator=g).cuda()
    r = backend.router(w, 7, max_rows=300)
    ids, weights = backend.route(r, x)
    for n in (1, 2, 8, 9, 16, 17, 64):
        i, v = backend.route(r, x[:n])
        assert torch.equal(i, ids[:n]) and torch.allclose(v, weights[:n], rtol=1e-6, atol=0)
    wide = torch.zeros(300, 1107, device="cuda")
    wide[:, 3:1103] = x
    ids2, weights2 = torch.full((300, 10), -5, dtype=torch.int32, device="cuda"), torch.full((300, 9), -5.0, device="cuda")
    backend.route(r, wide[:, 3:1103], ids2[:, 1:8], weights2[:, 2:])
    assert torch.equal(ids2[:, 1:8], ids) and torch.equal(weights2[:, 2:], weights)
    assert bool((ids2[:, [0, 8, 9]] == -5).all() and (weights2[:, :2] == -5).all())


# ---- adapters ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("m,k,ns,ranks,adapters", [
    (300, 64, [40], [4], 300),                       # more items than blocks: a block takes one after the other
    (100, 96, [24, 56, 8, 40], [3, 17], 100),
    (60, 1024, [2048, 256], [1, 256, 8, 64], 60),    # shares by bytes
    (512, 256, [96], [8, 40], 37),
    (2100, 64, [40, 24, 33, 16], [256, 5], 3),       # t in two pieces
])
@pytest.mark.parametrize("x_dtype,y_dtype", [(BF16, BF16), (F32, F32)])
def test_adapters_many_items(backend, m, k, ns, ranks, adapters, x_dtype, y_dtype):
    """The error of t = A x is sqrt(K) 2^-24 of its terms' root sum of squares, which is 1 here (x is normal, A normal / sqrt(K)), not of t itself: of
    rank 1 a row's t may be far less (0.033 among these), so that the row's change says nothing about its error.  The bound of
    test_gpu_adapters.py therefore holds relative to what the change is on average, scale * sqrt(rank), where the change itself is less."""
    slots = [(7 * i) % adapters if i % 11 else -1 for i in range(m)]
    max_rank = 256 if 256 in ranks else 40
    sets = [Set(backend, n, k, [ranks[i % len(ranks)] for i in range(adapters)], BF16, max_rank, m + i) for i, n in enumerate(ns)]
    g = torch.Generator().manual_seed(m)
    x = torch.randn((m, k), generator=g).to(x_dtype).cuda()
    ys = [torch.randn((m, n), generator=g).to(y_dtype).cuda() for n in ns]
    before = [y.clone() for y in ys]
    slots = torch.tensor(slots, dtype=torch.int32, device="cuda")
    backend.apply_adapters([s.handle for s in sets], x, slots, ys)
    for s, y, b in zip(sets, ys, before):
        want, change = s.want(x, slots, b)
        usual = torch.tensor([[s.parts[i][2] * s.parts[i][0].shape[0] ** 0.5 if i >= 0 else 0.0] for i in slots.tolist()], dtype=torch.float64)
        check_adapters(y, want, torch.maximum(change.square().mean(dim=1, keepdim=True).sqrt(), usual), slots, b)


@pytest.mark.parametrize("m", [1, 30, 600])
def test_adapters_come_and_go(backend, m):
    g = torch.Generator().manual_seed(6)
    x = torch.randn((m, 320), generator=g).cuda()
    slots = torch.tensor([i % 3 for i in range(m)], dtype=torch.int32, device="cuda")
    y0 = torch.randn((m, 96), generator=g).cuda()
    s = Set(backend, 96, 320, [8, 0, 24], BF16, 24, 7)

    def run():
        y = backend.apply_adapters([s.handle], x, slots, [y0.clone()])[0]
        check_adapters(y, *s.want(x, slots, y0), slots, y0)
        return y

    first = run()
    assert _same(first, run())
    s.handle.unload(0)
    s.parts[0] = None
    run()
    a, b = torch.randn((5, 320), generator=g).to(BF16), torch.randn((96, 5), generator=g).to(BF16)      # a smaller rank where a larger one was
    s.handle.load(0, a, b, -2.0)
    s.parts[0] = (a.double(), b.double(), -2.0)
    run()


@pytest.mark.parametrize("m", [5, 100, 600])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_adapters_a_bad_row_spoils_no_other(backend, m, dtype):
    s = Set(backend, 200, 256, [16, 8], BF16, 16, 8)
    g = torch.Generator().manual_seed(9)
    x = torch.randn((m, 256), generator=g).to(dtype).cuda()
    slots = torch.tensor([0 if i < 4 else i % 3 - 1 for i in range(m)], dtype=torch.int32, device="cuda")
    y0 = torch.randn((m, 200), generator=g).to(dtype).cuda()
    clean = backend.apply_adapters([s.handle], x, slots, [y0.clone()])[0]
    for bad in (float("nan"), float("inf")):
        x2 = x.clone()
        x2[3, 100] = bad
        got = backend.apply_adapters([s.handle], x2, slots, [y0.clone()])[0]
        assert not got[3].isfinite().any()
        keep = [r for r in range(m) if r != 3]
        assert _same(got[keep], clean[keep])


# ---- far apart -----

@pytest.fixture(scope="module")
def far():
    """Room for rows whose offsets pass 2^31 elements (5.4 GB of bf16; only the rows themselves are ever touched)."""
    free = torch.cuda.mem_get_info()[0]
    if free < 16 << 30:
        pytest.skip("too little device memory free")
    x, y = torch.empty(2 ** 31 + 2 ** 28, dtype=BF16, device="cuda"), torch.empty(2 ** 31 + 2 ** 28, dtype=BF16, device="cuda")
    return lambda m, n, second: (y if second else x).as_strided((m, n), (2 ** 31 // (m - 1) // 8 * 8 + 8, 1))


@pytest.mark.parametrize("m", [3, 12, 40])
def test_moe_and_router_rows_far_apart(backend, layer, far, m):
    x, ids, w = layer.inputs(m, BF16, 71)
    r = backend.router(torch.randn((8, 512), generator=torch.Generator().manual_seed(72)), 3, max_rows=m)
    ids, w = backend.route(r, x)
    fx, fy = far(m, 512, False), far(m, 512, True)
    fx.copy_(x)
    ids2, w2 = backend.route(r, fx)
    assert torch.equal(ids, ids2) and torch.equal(w, w2)
    assert _same(backend.run_moe(layer.layer, fx, ids, w, out=fy).contiguous(), backend.run_moe(layer.layer, x, ids, w, out_dtype=BF16))


@pytest.mark.parametrize("m", [3, 100, 600])
def test_adapters_rows_far_apart(backend, far, m):
    s = Set(backend, 200, 320, [8, 16], BF16, 16, 73)
    g = torch.Generator().manual_seed(74)
    x, y0 = torch.randn((m, 320), generator=g).to(BF16).cuda(), torch.randn((m, 200), generator=g).to(BF16).cuda()
    slots = torch.tensor([i % 3 - 1 for i in range(m)], dtype=torch.int32, device="cuda")
    fx, fy = far(m, 320, False), far(m, 200, True)
    fx.copy_(x)
    fy.copy_(y0)
    backend.apply_adapters([s.handle], fx, slots, [fy])
    assert _same(fy.contiguous(), backend.apply_adapters([s.handle], x, slots, [y0])[0])


# ---- together ----------------------------------------------------------------------------------------

class Block:
    """Projection with adapters, router and experts of one layer, as an engine holds them."""

    def __init__(self, backend, orc, layer, rows):
        self.be, self.moe, n, k = backend, layer, 512, 512
        self.packed = gq.synth_weights(mb.TYPE_Q4_K, n, k, 21)
        self.w = backend.upload(mb.TYPE_Q4_K, self.packed, n, k)
        self.orc = orc
        self.set = Set(backend, n, k, [8, 16, 0], BF16, 16, 22)
        self.gate = torch.randn((8, 512), generator=torch.Generator().manual_seed(23)) * 0.1
        self.router = backend.router(self.gate, 3, max_rows=rows)

    def run(self, x, slots, stream=None):
        h = self.be.project(self.w, x, out_dtype=F32, stream=stream)
        base = h.clone()
        self.be.apply_adapters([self.set.handle], x, slots, [h], stream=stream)
        ids, weights = self.be.route(self.router, h, stream=stream)
        y = self.be.run_moe(self.moe.layer, h, ids, weights, out=h.clone(), accumulate=True, stream=stream)
        return base, h, ids, weights, y


@pytest.mark.parametrize("m", [1, 5, 33])
def test_a_layer(backend, orc, layer, m):
    b = Block(backend, orc, layer, 64)
    g = torch.Generator().manual_seed(m)
    x = torch.randn((m, 512), generator=g).to(BF16).cuda()
    slots = torch.tensor([i % 4 - 1 for i in range(m)], dtype=torch.int32, device="cuda")
    base, h, ids, weights, y = b.run(x, slots)
    ref = orc.matmul_exact(mb.TYPE_Q4_K, b.packed, 512, 512, x.float().cpu().numpy())
    # The projection itself: up to 16 rows 1e-3, as test_gpu_parity.py has it.  More rows go to the tensor cores with weights and (bf16, exact in
    # fp16) activations in fp16: a weight is off by at most half a step, 2^-11 of itself, evenly spread 2^-11 / sqrt(3) = 2.8e-4; so is a sum of
    # independent terms, relative to its rms, and the largest of 17 thousand of them by 4.3 sigma, 1.2e-3: test_gpu_gemm.py's 5e-3
    assert orc.within_tolerance(base.cpu().numpy(), ref, 1e-3 if m <= 16 else 5e-3)[0]
    check_adapters(h, *b.set.want(x, slots, base), slots, base)                   # every step from what the one before left
    logits = h.double().cpu() @ b.gate.double().T
    order = torch.argsort(logits, dim=1, descending=True, stable=True)[:, :3]
    assert torch.equal(ids.cpu().long(), order)
    want = torch.softmax(torch.gather(logits, 1, order), dim=1)
    assert bool(((weights.cpu().double() - want).abs() <= 1e-6 * want).all())
    check_moe(y, layer.want(h, ids, weights) + h.double().cpu().numpy(), False)


def test_a_layer_on_another_stream_and_captured(backend, orc, layer):
    b = Block(backend, orc, layer, 64)
    g = torch.Generator().manual_seed(31)
    xs = [torch.randn((m, 512), generator=g).to(BF16).cuda() for m in (1, 6, 24)]
    slots = [torch.tensor([(i + j) % 4 - 1 for i in range(len(x))], dtype=torch.int32, device="cuda") for j, x in enumerate(xs)]
    want = [[t.clone() for t in b.run(x, s)] for x, s in zip(xs, slots)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x, s, w in zip(xs, slots, want):
            got = b.run(x, s)
            side.synchronize()
            assert all(_same(p, q) for p, q in zip(got, w))
    # graphs that share the workspaces, replayed one after the other, with inputs that change
    graphs, held = [], []
    for x, s in zip(xs, slots):
        x, s = x.clone(), s.clone()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = b.run(x, s)
        graphs.append(gr)
        held.append((x, s, out))
    for turn in range(3):
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for (x, s, out), w in zip(held, want):
            assert all(_same(p, q) for p, q in zip(out, w))
        for (x, s, _), i in zip(held, range(3)):
            x.copy_(torch.randn(x.shape, generator=g).to(BF16))
            s.copy_(s.roll(1))
            want[i] = [t.clone() for t in b.run(x, s)]
        torch.cuda.synchronize()
    # a stream handed over by hand, and no rows at all
    got = b.run(held[0][0], held[0][1], stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert all(_same(p, q) for p, q in zip(got, want[0]))
    none = torch.zeros((0, 512), dtype=BF16, device="cuda")
    assert backend.apply_adapters([b.set.handle], none, slots[0][:0], [torch.zeros(0, 512, device="cuda")])[0].shape == (0, 512)
    ids, weights = backend.route(b.router, none)
    assert backend.run_moe(layer.layer, none, ids, weights).shape == (0, 512)


def test_experts_of_a_gguf_file(backend, orc, tmp_path):
    """gate, up and down as the 3-D tensors of a GGUF file hold them."""
    c = Case(backend, orc, 4, 2, 256, 512, mb.TYPE_Q4_K, mb.TYPE_Q6_K, 8, seed=41)
    rng = np.random.default_rng(42)
    parts = {}
    for name, qt, n, k in (("gate", mb.TYPE_Q4_K, 512, 256), ("up", mb.TYPE_Q4_K, 512, 256), ("down", mb.TYPE_Q6_K, 256, 512)):
        parts[name] = (qt, [k, n, 4], orc.quantize(qt, rng.standard_normal((4 * n, k), dtype=np.float32) * np.float32(k ** -0.5)))
    path = tmp_path / "experts.gguf"
    infos, data = b"", b""
    for n, (qt, dims, packed) in parts.items():
        data += bytes(-len(data) % 32)
        name = f"blk.0.ffn_{n}_exps.weight".encode()
        infos += struct.pack("<Q", len(name)) + name + struct.pack("<IQQQIQ", 3, *dims, qt, len(data))
        data += packed.tobytes()
    head = b"GGUF" + struct.pack("<IQQ", 3, len(parts), 0) + infos
    path.write_bytes(head + bytes(-len(head) % 32) + data)
    f = mb.GgufFile(path)
    read = {n: f.read(f"blk.0.ffn_{n}_exps.weight") for n in parts}
    f.close()
    layer = backend.moe(read["gate"], read["up"], read["down"], gate_up_type=mb.TYPE_Q4_K, down_type=mb.TYPE_Q6_K, top_k=2, n_embd=256, n_ff=512, max_rows=8)
    assert layer.n_experts == 4
    value = lambda n, k: orc.dequantize(parts[n][0], parts[n][2], k).astype(np.float64).reshape(4, -1, k)  # noqa: E731
    c.g, c.u, c.d = value("gate", 256), value("up", 256), value("down", 512)
    x, ids, w = c.inputs(5, BF16, 43)
    check_moe(backend.run_moe(layer, x, ids, w), c.want(x, ids, w), False)


# ---- handles and refusals ------------------------------------------------------------------------------

def test_handles_outlive_their_context(layer):
    be = mb.Backend(0)
    blocks = np.zeros((2, 32, 34), np.uint8)
    made = [be.moe(blocks, blocks, blocks, gate_up_type=mb.TYPE_Q8_0, down_type=mb.TYPE_Q8_0, top_k=1, n_embd=32, n_ff=32, max_rows=4),
            be.router(np.zeros((4, 32), np.float32), 2), be.adapters(32, 32, BF16, 2, 8)]
    x = torch.zeros(2, 32, device="cuda")
    ids, w = be.route(made[1], x)
    assert not be.run_moe(made[0], x, ids[:, :1].contiguous(), w[:, :1].contiguous()).any()
    be._children.clear()                 # (it would close them first)
    be.close()
    for h in made:
        h.close()
        h.close()


def test_refusals(backend, layer):
    x, ids, w = layer.inputs(4, BF16, 51)
    lay, other = layer.layer, mb.Backend(0)
    no = lambda text, call: _refused(backend, text, call)  # noqa: E731
    no("max_rows=64", lambda: backend.run_moe(lay, x[:1].repeat(65, 1), ids[:1].repeat(65, 1), w[:1].repeat(65, 1)))
    no("another context", lambda: other.run_moe(lay, x, ids, w))
    no("not (rows, 512)", lambda: backend.run_moe(lay, x[:, :511], ids, w))
    no("x is torch.float16", lambda: backend.run_moe(lay, x.half(), ids, w))
    no("ids is torch.int64", lambda: backend.run_moe(lay, x, ids.long(), w))
    no("weights is on cpu", lambda: backend.run_moe(lay, x, ids, w.cpu()))
    no("ids has shape (3, 3)", lambda: backend.run_moe(lay, x, ids[:3], w))
    no("accumulate needs", lambda: backend.run_moe(lay, x, ids, w, accumulate=True))
    lib = B.lib()
    run = lambda flags=0, ldx=512, xd=B.TYPE_BF16, m=4, y=x.data_ptr(): lib.b200q_moe_run(  # noqa: E731
        backend._h, lay._h, x.data_ptr(), xd, m, ldx, ids.data_ptr(), 3, w.data_ptr(), 3, y, B.TYPE_BF16, 512, flags, None)
    assert [run(flags=2), run(ldx=511), run(xd=B.TYPE_F16), run(m=-1), run(y=None)] == [B.ERR_INVALID_CONFIG] * 5

    blocks = np.zeros((2, 32, 34), np.uint8)
    base = dict(gate_up_type=mb.TYPE_Q8_0, down_type=mb.TYPE_Q8_0, top_k=1, n_embd=32, n_ff=32, max_rows=4)
    for text, change in (("at most the experts", dict(top_k=3)), ("max_rows must be", dict(max_rows=513)), ("max_rows must be", dict(max_rows=0)),
                         ("do not match", dict(down_type=mb.TYPE_Q4_0)), ("unknown activation", dict(activation=7)),
                         ("a limit above 0", dict(activation=mb.MOE_SWIGLU_CLAMPED, alpha=1.0, limit=0.0)),
                         ("a limit above 0", dict(activation=mb.MOE_SWIGLU_CLAMPED, alpha=float("nan"), limit=1.0))):
        no(text, lambda: backend.moe(blocks, blocks, blocks, **{**base, **change}))

    gate = np.zeros((4, 32), np.float32)
    r = backend.router(gate, 2, max_rows=3)
    no("max_rows=3", lambda: backend.route(r, torch.zeros(4, 32, device="cuda")))
    no("another context", lambda: other.route(r, torch.zeros(3, 32, device="cuda")))
    no("not (3, 2)", lambda: backend.route(r, torch.zeros(3, 32, device="cuda"), ids=ids[:, :2]))
    for text, change in (("at most the experts", dict(top_k=5)), ("unknown scoring", dict(scoring=2)), ("scale is not finite", dict(scale=float("inf"))),
                         ("softmax takes logit_bias", dict(select_bias=np.zeros(4, np.float32))), ("max_rows must be", dict(max_rows=0))):
        no(text, lambda: backend.router(gate, **{**dict(top_k=2), **change}))

    s, s2, s16 = backend.adapters(32, 64, BF16, 2, 8), backend.adapters(16, 64, BF16, 2, 8), backend.adapters(32, 64, torch.float16, 2, 8)
    xa, sl, y = torch.zeros(3, 64, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, 32, device="cuda")
    no("slot 2 is outside", lambda: s.load(2, torch.zeros(4, 64, dtype=BF16), torch.zeros(32, 4, dtype=BF16)))
    no("rank 9 is outside", lambda: s.load(0, torch.zeros(9, 64, dtype=BF16), torch.zeros(32, 9, dtype=BF16)))
    no("not (rank, 64)", lambda: s.load(0, torch.zeros(4, 63, dtype=BF16), torch.zeros(32, 4, dtype=BF16)))
    no("not bfloat16", lambda: s.load(0, torch.zeros(4, 64), torch.zeros(32, 4)))
    no("max_rank must be", lambda: backend.adapters(32, 64, BF16, 2, 257))
    no("same output", lambda: backend.apply_adapters([s, s], xa, sl, [y, y]))
    no("activation itself", lambda: backend.apply_adapters([s], xa, sl, [xa[:, :32]]))
    no("share dtype and K", lambda: backend.apply_adapters([s, s16], xa, sl, [y, y.clone()]))
    no("of one dtype", lambda: backend.apply_adapters([s, s2], xa, sl, [y, torch.zeros(3, 16, dtype=BF16, device="cuda")]))
    no("another context", lambda: other.apply_adapters([s], xa, sl, [y]))
    no("1..4 sets", lambda: backend.apply_adapters([s], xa, sl, []))
    no("contiguous int32", lambda: backend.apply_adapters([s], xa, sl.long(), [y]))
    no("contiguous int32", lambda: backend.apply_adapters([s], xa, torch.zeros(6, dtype=torch.int32, device="cuda")[::2], [y]))
    other.close()
    backend.sync()


@pytest.mark.parametrize("m", [3, 600])
@pytest.mark.parametrize("x_dtype,dtype", [(BF16, BF16), (F32, torch.float16)])
def test_adapters_long_sums_keep_their_bits(backend, m, x_dtype, dtype):
    """Sums of 16 thousand terms, fp32 results, relative root mean square error.  The tensor cores cut off what they add: on average a third
    of 2^-23 of the sum so far.  A chunk of 32 terms is at most twelve such additions to sums that grow, half their number in effect: 6 * 0.3 * 2^-23 =
    2.1e-7 of the chunk, and as much of the whole, chunks being independent; adding some 20 partial sums up in fp32 costs sqrt(10) 2^-24 / sqrt(3) =
    1.1e-7, B t as much as a chunk again, 2.1e-7, the result's rounding 3e-8: 3.2e-7 together, and twice that is taken.  (All terms added on the
    tensor cores to one sum: above 1e-6.)"""
    g = torch.Generator().manual_seed(m)
    s = Set(backend, 256, 16000, [16], dtype, 16, 61)
    x = torch.randn((m, 16000), generator=g).to(x_dtype).cuda()
    slots = torch.zeros(m, dtype=torch.int32, device="cuda")
    y = torch.zeros(m, 256, device="cuda")
    backend.apply_adapters([s.handle], x, slots, [y])
    want, _ = s.want(x, slots, torch.zeros(m, 256))
    assert float((y.cpu().double() - want).norm() / want.norm()) <= 6.4e-7
