"""Expert layers (b200q_moe_run) against a plain implementation in 64 bits on the oracle's dequantized weights.

Tolerances, relative to the row's root mean square r of y (or to |y| where that is more).  With bf16 results the activations
enter as 16-bit fixed point per 256 elements: a step is largest / 32512, an error at most half of it and, being spread evenly,
step / sqrt(12) on average; for normal data (largest about 4 sigma) that is 3.6e-5 sigma on x and as much on h, whose error passes
through the gate's slope (at most 1.1) once.  Summed over independent terms the relative error of a result is of that size, and
the largest of some ten thousand results lies below 6 of it: 3 * 6 * 3.6e-5 = 6.5e-4, plus half a bf16 step, 2^-8 = 3.9e-3 of the
value; h has longer tails than x (largest about 10 sigma instead of 4), so 1e-3 is taken for the first: 4.9e-3 together.  With fp32 results the 31-bit form is exact to
2^-30 of the largest and fp32 sums of n terms err by about sqrt(n) 2^-24 r: with n of some thousand 4e-6, and 2e-5 is taken; expf
errs by 2 ulp, less."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import magnitude_b200 as mb  # noqa: E402

TYPES = [mb.TYPE_Q4_K, mb.TYPE_Q6_K, mb.TYPE_Q8_0, mb.TYPE_Q5_K, mb.TYPE_Q4_0, mb.TYPE_MXFP4]


def _packed(orc, qt, experts, n, k, seed):
    rng = np.random.default_rng(seed)
    return orc.quantize(qt, rng.standard_normal((experts * n, k), dtype=np.float32) * np.float32(k ** -0.5)).reshape(experts, n, -1)


class Case:
    def __init__(self, backend, orc, experts, top_k, n_embd, n_ff, gu, dn, max_rows, clamped=False, seed=0, on_gpu=False):
        self.be, self.top_k, self.experts, self.n_embd, self.n_ff, self.clamped = backend, top_k, experts, n_embd, n_ff, clamped
        g, u = _packed(orc, gu, experts, n_ff, n_embd, seed), _packed(orc, gu, experts, n_ff, n_embd, seed + 1)
        d = _packed(orc, dn, experts, n_embd, n_ff, seed + 2)
        value = lambda qt, p, k: orc.dequantize(qt, p.reshape(-1, p.shape[-1]), k).astype(np.float64).reshape(experts, -1, k)  # noqa: E731
        self.g, self.u, self.d = value(gu, g, n_embd), value(gu, u, n_embd), value(dn, d, n_ff)
        rng = np.random.default_rng(seed + 3)
        bias = {}
        if clamped:
            bias = {n: rng.standard_normal((experts, w)).astype(np.float32) for n, w in (("gate_bias", n_ff), ("up_bias", n_ff), ("down_bias", n_embd))}
        self.bias = bias
        put = (lambda a: torch.from_numpy(a).cuda()) if on_gpu else (lambda a: a)
        self.layer = backend.moe(put(g), put(u), put(d), gate_up_type=gu, down_type=dn, top_k=top_k, n_embd=n_embd, n_ff=n_ff, max_rows=max_rows,
                                 activation=mb.MOE_SWIGLU_CLAMPED if clamped else mb.MOE_SWIGLU, alpha=1.7, limit=1.5,
                                 **{n: put(b) for n, b in bias.items()})

    def inputs(self, m, dtype, seed, spread=True):
        rng = np.random.default_rng(seed)
        x = torch.from_numpy(rng.standard_normal((m, self.n_embd), dtype=np.float32)).cuda().to(dtype)
        ids = np.stack([rng.permutation(self.experts)[: self.top_k] for _ in range(m)]) if spread else np.tile(np.arange(self.top_k), (m, 1))
        return x, torch.from_numpy(ids.astype(np.int32)).cuda(), torch.from_numpy(rng.random((m, self.top_k), dtype=np.float32)).cuda()

    def want(self, x, ids, weights):
        x, ids, weights = x.float().cpu().numpy().astype(np.float64), ids.cpu().numpy(), weights.cpu().numpy().astype(np.float64)
        y = np.zeros((len(x), self.n_embd))
        for m in range(len(x)):
            for e, w in zip(ids[m], weights[m]):
                if not 0 <= e < self.experts:
                    continue
                a, b = self.g[e] @ x[m], self.u[e] @ x[m]
                if self.clamped:
                    a = np.minimum(a + self.bias["gate_bias"][e], 1.5)
                    b = np.clip(b + self.bias["up_bias"][e], -1.5, 1.5)
                    h = a / (1 + np.exp(-np.float64(np.float32(1.7)) * a)) * (b + 1)
                else:
                    h = a / (1 + np.exp(-a)) * b
                out = self.d[e] @ h
                if self.clamped:
                    out = out + self.bias["down_bias"][e]
                y[m] += w * out
        return y


def _check(got, want, bf16):
    got = got.float().cpu().numpy().astype(np.float64)
    rms = np.sqrt(np.mean(want ** 2, axis=1, keepdims=True))
    err = np.abs(got - want) / np.maximum(np.maximum(np.abs(want), rms), 1e-30)
    assert err.max() <= (4.9e-3 if bf16 else 2e-5), f"worst relative error {err.max():.2e}"


@pytest.mark.parametrize("qt", TYPES)
@pytest.mark.parametrize("y_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m", [1, 3, 16])
def test_types(backend, orc, qt, y_dtype, m):
    c = Case(backend, orc, 8, 2, 512, 768, qt, qt, 16, seed=qt)
    x, ids, w = c.inputs(m, torch.bfloat16, m)
    y = backend.run_moe(c.layer, x, ids, w, out_dtype=y_dtype)
    _check(y, c.want(x, ids, w), y_dtype == torch.bfloat16)


@pytest.mark.parametrize("experts,top_k,n_embd,n_ff,gu,dn,m,x_dtype,y_dtype,clamped", [
    (1, 1, 256, 256, mb.TYPE_Q4_K, mb.TYPE_Q6_K, 1, torch.bfloat16, torch.float32, False),
    (5, 3, 288, 96, mb.TYPE_Q8_0, mb.TYPE_Q8_0, 7, torch.float32, torch.float32, True),         # nothing is a multiple of 256 or 16
    (3, 2, 1056, 544, mb.TYPE_MXFP4, mb.TYPE_Q4_0, 5, torch.bfloat16, torch.bfloat16, True),
    (16, 16, 768, 256, mb.TYPE_Q4_K, mb.TYPE_Q8_0, 2, torch.float32, torch.bfloat16, False),     # every expert
    (300, 4, 256, 256, mb.TYPE_Q6_K, mb.TYPE_Q5_K, 9, torch.bfloat16, torch.float32, False),     # more experts than threads of a block
    (4, 2, 2304, 2816, mb.TYPE_Q5_K, mb.TYPE_Q6_K, 40, torch.bfloat16, torch.bfloat16, False),   # several groups an expert
    (4, 4, 512, 512, mb.TYPE_Q4_K, mb.TYPE_Q4_K, 130, torch.float32, torch.float32, False),      # sums beyond shared memory
])
def test_shapes(backend, orc, experts, top_k, n_embd, n_ff, gu, dn, m, x_dtype, y_dtype, clamped):
    c = Case(backend, orc, experts, top_k, n_embd, n_ff, gu, dn, m, clamped, seed=n_embd + m, on_gpu=True)
    x, ids, w = c.inputs(m, x_dtype, 5)
    y = backend.run_moe(c.layer, x, ids, w, out_dtype=y_dtype)
    _check(y, c.want(x, ids, w), y_dtype == torch.bfloat16)
