"""Routers (b200q_router_run) against the choice from logits in 64 bits.  ids have to be equal; a weight is the quotient of an fp32 value
by an fp32 sum of up to 32 such (each within 2^-23 of its own), times the scale: 1e-6 relative."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import magnitude_b200 as mb  # noqa: E402


def _want(logits, top_k, sigmoid, normalise, scale, select):
    logits = np.nan_to_num(logits, nan=-np.finfo(np.float64).max, posinf=np.finfo(np.float64).max, neginf=-np.finfo(np.float64).max)
    with np.errstate(over="ignore"):
        score = 1 / (1 + np.exp(-logits)) if sigmoid else np.exp(logits - logits.max(axis=1, keepdims=True))
    ids = np.argsort(-(score + select if sigmoid else logits), axis=1, kind="stable")[:, :top_k]
    w = np.take_along_axis(score, ids, axis=1)
    by = w.sum(axis=1, keepdims=True) if normalise else (1.0 if sigmoid else score.sum(axis=1, keepdims=True))
    return ids, w / by * scale


@pytest.mark.parametrize("experts,top_k,k,m,x_dtype,w_dtype,sigmoid,normalise,biased", [
    (1, 1, 1, 1, torch.float32, torch.float32, False, True, False),
    (8, 2, 4096, 1, torch.bfloat16, torch.float32, False, True, False),
    (128, 8, 2048, 3, torch.bfloat16, torch.float32, False, True, True),
    (60, 4, 777, 17, torch.bfloat16, torch.bfloat16, False, False, True),
    (256, 8, 1030, 33, torch.float32, torch.float32, True, True, True),
    (257, 32, 96, 5, torch.float32, torch.bfloat16, True, False, True),
    (1024, 6, 512, 9, torch.bfloat16, torch.float32, True, True, False),
    (160, 6, 640, 700, torch.bfloat16, torch.float32, False, True, False),
    (256, 8, 5120, 512, torch.bfloat16, torch.float32, True, True, True),
])
def test_choice(backend, experts, top_k, k, m, x_dtype, w_dtype, sigmoid, normalise, biased):
    g = torch.Generator().manual_seed(experts + m)
    w = (torch.randn((experts, k), generator=g) * k ** -0.5).to(w_dtype)
    x = torch.randn((m, k), generator=g).to(x_dtype)
    logit_bias = torch.randn(experts, generator=g) if biased else None
    select = torch.randn(experts, generator=g) * 0.1 if biased and sigmoid else None
    r = backend.router(w, top_k, scoring=mb.SCORING_SIGMOID if sigmoid else mb.SCORING_SOFTMAX, normalise=normalise, scale=2.5, logit_bias=logit_bias,
                       select_bias=select, max_rows=m)
    ids, weights = backend.route(r, x.cuda())
    logits = x.double().numpy() @ w.double().numpy().T + (logit_bias.double().numpy() if biased else 0.0)
    want_ids, want = _want(logits, top_k, sigmoid, normalise, 2.5, select.double().numpy() if select is not None else 0.0)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    assert np.all(np.abs(weights.cpu().numpy() - want) <= 1e-6 * want)
