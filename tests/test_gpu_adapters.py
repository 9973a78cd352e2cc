"""Low-rank adapters (b200q_adapters_apply) against y + scale * B (A x) in 64 bits.

Tolerances.  Products are exact and sums fp32: t = A x of K terms errs by about sqrt(K) 2^-24 of its root mean square, B t of at
most 256 more likewise; with K up to 5000 that is 70 * 6e-8 = 4.2e-6 of the root mean square r of the row's change, and the largest of some ten
thousand results may be five times that: 2e-5 r, and y's own rounding of the final sum, 2^-24 |y|.  With bf16 outputs t enters as two bf16
planes: truncation to 8 bits leaves less than 2^-7 of an element, of which rounding to 8 bits loses at most 2^-8: 2^-15 of each of its
elements, a third of that on average, and 2^-14 r for the largest of the results; and the result is rounded once, by at most half a step,
2^-8 of its value (8 significant bits)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import magnitude_b200 as mb  # noqa: E402

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


class Set:
    def __init__(self, backend, n, k, ranks, dtype, max_rank, seed, slots=None):
        g = torch.Generator().manual_seed(seed)
        self.handle = backend.adapters(n, k, dtype, max_adapters=slots or len(ranks), max_rank=max_rank)
        self.parts = []
        for i, r in enumerate(ranks):
            if r == 0:
                self.parts.append(None)
                continue
            a, b = (torch.randn((r, k), generator=g) * k ** -0.5).to(dtype), torch.randn((n, r), generator=g).to(dtype)
            scale = 0.5 + i
            self.handle.load(i, a.cuda() if i % 2 else a, b.cuda() if i % 2 else b, scale)
            self.parts.append((a.double(), b.double(), scale))

    def want(self, x, slots, y):
        x, y = x.cpu().double(), y.cpu().double().clone()
        change = torch.zeros_like(y)
        for m, s in enumerate(slots.tolist()):
            if 0 <= s < len(self.parts) and self.parts[s] is not None:
                a, b, scale = self.parts[s]
                change[m] = scale * (b @ (a @ x[m]))
        return y + change, change


def _check(got, want, change, slots, before):
    got = got.cpu()
    r = change.square().mean(dim=1, keepdim=True).sqrt()
    err = (got.double() - want).abs()
    bound = 2.0 ** -8 * want.abs() + 2.0 ** -14 * r if got.dtype == BF16 else 2.0 ** -24 * want.abs() + 2e-5 * r
    idle = r.flatten() == 0
    assert torch.equal(got[idle], before.cpu()[idle]), "a row without an adapter changed"
    assert bool((err <= bound)[~idle].all()), f"worst error / bound {(err / bound)[~idle].max():.2f}"


def _run(backend, m, k, ns, ranks, dtype, x_dtype, y_dtype, slots, max_rank, seed=0, ld_pad=0):
    g = torch.Generator().manual_seed(seed)
    sets = [Set(backend, n, k, ranks, dtype, max_rank, seed + i) for i, n in enumerate(ns)]
    x = torch.randn((m, k + ld_pad), generator=g).to(x_dtype).cuda()[:, :k]
    ys = [torch.randn((m, n + ld_pad), generator=g).to(y_dtype).cuda()[:, :n] for n in ns]
    before = [y.clone() for y in ys]
    slots = torch.tensor(slots, dtype=torch.int32, device="cuda")
    backend.apply_adapters([s.handle for s in sets], x, slots, ys)
    torch.cuda.synchronize()
    for s, y, b in zip(sets, ys, before):
        _check(y, *s.want(x, slots, b), slots, b)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("x_dtype", [BF16, F32])
@pytest.mark.parametrize("y_dtype", [BF16, F32])
@pytest.mark.parametrize("m", [1, 5, 700])
def test_types(backend, dtype, x_dtype, y_dtype, m):
    slots = [(7 * i) % 4 - 1 for i in range(m)] if m <= 5 else [i // 180 - 1 for i in range(m)]
    _run(backend, m, 1024, [768], [16, 8, 40], dtype, x_dtype, y_dtype, [0] if m == 1 else slots, 40)


@pytest.mark.parametrize("m,k,ns,ranks,slots,max_rank,ld_pad", [
    (1, 1, [1], [1], [0], 1, 0),
    (3, 33, [17, 5], [3, 1], [1, 0, 1], 5, 0),                                          # nothing is a multiple of anything
    (2, 4096, [4096, 1024, 1024], [16, 64], [1, 0], 64, 0),
    (4, 520, [264], [256, 130, 72, 65], [0, 1, 2, 3], 256, 0),                          # ranks of several blocks of 64
    (40, 320, [96], [8], [0] * 40, 8, 0),                                               # more rows of an adapter than a cluster takes
    (64, 256, [128], [4] * 64, list(range(63, -1, -1)), 4, 0),                           # every row its own
    (20, 256, [128], [4, 0, 12], [0, 1, 2, -1, 3, -7, 2 ** 31 - 1, -2 ** 31] + [2] * 12, 16, 0),   # empty, missing and absurd slots
    (6, 512, [96, 48], [24, 8], [0, 1, 0, -1, 1, 1], 24, 3),                             # rows that are not 16-byte aligned
    (600, 256, [300], [16, 32, 8], [i % 4 - 1 for i in range(600)], 32, 0),              # every tile of rows has every adapter
    (513, 1000, [200], [200], [0] * 513, 200, 8),
])
@pytest.mark.parametrize("x_dtype,y_dtype", [(BF16, BF16), (F32, F32)])
def test_shapes(backend, m, k, ns, ranks, slots, max_rank, ld_pad, x_dtype, y_dtype):
    _run(backend, m, k, ns, ranks, BF16, x_dtype, y_dtype, slots, max_rank, seed=m, ld_pad=ld_pad)
