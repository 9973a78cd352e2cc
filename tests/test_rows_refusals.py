"""What expert layers, routers and adapter sets refuse, as far as that needs no GPU."""
import ctypes
from ctypes import byref, c_void_p

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import magnitude_b200 as mb  # noqa: E402
from magnitude_b200 import _binding as B  # noqa: E402
from magnitude_b200.rows import AdapterSet, MoeLayer, Router, Source, matrix  # noqa: E402

F32 = {torch.float32: B.TYPE_F32, torch.bfloat16: B.TYPE_BF16}


def _refused(text, call):
    with pytest.raises(mb.B200QError) as e:
        call()
    assert e.value.status == B.ERR_INVALID_CONFIG and text in str(e.value), str(e.value)


def test_entry_points_without_a_context():
    lib, out = B.lib(), c_void_p(1)
    assert lib.b200q_moe_create(None, byref(B.MoeConfig()), byref(out)) == B.ERR_INVALID_CONFIG
    assert lib.b200q_router_create(None, byref(B.RouterConfig()), byref(out)) == B.ERR_INVALID_CONFIG
    assert lib.b200q_adapters_create(None, 8, 8, B.TYPE_BF16, 1, 1, byref(out)) == B.ERR_INVALID_CONFIG
    assert lib.b200q_moe_run(None, None, None, 0, 1, 1, None, 1, None, 1, None, 0, 1, 0, None) == B.ERR_INVALID_CONFIG
    assert lib.b200q_router_run(None, None, None, 0, 1, 1, None, 1, None, 1, None) == B.ERR_INVALID_CONFIG
    assert lib.b200q_adapters_load(None, None, 0, 1, 1.0, None, None) == B.ERR_INVALID_CONFIG
    assert lib.b200q_adapters_apply(None, None, 1, None, 0, 1, 1, None, None, 0, None, None) == B.ERR_INVALID_CONFIG
    for destroy in (lib.b200q_moe_destroy, lib.b200q_router_destroy, lib.b200q_adapters_destroy):
        destroy(None)


def test_rows_of_a_call():
    ok = torch.zeros(3, 8)
    assert matrix(ok, "x", -1, 8, F32, 3) == (ok.data_ptr(), B.TYPE_F32, 8)
    assert matrix(torch.zeros(3, 12)[:, :8], "x", -1, 8, F32)[2] == 12
    assert matrix(torch.zeros(1, 12)[:, :8], "x", -1, 8, F32)[2] == 8           # one row has no stride to speak of
    _refused("on cpu, not on cuda:0", lambda: matrix(ok, "x", 0, 8, F32))
    _refused("torch.float64", lambda: matrix(ok.double(), "x", -1, 8, F32))
    _refused("shape (3, 8), not (rows, 9)", lambda: matrix(ok, "x", -1, 9, F32))
    _refused("shape (3, 8), not (4, 8)", lambda: matrix(ok, "x", -1, 8, F32, 4))
    _refused("shape (24,)", lambda: matrix(ok.flatten(), "x", -1, 8, F32))
    _refused("not contiguous", lambda: matrix(torch.zeros(8, 3).t(), "x", -1, 8, F32))
    _refused("overlap", lambda: matrix(torch.zeros(8).expand(3, 8), "x", -1, 8, F32))
    _refused("overlap", lambda: matrix(torch.zeros(40).as_strided((3, 8), (4, 1)), "x", -1, 8, F32))


def test_sources():
    assert Source(np.zeros((2, 3), np.uint8), "gate", "uint8").bytes == 6
    assert Source(torch.zeros(2, 3, dtype=torch.bfloat16), "a", "bfloat16").bytes == 12
    _refused("float64, not float32", lambda: Source(np.zeros(3), "gate_bias", "float32"))
    _refused("torch.int8, not uint8", lambda: Source(torch.zeros(3, dtype=torch.int8), "gate", "uint8"))
    _refused("list", lambda: Source([1, 2], "gate", "uint8"))


def _layer(gate=None, **other):
    blocks = np.zeros((2, 32, 34), np.uint8)         # two experts of 32 x 32, Q8_0
    args = dict(gate_up_type=mb.TYPE_Q8_0, down_type=mb.TYPE_Q8_0, top_k=1, n_embd=32, n_ff=32, max_rows=1, activation=0, alpha=0.0, limit=0.0,
                gate_bias=None, up_bias=None, down_bias=None)
    return MoeLayer(None, blocks if gate is None else gate, blocks, blocks, **{**args, **other})


def test_layers_and_routers():
    _refused("no whole number of experts", lambda: _layer(np.zeros(34 * 32 * 2 - 1, np.uint8)))
    _refused("no whole number of experts", lambda: _layer(gate_up_type=99))
    _refused("no whole number of experts", lambda: _layer(n_embd=31))
    _refused("gate_bias has shape (2, 31)", lambda: _layer(gate_bias=np.zeros((2, 31), np.float32)))
    _refused("down_bias is int32", lambda: _layer(down_bias=np.zeros((2, 32), np.int32)))
    args = dict(scoring=0, normalise=True, scale=1.0, logit_bias=None, select_bias=None, max_rows=1)
    _refused("not (experts, n_embd)", lambda: Router(None, np.zeros(8, np.float32), 1, **args))
    _refused("not float32", lambda: Router(None, np.zeros((4, 8)), 1, **args))
    _refused("logit_bias has shape (5,)", lambda: Router(None, np.zeros((4, 8), np.float32), 1, **{**args, "logit_bias": np.zeros(5, np.float32)}))
    _refused("not float16 or bfloat16", lambda: AdapterSet(None, 8, 8, torch.float32, 1, 1))


def test_config_structs_match_the_header():
    # field order and widths as a C compiler lays them out: eight-byte fields are aligned, no holes but those named here
    assert ctypes.sizeof(B.MoeConfig) == 2 * 4 + 3 * 8 + 2 * 4 + 9 * 8 + 4 * 4
    assert ctypes.sizeof(B.RouterConfig) == 2 * 4 + 2 * 8 + 4 * 4 + 3 * 8 + 4 + 4
