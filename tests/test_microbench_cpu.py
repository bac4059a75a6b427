"""The step benchmark's lines, with the library and the device taken away."""
import types

import numpy as np

from system1_omni_b200 import microbench as M


class Buffer:
    def __init__(self, nbytes=16):
        self.ptr = types.SimpleNamespace(value=1 << 20)


class Library:
    def __getattr__(self, name):
        return lambda *a: 1 if name.endswith("floats") else 0


def test_step_lines_say_what_their_fraction_is_of(monkeypatch):
    monkeypatch.setattr(M.L, "DeviceBuffer", Buffer)
    monkeypatch.setattr(M.L, "to_device", lambda a, stream, offset_elems=0: Buffer())
    bench = types.SimpleNamespace(lib=Library(), stream=types.SimpleNamespace(handle=types.SimpleNamespace(value=0)),
                                  copies=lambda nbytes: 1, bf16=lambda n, scale=1.0: Buffer(), time=lambda call, copies: call(0) or 10.0)
    lines = []
    M.step(bench, lines.append)
    hbm, _, source = M.peaks()
    assert {line["op"] for line in lines} == {"gdn_step", "gdn_conv_gates_step", "attn_prep_paged", "attention_paged", "fork_states", "fork_pages"}
    for line in lines:
        assert line["peak"] == source and line["peak"] in ("measured", "fallback")
        assert abs(line["fraction"] - line["gb_s"] / hbm) < 1e-3
    assert np.isfinite([line["gb_s"] for line in lines]).all()
