"""Layers of experts in the packed file (mbp.store): their columns are in another order than a plain layer's, so a reader
that does not know them has to refuse the file."""
import json
import struct

import pytest
import torch

from mbp import store
from mbp.epilogue import PackedExperts
from test_store_cpu import _c12_state


def _experts_state(experts=4):
    _, _, st = _c12_state(seed=2)
    st["experts"] = {"up": PackedExperts(_c12_state(seed=3)[2]["layers"]["o"], experts)}
    st["k"]["up"] = 256
    return st


def _header(path):
    data = path.read_bytes()
    (n,) = struct.unpack("<Q", data[8:16])
    return json.loads(data[16:16 + n]), n, data


def _rewrite(path, change):
    header, n, data = _header(path)
    change(header)
    text = json.dumps(header, separators=(",", ":")).encode()
    assert len(text) <= n
    path.write_bytes(data[:16] + text + b" " * (n - len(text)) + data[16 + n:])


def test_only_files_with_experts_are_of_the_newer_version(tmp_path):
    plain, with_experts = tmp_path / "a.mbp", tmp_path / "b.mbp"
    store.save_packed(_c12_state()[2], str(plain), {"o": "a", "router": "b"}, base_mode=1)
    store.save_packed(_experts_state(), str(with_experts), {"o": "a", "router": "b", "up": "c"}, base_mode=1)
    assert _header(plain)[0]["version"] == 1      # what builds without experts read ...
    assert _header(with_experts)[0]["version"] == 2  # ... and what they refuse
    back = store.load_packed(str(with_experts), device="cpu")
    a, b = _experts_state()["experts"]["up"], back["experts"]["up"]
    assert (b.experts, b.n, b.k) == (4, 16, 256) and set(back["layers"]) == {"o"} and back["k"]["up"] == 256
    for name in ("units", "bases", "esc_off", "esc"):
        assert torch.equal(getattr(a.packed, name), getattr(b.packed, name)), name
    assert store.matches(str(with_experts), {"o": "a", "router": "b", "up": "c"}, 1)
    assert not store.matches(str(with_experts), {"o": "a", "router": "b", "up": "c"}, 0)
    _rewrite(plain, lambda h: h.update(version=3))
    with pytest.raises(ValueError):
        store.load_packed(str(plain), device="cpu")


def test_files_with_experts_of_the_first_form_are_read(tmp_path):
    """Version 1 with an "experts" entry: the only form before the version said so."""
    path = tmp_path / "w.mbp"
    store.save_packed(_experts_state(), str(path), {}, base_mode=1)
    _rewrite(path, lambda h: h.update(version=1))
    assert store.load_packed(str(path), device="cpu")["experts"]["up"].experts == 4


@pytest.mark.parametrize("experts", [3, 8, 5000, -4, "4", 2.0, True])
def test_a_number_of_experts_that_does_not_divide_the_rows_is_refused(tmp_path, experts):
    """64 rows: 8 experts would have 8 rows each, which is no whole tile of 16."""
    path = tmp_path / "w.mbp"
    fps = {"o": "a", "router": "b", "up": "c"}
    store.save_packed(_experts_state(), str(path), fps, base_mode=1)
    _rewrite(path, lambda h: h["layers"]["up"].update(experts=experts))
    with pytest.raises(ValueError):
        store.load_packed(str(path), device="cpu")
    assert not store.matches(str(path), fps, 1)  # prepare packs again
