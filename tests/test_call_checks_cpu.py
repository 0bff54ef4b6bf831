"""Checks that the 8-bit cache and sink methods make of their arguments before the library is called: devices and types.

Host only: the tensors say that they are on the handle's device, and the library behind the handle is a stand-in that counts."""
import pytest
import torch

F16, U32, ADDR = "f16", "u32", "addr"
# the tensors of each call, in order; "layout" is the paged layout
CALLS = {
    "append_q8": ([F16] * 8 + [U32, "q8", U32], ()),
    "decode_attn_q8": ([F16] * 3 + ["q8", U32], ()),
    "prefill_attn_q8": ([F16] * 3 + ["q8", U32, U32], ()),
    "decode_attn_sinks": ([F16] * 3 + [ADDR, ADDR, U32], (4, 2)),
    "decode_attn_paged_sinks": ([F16] * 3 + ["paged", U32], (4, 2)),
    "append_decode_sinks": ([F16] * 9 + [U32, U32, ADDR, ADDR], (4, 2)),
    "append_decode_paged_sinks": ([F16] * 9 + [U32, "paged"], (4, 2)),
    "prefill_attn_sinks": ([F16] * 3 + [ADDR, ADDR, U32], (4, 2)),
    "prefill_attn_paged_sinks": ([F16] * 3 + ["paged", U32, U32], (4, 2)),
}
DTYPE = {F16: torch.float16, U32: torch.int32, ADDR: torch.int64}


class _Near(torch.Tensor):
    """Says that it is on the handle's device."""
    def get_device(self):
        return 0


class _Library:
    def __init__(self):
        self.called = 0

    def __getattr__(self, name):
        def call(*a):
            self.called += 1
            return 0
        return call


def _layout(kind, device):
    from oxide_infer_b200 import PagedLayout, PagedQ8Layout
    table = torch.zeros(2, 3, dtype=torch.int32)
    if kind == "q8":
        lay = PagedQ8Layout.of(*(torch.zeros(5, 16, 4, 128, dtype=torch.int8) for _ in range(2)), *(torch.zeros(5, 4) for _ in range(2)), table)
    else:
        lay = PagedLayout.of(*(torch.zeros(5, 16, 4, 128, dtype=torch.float16) for _ in range(2)), table, 16)
    assert lay.device == -1  # host tensors
    lay.device = device
    return lay


def _call(name, change=None, value=None):
    """Calls the method with sound arguments, the one at `change` replaced; returns how often the library was called."""
    from oxide_infer_b200 import KvPath
    kinds, rest = CALLS[name]
    kv = KvPath.__new__(KvPath)
    kv.device, kv.lib, kv.h = 0, _Library(), None
    kv._stream = lambda: 0
    near = lambda dt: torch.zeros(1, 16, 128, dtype=dt).as_subclass(_Near)  # noqa: E731
    args = [_layout(k, 0) if k in ("q8", "paged") else near(DTYPE[k]) for k in kinds]
    if change is not None:
        args[change] = value
    getattr(kv, name)(*args, *rest)
    return kv.lib.called


@pytest.mark.parametrize("name", list(CALLS))
def test_sound_arguments_reach_the_library(name):
    assert _call(name) == 1


@pytest.mark.parametrize("name", [n for n, (kinds, _) in CALLS.items() if {"q8", "paged"} & set(kinds)])
def test_a_layout_on_another_device_is_refused(name):
    at = [i for i, k in enumerate(CALLS[name][0]) if k in ("q8", "paged")][0]
    for device in (-1, 1):
        with pytest.raises(ValueError, match="device"):
            _call(name, at, _layout(CALLS[name][0][at], device))


@pytest.mark.parametrize("name", list(CALLS))
def test_a_tensor_of_another_type_is_refused(name):
    """An int64 length, position or row would be read as two."""
    wrong = {F16: torch.bfloat16, U32: torch.int64, ADDR: torch.int32}
    for i, kind in enumerate(CALLS[name][0]):
        if kind in wrong:
            with pytest.raises(ValueError, match="a tensor is"):
                _call(name, i, torch.zeros(1, 16, 128, dtype=wrong[kind]).as_subclass(_Near))


def test_the_paged_layout_refuses_tables_of_another_type_and_tensors_apart():
    from oxide_infer_b200 import PagedLayout
    pools = [torch.zeros(5, 16, 4, 128, dtype=torch.float16) for _ in range(2)]
    table = torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(ValueError, match="int32"):
        PagedLayout.of(*pools, table.long(), 16)
    for i in range(3):
        parts = [*pools, table]
        parts[i] = parts[i].to("meta")
        with pytest.raises(ValueError, match="one device"):
            PagedLayout.of(*parts, 16)
