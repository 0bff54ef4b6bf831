"""Host-only checks of the 8-bit cache and sink entry points: null handles, the layout's checks, its C form."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from oxide_infer_b200 import build, _lib
    build.build()
    return _lib.load()


def test_null_handles_are_refused_before_cuda_is_touched(lib):
    n = None
    assert lib.oxi_append_q8(n, *([n] * 12), 1, 1e-5) == -1
    assert lib.oxi_decode_attn_q8(n, *([n] * 6), 1, 0, 0) == -1
    assert lib.oxi_prefill_attn_q8(n, *([n] * 7), 1, 0, 0) == -1
    for window, sinks in ((0, 0), (5, 2)):
        assert lib.oxi_decode_attn_sinks(n, *([n] * 7), 1, window, sinks) == -1
        assert lib.oxi_decode_attn_paged_sinks(n, *([n] * 6), 1, window, sinks) == -1
        assert lib.oxi_append_decode_sinks(n, *([n] * 14), 1, window, sinks, 1e-5) == -1
        assert lib.oxi_append_decode_paged_sinks(n, *([n] * 12), 1, window, sinks, 1e-5) == -1
        assert lib.oxi_prefill_attn_sinks(n, *([n] * 7), 1, window, sinks) == -1
        assert lib.oxi_prefill_attn_paged_sinks(n, *([n] * 7), 1, window, sinks) == -1


def _parts(dtype=torch.int8):
    return [torch.zeros(5, 16, 4, 128, dtype=dtype), torch.zeros(5, 16, 4, 128, dtype=dtype), torch.zeros(5, 4), torch.zeros(5, 4),
            torch.zeros(2, 3, dtype=torch.int32)]


def test_layout_fields():
    from oxide_infer_b200 import PagedQ8Layout
    assert C.sizeof(PagedQ8Layout) == 5 * 8 + 2 * 8 + 5 * 4 + 4  # 4 bytes of padding
    p = _parts()
    lay = PagedQ8Layout.of(*p)
    assert (lay.k_pool, lay.v_scales, lay.block_tables) == (p[0].data_ptr(), p[3].data_ptr(), p[4].data_ptr())
    assert (lay.block_stride_bytes, lay.scale_stride) == (16 * 512, 4)
    assert (lay.max_blocks, lay.block_size, lay.num_blocks, lay.format, lay.table_rows) == (3, 16, 5, 0, 2)
    assert PagedQ8Layout.of(*_parts(torch.float8_e4m3fn)).format == 1
    wide = [torch.zeros(5, 2, 16, 4, 128, dtype=torch.int8) for _ in range(2)]
    lay = PagedQ8Layout.of(wide[0][:, 0], wide[1][:, 1], *_parts()[2:])
    assert lay.block_stride_bytes == 2 * 16 * 512 and lay.v_pool == wide[1].data_ptr() + 16 * 512


@pytest.mark.parametrize("change", [
    lambda p: p.__setitem__(0, p[0].half()),
    lambda p: p.__setitem__(1, p[1].to(torch.float8_e4m3fn)),
    lambda p: p.__setitem__(0, p[0].transpose(1, 2)),
    lambda p: p.__setitem__(1, p[1][:4]),
    lambda p: p.__setitem__(0, p[0].view(5, 16, 8, 64)),
    lambda p: p.__setitem__(2, p[2].double()),
    lambda p: p.__setitem__(3, torch.zeros(4, 5).t()),
    lambda p: p.__setitem__(2, torch.zeros(5, 8)[:, :4]),
    lambda p: p.__setitem__(4, p[4].long()),
    lambda p: p.__setitem__(4, torch.zeros(3, 2, dtype=torch.int32).t()),
    lambda p: p.__setitem__(4, p[4].to("meta")),
])
def test_layout_refuses_tensors_of_another_form(change):
    from oxide_infer_b200 import PagedQ8Layout
    p = _parts()
    change(p)
    with pytest.raises(ValueError):
        PagedQ8Layout.of(*p)


def test_tensors_on_another_device_than_the_handle_are_refused():
    """Before anything is called: a handle without a library behind it, host tensors, a layout of host tensors."""
    from oxide_infer_b200 import KvPath, PagedQ8Layout

    class Somewhere(torch.Tensor):
        """Says that it is on the handle's device."""
        def get_device(self):
            return 0

    kv = KvPath.__new__(KvPath)
    kv.device, kv.lib, kv.h = 0, None, None
    kv._stream = lambda: 0
    there = lambda: torch.zeros(1, 16, 128).as_subclass(Somewhere)  # noqa: E731
    here = torch.zeros(1, 16, 128)
    lay = PagedQ8Layout.of(*_parts())
    near = PagedQ8Layout.of(*_parts())
    near.device = 0
    assert lay.device == -1

    class _Refuses:
        def __getattr__(self, name):
            def call(*a):
                raise AssertionError("called")
            return call

    def refused(name, n, layout_at, rest):
        fn = getattr(kv, name)
        for bad in range(n):
            args = [here if i == bad else near if i == layout_at else there() for i in range(n)]
            if bad == layout_at:
                if name.endswith("q8"):
                    args[bad] = lay
                else:
                    continue
            kv.lib = _Refuses()
            with pytest.raises(ValueError):
                fn(*args, *rest)

    refused("append_q8", 11, 9, ())
    refused("decode_attn_q8", 5, 3, ())
    refused("prefill_attn_q8", 6, 3, ())
    refused("decode_attn_sinks", 6, None, (4, 2))
    refused("decode_attn_paged_sinks", 5, 3, (4, 2))
    refused("append_decode_sinks", 13, None, (4, 2))
    refused("append_decode_paged_sinks", 11, 10, (4, 2))
    refused("prefill_attn_sinks", 6, None, (4, 2))
    refused("prefill_attn_paged_sinks", 6, 3, (4, 2))
