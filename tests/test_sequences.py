"""The token-sequence operators without a GPU: their descs' layouts, the queries and every
refusal that needs no device."""

import ctypes
import os
import subprocess

import pytest

from eagle_b200 import _abi

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "eagle_b200.h")


@pytest.mark.parametrize("cname,ct", [("eagle_b200_embedding_desc", _abi.EmbeddingDesc),
                                      ("eagle_b200_paged_desc", _abi.PagedDesc)])
def test_layouts_match_the_header(tmp_path, cname, ct):
    lines = ['#include <stddef.h>', '#include <stdio.h>', f'#include "{HEADER}"', "int main(void) {",
             f'printf("%zu\\n", sizeof(struct {cname}));']
    lines += [f'printf("%zu\\n", offsetof(struct {cname}, {name}));' for name, _ in ct._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(exe), str(src)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(ct)] + [getattr(ct, name).offset for name, _ in ct._fields_]


def _embedding(**fields):
    d = _abi.new(_abi.EmbeddingDesc, table_type=_abi.TYPE_BF16, values_type=_abi.TYPE_BF16, token_type=_abi.TYPE_I64,
                 table=1 << 20, tokens=1 << 20, values=1 << 20, rows=100, dim=64, batch=2, seq=8, table_stride=64,
                 scale=1.0)
    d.token_strides[:] = [8, 1]
    d.value_strides[:] = [512, 64, 1]
    for k, v in fields.items():
        setattr(d, k, v)
    return d


def _paged(**fields):
    d = _abi.new(_abi.PagedDesc, length_type=_abi.TYPE_I32, slot_type=_abi.TYPE_I64, requests=4, width=8,
                 table_stride=8, block=16, pool_size=64, used_size=64, capacity=32)
    for name in ("table", "lengths", "held", "pool", "count", "used", "blocks", "cells", "start", "fresh", "slots",
                 "positions", "token_requests", "offsets"):
        setattr(d, name, (1 << 20) + 4096 * (1 + len(name)))
    for k, v in fields.items():
        setattr(d, k, v)
    return d


BAD_EMBEDDING = [
    (dict(table_type=9), _abi.UNSUPPORTED), (dict(values_type=_abi.TYPE_I32), _abi.UNSUPPORTED),
    (dict(token_type=_abi.TYPE_F32), _abi.UNSUPPORTED), (dict(flags=2), _abi.UNSUPPORTED),
    (dict(rows=-1), _abi.INVALID_ARGUMENT), (dict(rows=2**31 - 1), _abi.INVALID_ARGUMENT),
    (dict(dim=-1), _abi.INVALID_ARGUMENT), (dict(dim=2**24 + 1), _abi.INVALID_ARGUMENT),
    (dict(first=-1), _abi.INVALID_ARGUMENT), (dict(batch=-1), _abi.INVALID_ARGUMENT),
    (dict(batch=2**16, seq=2**16), _abi.INVALID_ARGUMENT), (dict(batch=2**40, seq=2**40), _abi.INVALID_ARGUMENT),
    (dict(table_stride=63), _abi.INVALID_ARGUMENT),
]


@pytest.mark.parametrize("fields,status", BAD_EMBEDDING)
@pytest.mark.parametrize("entry", ["embedding", "embedding_grad"])
def test_embedding_refuses(entry, fields, status):
    d = _embedding(**fields)
    assert getattr(_abi.lib(), "eagle_backend_x_b200_" + entry)(ctypes.byref(d)) == status
    assert entry in _abi.last_error()


def test_embedding_refuses_accumulate_and_a_short_desc():
    d = _embedding(flags=_abi.EMBEDDING_ACCUMULATE)
    assert _abi.lib().eagle_backend_x_b200_embedding(ctypes.byref(d)) == _abi.UNSUPPORTED
    d = _embedding(struct_size=ctypes.sizeof(_abi.EmbeddingDesc) - 8)
    assert _abi.lib().eagle_backend_x_b200_embedding_grad(ctypes.byref(d)) == _abi.INVALID_ARGUMENT


def test_embedding_calls_without_work_need_no_device():
    for fields in (dict(batch=0), dict(seq=0), dict(dim=0, table_stride=0)):
        d = _embedding(**fields)
        assert _abi.lib().eagle_backend_x_b200_embedding(ctypes.byref(d)) == _abi.OK


def test_gradient_query_depends_on_sizes_alone():
    def ask(**fields):
        d = _embedding(**fields)
        assert _abi.lib().eagle_backend_x_b200_embedding_grad(ctypes.byref(d)) == _abi.OK
        return d.scratch_bytes

    base = ask(batch=64, seq=1024, rows=5000)
    assert base % 256 == 0 and base > 64 * 1024 * 16
    for other in (dict(table=(1 << 20) + 2), dict(values=(1 << 20) + 2), dict(table_type=_abi.TYPE_F32),
                  dict(values_type=_abi.TYPE_F32), dict(token_type=_abi.TYPE_I32), dict(table_stride=65),
                  dict(flags=_abi.EMBEDDING_ACCUMULATE)):
        assert ask(batch=64, seq=1024, rows=5000, **other) == base, other
    assert ask(batch=64, seq=2048, rows=5000) > base


BAD_PAGED = [
    (dict(length_type=_abi.TYPE_F32), _abi.UNSUPPORTED), (dict(flags=1), _abi.UNSUPPORTED),
    (dict(reserved0=1), _abi.INVALID_ARGUMENT), (dict(requests=-1), _abi.INVALID_ARGUMENT),
    (dict(requests=2**20 + 1), _abi.INVALID_ARGUMENT), (dict(block=0), _abi.INVALID_ARGUMENT),
    (dict(block=2**31), _abi.INVALID_ARGUMENT), (dict(width=-1), _abi.INVALID_ARGUMENT),
    (dict(width=2**27, table_stride=2**27), _abi.INVALID_ARGUMENT), (dict(table_stride=7), _abi.INVALID_ARGUMENT),
]


@pytest.mark.parametrize("fields,status", BAD_PAGED)
@pytest.mark.parametrize("entry", ["block_tables", "slot_map"])
def test_paged_refuses(entry, fields, status):
    d = _paged(**fields)
    assert getattr(_abi.lib(), "eagle_backend_x_b200_" + entry)(ctypes.byref(d)) == status
    assert entry in _abi.last_error()


@pytest.mark.parametrize("entry,fields,status", [
    ("block_tables", dict(pool_size=-1), _abi.INVALID_ARGUMENT),
    ("block_tables", dict(pool_size=2**31 - 1), _abi.INVALID_ARGUMENT),
    ("block_tables", dict(used_size=-1), _abi.INVALID_ARGUMENT),
    ("block_tables", dict(scratch=1 << 20, count=0), _abi.INVALID_ARGUMENT),
    ("block_tables", dict(scratch=1 << 20, held=0), _abi.INVALID_ARGUMENT),
    ("block_tables", dict(scratch=1 << 20, lengths=(1 << 20) + 2), _abi.INVALID_ARGUMENT),
    ("block_tables", dict(scratch=1 << 20, blocks=1 << 21, held=1 << 21), _abi.INVALID_ARGUMENT),
    ("block_tables", dict(scratch=8), _abi.INVALID_ARGUMENT),
    ("slot_map", dict(slot_type=_abi.TYPE_BF16), _abi.UNSUPPORTED),
    ("slot_map", dict(capacity=-1), _abi.INVALID_ARGUMENT),
    ("slot_map", dict(capacity=2**31 - 1), _abi.INVALID_ARGUMENT),
    ("slot_map", dict(scratch=1 << 20, slots=(1 << 20) + 8), _abi.INVALID_ARGUMENT),
    ("slot_map", dict(scratch=1 << 20, offsets=0), _abi.INVALID_ARGUMENT),
    ("slot_map", dict(scratch=1 << 20, length_type=_abi.TYPE_I64, start=(1 << 20) + 4), _abi.INVALID_ARGUMENT),
])
def test_paged_refuses_its_own(entry, fields, status):
    d = _paged(**fields)
    assert getattr(_abi.lib(), "eagle_backend_x_b200_" + entry)(ctypes.byref(d)) == status


def test_paged_queries():
    for entry in ("block_tables", "slot_map"):
        for requests, least in ((0, 0), (4, 0), (2048, 0), (8193, 4 * 8193), (2**20, 4 * 2**20)):
            d = _paged(requests=requests)
            assert getattr(_abi.lib(), "eagle_backend_x_b200_" + entry)(ctypes.byref(d)) == _abi.OK
            assert d.scratch_bytes >= max(least, 16)


def test_host_tensors_are_refused(eb):
    table, ids = torch.zeros(4, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA tensor"):
        eb.embedding(table, ids)
    with pytest.raises(ValueError, match="CUDA tensor"):
        eb.embedding_grad(torch.zeros(3, 8), ids, 4)
    tables = torch.zeros(2, 4, dtype=torch.int32)
    lengths = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensor"):
        eb.block_tables(lengths, lengths, tables, lengths, lengths[:1], block=16)
    with pytest.raises(ValueError, match="CUDA tensor"):
        eb.slot_map(tables, lengths, lengths, 8, block=16)


@pytest.mark.parametrize("fields,polls", [
    (dict(batch=0), 100), (dict(rows=0), 100), (dict(dim=0, table_stride=0), 100),
    (dict(), 100),  # 128 bytes a row: read without the copy engine
    (dict(dim=1024, table_stride=1024), 0), (dict(dim=1024, table_stride=1024), 2**22 + 1),
    (dict(dim=1024, table_stride=1024, scratch=0), 100), (dict(dim=1024, table_stride=1024, first=-1), 100),
])
def test_gradient_wait_check_refuses(fields, polls):
    d = _embedding(**{"scratch": 1 << 20, **fields})
    d.value_strides[:] = [8 * d.dim, d.dim, 1]
    entry = _abi.lib().eagle_backend_x_b200_embedding_grad_wait_check
    assert entry(ctypes.byref(d), polls, 1) == _abi.INVALID_ARGUMENT
    assert "wait_check" in _abi.last_error()


@pytest.mark.parametrize("entry,fields,status", [
    ("slot_map", dict(flags=_abi.SLOT_MAP_HELD, scratch=1 << 20, held=0), _abi.INVALID_ARGUMENT),
    ("slot_map", dict(flags=_abi.SLOT_MAP_HELD, scratch=1 << 20, held=(1 << 20) + 2), _abi.INVALID_ARGUMENT),
    ("slot_map", dict(flags=4), _abi.UNSUPPORTED),
    ("block_tables", dict(flags=_abi.SLOT_MAP_HELD), _abi.UNSUPPORTED),
])
def test_slot_map_held_refuses(entry, fields, status):
    d = _paged(**fields)
    assert getattr(_abi.lib(), "eagle_backend_x_b200_" + entry)(ctypes.byref(d)) == status


def _offsets(shape, strides):
    grid = torch.zeros(tuple(shape), dtype=torch.int64)
    for axis, (n, s) in enumerate(zip(shape, strides)):
        grid += (torch.arange(n) * s).view([-1 if a == axis else 1 for a in range(len(shape))])
    return grid.flatten()


def test_axes_join_wherever_one_stride_serves_them():
    """Any number of axes, as long as they make two of one stride each; which ones join does not matter."""
    from eagle_b200._sequences import _axes

    ids = torch.arange(2 * 3 * 4 * 5)
    vectors = torch.zeros(120, 7)
    wide = torch.zeros(3, 40, 9)[:, :20, 1:8]
    for tokens, values in (
            (ids[0], vectors[0]), (ids, vectors), (ids.view(24, 5), vectors.view(24, 5, 7)),
            (ids.view(24, 5).t(), vectors.view(5, 24, 7)), (ids[:1].view(1, 1, 1), vectors[:1].view(1, 1, 1, 7)),
            (ids.view(2, 3, 4, 5), vectors.view(2, 3, 4, 5, 7)), (ids.view(12, 1, 10), vectors.view(12, 1, 10, 7)),
            # the last two axes join and the first two do not, and the other way round
            (ids.view(40, 3).t().view(3, 8, 5), vectors.view(3, 8, 5, 7)),
            (ids.view(24, 5)[:, :4].unflatten(0, (4, 6)), vectors[:96].view(4, 6, 4, 7)),
            (ids[:60].view(3, 4, 5), wide.unflatten(1, (4, 5))), (ids[:8].expand(5, 3, 8), vectors.view(5, 3, 8, 7)),
            (ids.view(2, 60)[:0], vectors.view(2, 60, 7)[:0]), (ids.view(2, 3, 20)[:, :0], vectors.view(2, 3, 20, 7)[:, :0]),
            (ids.view(2, 3, 20).transpose(0, 2)[:0], vectors.view(20, 3, 2, 7)[:0])):
        shape, at, to = _axes(tokens, values)
        assert len(shape) == len(at) == len(to) == 2 and shape[0] * shape[1] == tokens.numel()
        assert torch.equal(_offsets(shape, at), _offsets(tokens.shape, tokens.stride()))
        assert torch.equal(_offsets(shape, to), _offsets(tokens.shape, values.stride()[:-1]))
    for tokens, values in ((ids.view(5, 4, 6).transpose(0, 2), vectors.view(6, 4, 5, 7)),
                           (ids.view(24, 5)[:, :4].unflatten(0, (4, 6)), vectors.view(4, 30, 7)[:, :24].unflatten(1, (6, 4)))):
        with pytest.raises(ValueError, match="join"):
            _axes(tokens, values)


def test_planes_apart():
    """What shares no element is apart, columns of one plane too; whatever does share one is refused."""
    from eagle_b200._sequences import _apart

    plane = torch.zeros(12, 40)
    flat = plane.view(-1)

    def places(x):
        first = (x.data_ptr() - plane.data_ptr()) // 4
        each = x.element_size() // 4
        return {int(first + o * each + i) for o in _offsets(x.shape, x.stride()) for i in range(each)}

    views = [plane[:, :16], plane[:, 16:40], plane[:, 15:17], plane[3:5], plane[:, 3], plane[::2, 20:30], plane[1::2, 20:30],
             flat[40:56], flat[100:101], flat[7], plane[:, :20].unflatten(1, (4, 5))[..., :3],
             plane[:, :20].unflatten(1, (4, 5))[..., 3:], plane[:1, :8].expand(5, 8), plane[:, 30:].t(), plane[:0],
             plane.view(torch.int64)[:, 8:12], flat.as_strided((3, 2, 4), (80, 20, 1)), flat.as_strided((3, 4), (80, 2), 41)]
    beside = 0
    for out in views:
        for x in views:
            try:
                _apart(out, "out", x)
            except ValueError:
                continue
            assert not places(out) & places(x)
            beside += 1
    assert beside > len(views)
    for out, x in ((plane[:, :16], plane[:, 16:40]), (plane[:, 16:40], plane[:, :16]), (plane[:, 3], plane[:, 4:9]),
                   (plane[:, :20].unflatten(1, (4, 5))[..., :3], plane[:, :20].unflatten(1, (4, 5))[..., 3:])):
        _apart(out, "out", x)
    with pytest.raises(ValueError, match="overlaps"):
        _apart(plane[:, :16], "out", None, plane[:, 15:])


def test_tangents_are_refused():
    """A dual tensor's tangent would be lost without a word."""
    from torch.autograd import forward_ad

    from eagle_b200._sequences import _no_grad

    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.zeros(3, 4), torch.ones(3, 4))
        for grad in (False, True):
            with torch.set_grad_enabled(grad):
                with pytest.raises(ValueError, match="tangent"):
                    _no_grad("embedding", None, dual)
                _no_grad("embedding", torch.zeros(3, 4), None)
                _no_grad("embedding", forward_ad.unpack_dual(dual).primal)
    _no_grad("embedding", torch.zeros(3, 4))


def test_negated_views_are_refused():
    """The imaginary part of a conjugate is a float32 view of memory that holds its negatives."""
    from eagle_b200._sequences import _plain

    view = torch.randn(4, 1, dtype=torch.complex64).conj().imag
    assert view.dtype == torch.float32 and view.is_neg()
    with pytest.raises(ValueError, match="negates"):
        _plain(view, "grad")
    _plain(view.resolve_neg(), "grad")


@pytest.mark.parametrize("value", (2**64 + 5, -2**64 + 5, 2**63, 16.5, float("inf"), float("nan")))
def test_numbers_that_a_desc_would_cut_are_refused(value):
    from eagle_b200._sequences import _whole

    with pytest.raises((ValueError, OverflowError)):
        _whole(value, "first")
    assert (_whole(5, "first"), _whole(16.0, "block"), _whole(-2**63, "first")) == (5, 16, -2**63)
