"""CPU tests of dropout and the adapters beside a projection: the oracle's generator against the published vectors, the
struct's layout, and what the entry points refuse (no GPU needed: nothing is launched)."""
import ctypes
import gc
import os
import subprocess
import tempfile

import numpy as np
import pytest
import torch

import adapter_oracle as AO
from hortimapping_amd import _lib, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_generator_known_answers():
    """The vectors of the generator's publication (Philox4x32-10, counter and key of zeros / ones)."""
    z = AO.philox([[0]] * 4, (0, 0))[:, 0]
    assert [int(v) for v in z] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    f = AO.philox([[0xFFFFFFFF]] * 4, (0xFFFFFFFF, 0xFFFFFFFF))[:, 0]
    assert [int(v) for v in f] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_mask_depends_on_the_place_alone():
    k, up = AO.keep_mask(64, 40, 0.3, 77, tag=5)
    assert abs(up - 65536 / (65536 - 19661)) < 1e-12
    part, _ = AO.keep_mask(10, 19, 0.3, 77, tag=5, row0=7)
    assert torch.equal(part, k[7:17, :19])
    assert not torch.equal(AO.keep_mask(64, 40, 0.3, 77, tag=6)[0], k)


def test_args_struct_matches_the_header():
    cls = _lib.HmAdapterArgs
    names = [f[0] for f in cls._fields_]
    prog = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{ROOT}/include/hortimapping_amd.h"', 'int main(void){',
            'printf("%zu\\n", sizeof(hm_adapter_args));']
    prog += [f'printf("%zu\\n", offsetof(hm_adapter_args, {n}));' for n in names] + ['return 0;}']
    with tempfile.TemporaryDirectory() as td:
        c, exe = os.path.join(td, "t.c"), os.path.join(td, "t")
        open(c, "w").write("\n".join(prog))
        subprocess.check_call(["gcc", "-std=c99", "-o", exe, c])
        got = [int(v) for v in subprocess.check_output([exe]).decode().split()]
    assert got == [ctypes.sizeof(cls)] + [getattr(cls, n).offset for n in names]


def args(**kw):
    """A call that is refused for one reason: pointers are non-zero but never read on the host."""
    d = dict(type=0, k=8, n=8, rank=4, adapters=2, segments=2, tag=0, rows=16, d_x=4096, ld_x=8, d_w=4096, ld_w=8, d_bias=0,
             d_a=4096, d_b=4096, d_scale=0, d_row_start=4096, d_adapter=4096, p=0.0, seed=0, d_seed=0, row0=0)
    d.update(kw)
    return _lib.HmAdapterArgs(**d)


@pytest.mark.parametrize("kw,word", [
    (dict(type=3), b"type"), (dict(rows=-1), b"rows"), (dict(rows=1 << 25), b"rows"), (dict(k=0), b"k = 0"), (dict(n=70000), b"70000"),
    (dict(rank=0), b"rank"), (dict(rank=257), b"rank"), (dict(adapters=-1), b"adapters"), (dict(segments=-1), b"requests"),
    (dict(adapters=70000), b"adapters"), (dict(p=-0.1), b"p must"), (dict(p=1.5), b"p must"), (dict(p=float("nan")), b"p must"),
    (dict(d_x=0), b"null"), (dict(d_w=0), b"null"), (dict(d_a=0), b"null"), (dict(d_row_start=0), b"null"), (dict(d_adapter=0), b"null"),
    (dict(ld_x=7), b"stride"), (dict(ld_w=7), b"stride"), (dict(ld_x=1 << 22), b"stride"), (dict(ld_w=1 << 22), b"stride")])
def test_adapter_entries_refuse(kw, word):
    lib, a = _lib.lib(), args(**kw)
    assert lib.hm_adapter_linear(ctypes.byref(a), 4096, 8, 4096, None) < 0 and word in lib.hm_last_error()
    assert lib.hm_adapter_linear_backward(ctypes.byref(a), 4096, 8, 4096, 4096, 8, 4096, 4096, 4096, 1 << 40, None) < 0
    assert word in lib.hm_last_error()


def test_adapter_entries_refuse_outputs_and_workspaces():
    lib, a = _lib.lib(), args()
    ref = ctypes.byref(a)
    assert lib.hm_adapter_linear(None, 4096, 8, 4096, None) < 0
    assert lib.hm_adapter_linear(ref, None, 8, 4096, None) < 0 and b"null" in lib.hm_last_error()
    assert lib.hm_adapter_linear(ref, 4096, 8, None, None) < 0 and b"null" in lib.hm_last_error()
    assert lib.hm_adapter_linear(ref, 4096, 7, 4096, None) < 0 and b"stride" in lib.hm_last_error()
    need = lib.hm_adapter_linear_backward_bytes(ref)
    assert need > 0 and lib.hm_adapter_linear_backward_bytes(None) == -1
    assert lib.hm_adapter_linear_backward_bytes(ctypes.byref(args(rank=0))) == -1
    back = lambda dy=4096, ldy=8, t=4096, ldx=8, ws=4096, size=need: lib.hm_adapter_linear_backward(  # noqa: E731
        ref, dy, ldy, t, 4096, ldx, 4096, 4096, ws, size, None)
    for bad, word in ((dict(dy=None), b"null"), (dict(t=None), b"null"), (dict(ldy=7), b"stride"), (dict(ldx=7), b"stride"),
                      (dict(ws=None), b"workspace"), (dict(size=need - 1), b"workspace")):
        assert back(**bad) < 0 and word in lib.hm_last_error(), bad


def test_the_workspace_stays_bounded():
    """Many short requests do not ask for a slot of partial sums each."""
    lib = _lib.lib()
    for rows, seg, k in ((131072, 131072, 512), (16777216, 1 << 20, 4096), (8192, 256, 4096)):
        a = args(rows=rows, segments=seg, k=k, n=k, ld_x=k, ld_w=k, rank=64, adapters=64)
        size = lib.hm_adapter_linear_backward_bytes(ctypes.byref(a))
        assert 0 < size < (513 << 20) + rows * 64 * 4 + 2 * (k * k + 64 * 64 * k) * 4 + 4096


@pytest.mark.parametrize("kw,word", [(dict(rows=-1), b"negative"), (dict(cols=-1), b"negative"), (dict(p=2.0), b"p must"),
                                     (dict(p=float("nan")), b"p must"), (dict(type=9), b"type"), (dict(x=None), b"null"),
                                     (dict(y=None), b"null"), (dict(ldx=3), b"stride"), (dict(ldy=3), b"stride")])
def test_dropout_entries_refuse(kw, word):
    lib = _lib.lib()
    d = dict(x=4096, ldx=4, y=4096, ldy=4, rows=2, cols=4, type=0, p=0.5)
    d.update(kw)
    rc = lib.hm_dropout(d["x"], d["ldx"], d["y"], d["ldy"], d["rows"], d["cols"], d["type"], 0, d["p"], 1, None, 0, 0, None)
    assert rc < 0 and word in lib.hm_last_error()
    rc = lib.hm_dropout_backward(d["x"], d["ldx"], 4096, 4, d["y"], d["ldy"], d["rows"], d["cols"], d["type"], 1, d["p"], 1, None,
                                 0, 0, None)
    assert rc < 0 and word in lib.hm_last_error()


def test_dropout_entry_needs_the_output_for_relu():
    lib = _lib.lib()
    assert lib.hm_dropout_backward(4096, 4, None, 4, 4096, 4, 2, 4, 0, 1, 0.5, 1, None, 0, 0, None) < 0
    assert b"null" in lib.hm_last_error()


def test_nothing_to_do_needs_no_gpu():
    lib = _lib.lib()
    assert lib.hm_dropout(None, 0, None, 0, 0, 4, 0, 0, 0.5, 1, None, 0, 0, None) == 0
    assert lib.hm_adapter_linear(ctypes.byref(args(rows=0)), None, 8, None, None) == 0


def test_wrappers_refuse_host_tensors():
    x = torch.zeros(2, 4)
    with pytest.raises(ValueError, match="on the GPU"):
        ops.dropout(x, 0.5, 1)
    with pytest.raises(ValueError, match="on the GPU"):
        ops.adapter_linear(x, x, x, x, x, x)


@pytest.mark.parametrize("shape,strides,want", [
    ((4, 6), (6, 1), (4, 6, 6)), ((4, 6), (9, 1), (4, 6, 9)), ((2, 3, 6), (27, 9, 1), (6, 6, 9)), ((6,), (1,), (1, 6, 6)),
    ((5, 1), (7, 3), (5, 1, 7)), ((1, 6), (0, 1), (1, 6, 6)), ((0, 6), (6, 1), (0, 6, 6)), ((4, 1, 6), (9, 77, 1), (4, 6, 9))])
def test_rows_of_a_tensor(shape, strides, want):
    t = torch.zeros(400).as_strided(shape, strides)
    assert ops._rows("x", t) == want


@pytest.mark.parametrize("shape,strides", [((4, 6), (1, 4)), ((4, 6), (0, 1)), ((2, 3, 6), (100, 9, 1)), ((4, 6), (3, 1))])
def test_rows_that_are_refused(shape, strides):
    t = torch.zeros(400).as_strided(shape, strides)
    with pytest.raises(ValueError):
        ops._rows("x", t)
    assert ops._rows_of_grad(t)[1:] == (int(np.prod(shape[:-1])), shape[-1], shape[-1])


def test_a_leaf_of_another_stream_is_refused_within_a_capture(monkeypatch):
    x = torch.zeros(3, requires_grad=True)
    y = ops._of_one_stream(x * 2, 7)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    assert ops._of_one_stream(x * 3, 8).shape == (3,)                         # no capture: nothing to refuse
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    assert ops._of_one_stream(x * 3, 7).shape == (3,)
    with pytest.raises(RuntimeError, match="another stream"):
        ops._of_one_stream(x * 3, 8)
    del y
    gc.collect()                                                              # (the refusal's traceback held its argument)
    assert ops._of_one_stream(x * 3, 8).shape == (3,)                         # the older graph is gone
    h = torch.zeros(3, requires_grad=True) * 1
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    ops._of_one_stream(h * 2, 1), ops._of_one_stream(h * 2, 2)                # no leaf: its nodes are not looked at


def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as fwd
    x, v = torch.ones(3), torch.full((3,), 2.0)
    ops._no_tangents(x=x, bias=None)
    with fwd.dual_level():
        d = fwd.make_dual(x, v)
        assert not d.requires_grad                                           # why nothing else would notice
        ops._no_tangents(x=x, bias=None)
        with pytest.raises(NotImplementedError, match="bias carries"):
            ops._no_tangents(x=x, bias=d)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="x carries"):
            ops._no_tangents(x=d)
    with pytest.raises(NotImplementedError, match="x carries"):
        torch.func.jvp(lambda t: (ops._no_tangents(x=t), t * 2)[1], (x,), (v,))
    ops._no_tangents(x=x)


@pytest.mark.parametrize("kind", [0, 1, 2])
def test_dropout_of_more_values_than_a_launch_takes(kind):
    """2^32 threads (2^31 rows of eight blocks, 1024 blocks a workgroup of 256): refused before anything is launched."""
    lib = _lib.lib()
    for rows in (1 << 31, (1 << 63) - 1):
        rc = lib.hm_dropout(4096, 64, 4096, 64, rows, 64, kind, 0, 0.5, 1, None, 0, 0, None)
        assert rc < 0 and b"too many" in lib.hm_last_error()
        rc = lib.hm_dropout_backward(4096, 64, 4096, 64, 4096, 64, rows, 64, kind, 1, 0.5, 1, None, 0, 0, None)
        assert rc < 0 and b"too many" in lib.hm_last_error()


def test_adapter_outputs_of_more_tiles_than_a_launch_takes():
    """2^18 x 2^6 tiles of 64 x 64 outputs in fp32, of 256 threads each: refused before anything is launched."""
    lib, rows = _lib.lib(), 1 << 24
    a = args(rows=rows, k=16, n=4096, segments=0, ld_x=16, ld_w=16)
    assert lib.hm_adapter_linear(ctypes.byref(a), 4096, 4096, 4096, None) < 0 and b"too many" in lib.hm_last_error()
    a = args(rows=rows, k=4096, n=16, segments=0, ld_x=4096, ld_w=4096)
    assert lib.hm_adapter_linear_backward(ctypes.byref(a), 4096, 16, 4096, 4096, 4096, None, None, 4096, 1 << 40, None) < 0
    assert b"too many" in lib.hm_last_error()
