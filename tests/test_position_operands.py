"""CPU checks of the position operators' operands: status codes before anything touches a device, and descriptors."""

import pytest

from tests.test_positions import _attention_call, _t
from substation_b200 import _lib
import ctypes


def _norm_forward(**kw):
    a = dict(q=_t([64, 4, 2, 8], ptr=0x10000), k=_t([64, 2, 2, 8], ptr=0x20000), qg=_t([64], ptr=0x30000), kg=_t([64], ptr=0x31000),
             pos=_t([2, 8], ptr=0x32000), qo=_t([64, 4, 2, 8], ptr=0x40000), ko=_t([64, 2, 2, 8], ptr=0x50000))
    a.update(kw)
    lib, r, b = _lib.load(), _lib.SbRotation(), ctypes.byref
    r.base, r.rotary, r.pairing, r.eps = 1e4, 64, 0, 1e-6
    st = lib.sb_query_key_norm_rotation(None, *(b(a[n]) for n in ('q', 'k', 'qg', 'kg', 'pos', 'qo', 'ko')), b(r))
    return st, lib.sb_last_error().decode()


def _norm_backward(**kw):
    a = dict(gq=_t([64, 4, 2, 8], ptr=0x11000), gk=_t([64, 2, 2, 8], ptr=0x22000), q=_t([64, 4, 2, 8], ptr=0x10000),
             k=_t([64, 2, 2, 8], ptr=0x20000), qg=_t([64], ptr=0x30000), kg=_t([64], ptr=0x31000), pos=_t([2, 8], ptr=0x32000),
             dq=_t([64, 4, 2, 8], ptr=0x40000), dk=_t([64, 2, 2, 8], ptr=0x50000), dqg=_t([64], ptr=0x33000), dkg=_t([64], ptr=0x34000))
    a.update(kw)
    lib, r, b = _lib.load(), _lib.SbRotation(), ctypes.byref
    r.base, r.rotary, r.pairing, r.eps = 1e4, 64, 0, 1e-6
    st = lib.sb_backward_query_key_norm_rotation(None, 0x1000000, lib.sb_query_key_norm_scratch_bytes(), *(b(t) for t in a.values()), b(r))
    return st, lib.sb_last_error().decode()


@pytest.mark.parametrize('call,kw', [
    (_norm_forward, dict(pos=_t([2, 8], ptr=0x32002))),
    (_norm_forward, dict(q=_t([64, 4, 2, 8], ptr=0x10001))),
    (_norm_forward, dict(qg=_t([64], ptr=0x30001))),
    (_norm_forward, dict(ko=_t([64, 2, 2, 8], ptr=0x50001))),
    (_norm_backward, dict(pos=_t([2, 8], ptr=0x32001))),
    (_norm_backward, dict(gk=_t([64, 2, 2, 8], ptr=0x22001))),
    (_norm_backward, dict(dqg=_t([64], ptr=0x33001))),
])
def test_misaligned_operands_of_norms(call, kw):
    st, text = call(**kw)
    assert st == 5 and 'aligned' in text, (st, text)


@pytest.mark.parametrize('call,kw', [
    # queries and keys are worked on at the same time
    (_norm_forward, dict(qo=_t([64, 4, 2, 8], ptr=0x20000))),
    (_norm_forward, dict(ko=_t([64, 2, 2, 8], ptr=0x10000))),
    (_norm_forward, dict(ko=_t([64, 2, 2, 8], ptr=0x40000))),
    (_norm_forward, dict(qo=_t([64, 4, 2, 8], ptr=0x31000))),
    (_norm_forward, dict(ko=_t([64, 2, 2, 8], ptr=0x32000))),
    (_norm_backward, dict(dq=_t([64, 4, 2, 8], ptr=0x20000))),
    (_norm_backward, dict(dq=_t([64, 4, 2, 8], ptr=0x22000))),
    (_norm_backward, dict(dk=_t([64, 2, 2, 8], ptr=0x10000))),
    (_norm_backward, dict(dk=_t([64, 2, 2, 8], ptr=0x11000))),
    (_norm_backward, dict(dk=_t([64, 2, 2, 8], ptr=0x40000))),
    (_norm_backward, dict(dkg=_t([64], ptr=0x33000))),
    (_norm_backward, dict(dqg=_t([64], ptr=0x40000))),
])
def test_outputs_of_norms_in_the_wrong_place(call, kw):
    st, text = call(**kw)
    assert st == 1 and 'place' in text, (st, text)


_APART = dict(q=_t([64, 4, 2, 8], ptr=0x10000), k=_t([64, 2, 2, 12], ptr=0x20000), v=_t([64, 2, 2, 12], ptr=0x30000), table=_t([8, 4], ptr=0x40000),
              lse=_t([4, 2, 8], ptr=0x50000), dout=_t([64, 4, 2, 8], ptr=0x60000))


@pytest.mark.parametrize('backward,kw', [
    (False, dict(lse=_t([4, 2, 8], ptr=0x50002))),
    (True, dict(lse=_t([4, 2, 8], ptr=0x50001))),
    (False, dict(v=_t([64, 2, 2, 12], ptr=0x30001))),
    (False, dict(table=_t([8, 4], ptr=0x40001))),
    (True, dict(dtable=_t([8, 4], ptr=0xa0001))),
    (True, dict(dout=_t([64, 4, 2, 8], ptr=0x60001))),
])
def test_misaligned_operands_of_attention(backward, kw):
    st, text = _attention_call(backward, **{**_APART, **kw})
    assert st == 5, (st, text)


@pytest.mark.parametrize('backward,kw', [
    (False, dict(lse=_t([4, 2, 8], ptr=0x20000))),
    (False, dict(lse=_t([4, 2, 8], ptr=0x90000))),               # the output
    (False, dict(lengths=0x90000)),
    (False, dict(first=0x50000)),
    (True, dict(dq=_t([64, 4, 2, 8], ptr=0xc0000))),             # dk
    (True, dict(dk=_t([64, 2, 2, 12], ptr=0xd0000))),            # dv
    (True, dict(dtable=_t([8, 4], ptr=0xb0000))),                # dq
    (True, dict(lengths=0xd0000)),
])
def test_outputs_of_attention_in_the_wrong_place(backward, kw):
    st, text = _attention_call(backward, **{**_APART, **kw})
    assert st == 1 and 'place' in text, (st, text)


def test_packed_descriptors_are_the_structures():
    """What ``ops`` packs as bytes reads back field by field through the structures that follow the header."""
    import torch
    from substation_b200 import ops
    x = torch.empty(3, 5, 7, 11)
    for t in (x.permute(2, 0, 3, 1), x[0, 0], x[:, 0, 0, 0], x[0], x[..., None].expand(-1, -1, -1, -1, 2)):
        raw = ops._packed(t)
        d = _lib.SbTensor.from_buffer_copy(raw)
        assert len(raw) == ctypes.sizeof(_lib.SbTensor) and d.ptr == t.data_ptr() and d.ndim == t.dim()
        assert tuple(d.size)[:t.dim()] == t.shape and tuple(d.stride)[:t.dim()] == t.stride()
    raw = ops._rotation(x, 5e5, 2, 'adjacent', 0.25)
    r = _lib.SbRotation.from_buffer_copy(raw)
    assert len(raw) == ctypes.sizeof(_lib.SbRotation) and (r.base, r.rotary, r.pairing, r.eps) == (5e5, 2, _lib.SB_PAIR_ADJACENT, 0.25)
    buckets = ops.RelativeBuckets([0, 1, 4], bidirectional=True)
    raw = ops._relative_bias(x[0, 0], buckets)
    b = _lib.SbRelativeBias.from_buffer_copy(raw)
    assert len(raw) == ctypes.sizeof(_lib.SbRelativeBias) and (b.n, b.bidirectional) == (3, 1)
    assert b.starts[:3] == [0, 1, 4] and b.table.contents.ptr == x.data_ptr() and b.table.contents.size[:2] == [7, 11]
    lengths, first = torch.zeros(7, dtype=torch.int32), torch.ones(7, dtype=torch.int32)
    raw = ops._span(x, 0.5, True, lengths, first)
    s = _lib.SbAttentionSpan.from_buffer_copy(raw)
    assert len(raw) == ctypes.sizeof(_lib.SbAttentionSpan)
    assert (s.scale, s.causal, s.lengths, s.first) == (0.5, 1, lengths.data_ptr(), first.data_ptr())
    s = _lib.SbAttentionSpan.from_buffer_copy(ops._span(x, 2.0, False, None, None))
    assert (s.scale, s.causal, s.lengths, s.first) == (2.0, 0, None, None)


def test_structures_are_the_headers(tmp_path):
    """Sizes and offsets of the ctypes structures against what a C compiler makes of the header."""
    import os
    import shutil
    import subprocess
    cc = shutil.which('gcc') or shutil.which('cc')
    if cc is None:
        pytest.skip('no C compiler')
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'include')
    classes = {'sb_tensor': _lib.SbTensor, 'sb_rotation': _lib.SbRotation, 'sb_relative_bias': _lib.SbRelativeBias,
               'sb_attention_span': _lib.SbAttentionSpan}
    lines = ['#include <stddef.h>', '#include "substation_b200.h"']
    for name, cls in classes.items():
        lines.append(f'_Static_assert(sizeof({name}) == {ctypes.sizeof(cls)}, "{name}");')
        for field, *_ in cls._fields_:
            lines.append(f'_Static_assert(offsetof({name}, {field}) == {getattr(cls, field).offset}, "{name}.{field}");')
    source = tmp_path / 'layout.c'
    source.write_text('\n'.join(lines) + '\n')
    r = subprocess.run([cc, '-std=c11', '-fsyntax-only', '-I', include, str(source)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
