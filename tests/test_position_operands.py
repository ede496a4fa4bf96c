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
