"""Lists of states of several layouts that follow their beams, without a GPU: what is refused, and that it is refused before anything moves."""
import ctypes

import pytest

from test_int8_experts_binding import BAD, UNSUPPORTED, Fake, _no_gpu

A, P, L = 0x10000000, 0x20000000, 0x30000000      # addresses far apart
WHOLE = dict(sentences=2, beams=4, outer=3, positions=16, bytes=64, row_stride=3 * 16 * 64, outer_stride=16 * 64, position_stride=64)


def looked_over(*groups, parents=P, lengths=L):
    """The library's answer to several calls at once: a dict of what differs from WHOLE and a list of addresses for each."""
    from excalibur_b200 import capi
    descriptors = (capi.ReorderDesc * len(groups))(*[capi.ReorderDesc(**{**WHOLE, "n_states": len(at), **d}) for d, at in groups])
    lists = [(ctypes.c_void_p * len(at))(*at) for _, at in groups]
    rc = capi.lib().exb_reorder_beams_check(ctypes.byref(descriptors), len(groups), (ctypes.c_void_p * len(groups))(*[ctypes.addressof(x) for x in lists]), parents, lengths)
    return rc, capi.last_error()


def test_each_call_is_looked_over():
    far = A + (1 << 20)
    assert looked_over()[0] == 0 and looked_over(({}, [A]))[0] == 0 and looked_over(({}, [A]), (dict(bytes=32, position_stride=32), [far]))[0] == 0
    assert looked_over(({}, [A]), (dict(outer=0), [None]))[0] == 0
    for d, at, code in ((dict(beams=33), [far], UNSUPPORTED), (dict(position_stride=32), [far], BAD), ({}, [None], BAD), (dict(bytes=-1), [far], BAD),
                        (dict(bytes=32), [far, far + 31], BAD)):
        assert looked_over(({}, [A]), (d, at))[0] == code, d
        assert looked_over((d, at), ({}, [A]))[0] == code, d
    assert looked_over(({}, [A]), (dict(bytes=32), [far]), parents=far + 4)[0] == BAD
    assert looked_over(({}, [A]), (dict(bytes=32), [far]), lengths=far + 4)[0] == BAD
    assert looked_over(({}, [A]), parents=None)[0] == BAD


@pytest.mark.skipif(not _no_gpu(), reason="there is no context")
@pytest.mark.parametrize("what", ["parents", "lengths"])
def test_the_binding_looks_all_states_over_before_the_first_moves(monkeypatch, what):
    """Parents or lengths among the rows of a state of another layout than the first one's; without a GPU a call that moves ends at the device instead."""
    import torch
    from excalibur_b200 import capi
    capi._torch()
    monkeypatch.setattr(capi, "_stream", lambda: None)
    first, second = torch.zeros((4, 3, 8, 16), dtype=torch.float16), torch.zeros((4, 1, 8, 4), dtype=torch.int32)
    parents, lengths = torch.zeros((1, 4), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(capi.ExbError) as good:
        capi.reorder_beams(Fake(), [first, second], parents, lengths)
    assert "lie" not in str(good.value)
    if what == "parents":
        parents = second[:1, 0, 0]
    else:
        lengths = second[0, 0, 0, :1]
    with pytest.raises(capi.ExbError) as bad:
        capi.reorder_beams(Fake(), [first, second], parents, lengths)
    assert "parents or lengths lie among a state's rows" in str(bad.value)
