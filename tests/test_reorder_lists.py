"""Lists of states of several layouts that follow their beams: what is refused, that it is refused before anything moves, and what moves."""
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


def bytes_at(first, sentences, beams, outer, positions, bytes, row_stride, outer_stride, position_stride):
    return {first + r * row_stride + o * outer_stride + p * position_stride + b for r in range(sentences * beams) for o in range(outer) for p in range(positions)
            for b in range(bytes)}


def layout(rows, outer, positions, size, row, out, pos):
    return dict(sentences=1, beams=rows, outer=outer, positions=positions, bytes=size, row_stride=row, outer_stride=out, position_stride=pos)


@pytest.mark.parametrize("a,b", [
    (layout(3, 2, 3, 4, 36, 18, 6), layout(3, 2, 3, 2, 36, 18, 6)),                # keys beside narrower values
    (layout(3, 2, 3, 4, 36, 18, 6), layout(3, 3, 2, 2, 36, 6, 18)),                # the same memory in another order
    (layout(4, 1, 1, 20, 60, 0, 0), layout(4, 2, 5, 3, 60, 20, 4)),                # a part of rows beside finer ones
    (layout(2, 1, 1, 3, 100, 0, 0), layout(2, 1, 1, 3, 7, 0, 0)),                   # one inside a step of the other
    (layout(4, 2, 2, 2, 50, 20, 5), layout(4, 3, 2, 1, 31, 9, 4)),                  # nothing in common
    (layout(1, 1, 1, 5, 0, 0, 0), layout(3, 2, 2, 1, 40, 11, 3)),
])
def test_states_of_two_layouts_meet_where_bytes_do(a, b):
    """The library's answer at every distance against sets of bytes."""
    far = max(max(bytes_at(0, **a)), max(bytes_at(0, **b))) + 3
    seen = set()
    for d in range(-far, far + 1):
        rc, said = looked_over((a, [A]), (b, [A + d]), lengths=None)
        meet = bool(bytes_at(0, **a) & bytes_at(d, **b))
        assert (rc, meet) in ((0, False), (BAD, True)), (d, rc, said)
        seen.add(meet)
    assert seen == {False, True}


@pytest.mark.parametrize("seed", range(4))
def test_states_of_drawn_layouts_meet_where_bytes_do(seed):
    import random
    rng = random.Random(seed)
    tried = 0
    while tried < 600:
        drawn = []
        for _ in range(2):
            steps, extent, dims = [], rng.randint(1, 4), []
            size = extent
            for _ in range(3):
                n = rng.choice((1, 1, 2, 3, 4))
                stride = extent + rng.choice((0, 0, 1, 5, 20))
                dims.append((n, stride))
                extent += (n - 1) * stride
            rng.shuffle(dims)
            drawn.append(layout(dims[0][0], dims[1][0], dims[2][0], size, dims[0][1], dims[1][1], dims[2][1]))
        d = rng.randint(-40, 60)
        rc, said = looked_over((drawn[0], [A]), (drawn[1], [A + d]), lengths=None)
        assert (rc == BAD) == bool(bytes_at(0, **drawn[0]) & bytes_at(d, **drawn[1])) and rc in (0, BAD), (drawn, d, rc, said)
        tried += 1


def test_states_that_take_too_long_to_tell_apart_count_as_one():
    """Rows of 1 byte in all even places beside some in odd ones: they never meet, but every row of the one is within reach of every row of the other."""
    for sentences, code in ((10, 0), (10000, BAD)):
        fine = dict(layout(32, 1, 1, 1, 2, 0, 0), sentences=sentences)
        assert looked_over((fine, [A]), (dict(fine, row_stride=4), [A + 1]), lengths=None)[0] == code
        assert looked_over((fine, [A]), (dict(fine, row_stride=6), [A + 6]), lengths=None)[0] == BAD      # (the same bytes)


@pytest.mark.skipif(not _no_gpu(), reason="there is no context")
def test_the_binding_takes_lists_that_lie_among_each_other(monkeypatch):
    """Layers inside rows or keys beside values, together with a tensor elsewhere or with wider values in the same buffer: these get as far as the device."""
    import torch
    from excalibur_b200 import capi
    capi._torch()
    monkeypatch.setattr(capi, "_stream", lambda: None)
    parents, lengths = torch.zeros((1, 4), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    layers, other, beside = torch.zeros((4, 5, 3, 8, 16)), torch.zeros((4, 3, 8, 16)), torch.zeros((4, 3, 8, 48))
    both = torch.zeros((4, 6, 3, 8, 48))      # layers of keys and wider values inside rows
    for states in (list(layers.unbind(1)) + [other], [beside[..., :16], beside[..., 16:], other], [beside[..., :24], beside[..., 24:40], beside[..., 40:]],
                   [x for layer in both.unbind(1) for x in (layer[..., :16], layer[..., 16:])]):
        with pytest.raises(capi.ExbError) as said:
            capi.reorder_beams(Fake(), states, parents, lengths)
        assert " -3" in str(said.value), said.value      # there is no device
    for states in ([beside[..., :17], beside[..., 16:]], [other, layers[:, 0], layers[:, :1, :2].squeeze(1)], [beside, other, beside[:, :, :1, :1]]):
        with pytest.raises(capi.ExbError) as said:
            capi.reorder_beams(Fake(), states, parents, lengths)
        assert "share memory" in str(said.value), said.value


@pytest.mark.gpu
def test_states_of_unlike_layouts_in_one_buffer_follow_their_beams(ctx):
    """Layers of keys beside wider values inside rows, and a tensor elsewhere; a list that is refused leaves all of them as they were."""
    import torch
    from excalibur_b200 import capi
    g = torch.Generator(device="cuda").manual_seed(4)
    both, other = torch.randn((6, 5, 3, 8, 48), device="cuda", generator=g).half(), torch.randn((6, 2, 8, 5), device="cuda", generator=g)
    states = [x for layer in both.unbind(1) for x in (layer[..., :16], layer[..., 16:])] + [other]
    parents = torch.tensor([[1, 2, 0], [2, 2, -1]], device="cuda", dtype=torch.int32)
    lengths = torch.tensor([5, 8], device="cuda", dtype=torch.int32)
    for by in (lengths, None):
        want = []
        for t in (both, other):
            new = t.clone()
            for i in range(2):
                n = 8 if by is None else int(lengths[i])
                for j in range(3):
                    p = int(parents[i, j])
                    if p >= 0:
                        new[i * 3 + j, ..., :n, :] = t[i * 3 + p, ..., :n, :]
            want.append(new)
        capi.reorder_beams(ctx, states, parents, by)
        ctx.sync_check()
        assert torch.equal(both, want[0]) and torch.equal(other, want[1])
    before = both.clone(), other.clone()
    one = torch.empty((6, 1, 8, 4), device="cuda", dtype=torch.int32)
    one.view(-1)[:6] = parents.view(-1)
    for bad, at in ((one, one.view(-1)[:6].view(2, 3)), (both[:, :, 0, :, 8:24], parents), (both.view(6, -1)[:, :7], parents)):
        with pytest.raises(capi.ExbError):
            capi.reorder_beams(ctx, states + [bad], at)
    ctx.sync_check()
    assert torch.equal(both, before[0]) and torch.equal(other, before[1])
