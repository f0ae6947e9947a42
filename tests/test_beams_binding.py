"""Beam search's selection and the reordering of states, without a GPU: descriptors, refusals, layouts of states."""
import ctypes

import pytest

from test_int8_experts_binding import BAD, UNSUPPORTED, Fake, _no_gpu, offsets_agree, refusal

DESCRIPTORS = {"exb_beam_desc": ("BeamDesc", "@3q5if"), "exb_reorder_desc": ("ReorderDesc", "@q2i6q")}


def test_descriptors_are_laid_out_alike(tmp_path):
    offsets_agree(DESCRIPTORS, tmp_path)


A, S, N, O, P, T, W, L = (0x10000000 * i for i in range(1, 9))      # addresses far apart


def select(**changed):
    from excalibur_b200 import capi
    d = dict(sentences=3, stride=1000, workspace_bytes=8 * 12 * 9, beams=4, V=1000, dtype=capi.EXB_F16, select=8, end_token=2, scale=1.0)
    at = dict(logits=A, scores=S, ended=N, out=O, parents=P, tokens=T, workspace=W)
    for k, v in changed.items():
        (d if k in d else at)[k] = v
    return refusal("exb_beam_select_fwd", ctypes.byref(capi.BeamDesc(**d)), *(at[k] for k in ("logits", "scores", "ended", "out", "parents", "tokens", "workspace")))


def reorder(states=(A, A + 0x100000), parents=P, lengths=L, **changed):
    from excalibur_b200 import capi
    d = dict(sentences=2, beams=4, n_states=len(states), outer=3, positions=16, bytes=64, row_stride=3 * 16 * 64, outer_stride=16 * 64, position_stride=64)
    d.update(changed)
    return refusal("exb_reorder_beams_fwd", ctypes.byref(capi.ReorderDesc(**d)), (ctypes.c_void_p * len(states))(*states), parents, lengths)


@pytest.mark.skipif(not _no_gpu(), reason="the addresses are not real")
@pytest.mark.parametrize("call,changed", [
    (select, {}), (select, dict(ended=None, end_token=-1)), (select, dict(select=32, workspace_bytes=8 * 12 * 33)), (select, dict(V=5, workspace_bytes=8 * 12 * 6)),
    (reorder, {}), (reorder, dict(lengths=None)),
    (reorder, dict(position_stride=3 * 64, outer_stride=64)),                                                       # heads inside positions
    (reorder, dict(states=(A, A + 64), row_stride=3 * 16 * 128, outer_stride=16 * 128, position_stride=128)),      # keys and values side by side
    (reorder, dict(states=(A, A + 3 * 16 * 64), row_stride=2 * 3 * 16 * 64)),                                       # layers inside rows
    (reorder, dict(outer=1, outer_stride=0)),
])
def test_a_good_call_gets_as_far_as_the_device(call, changed):
    assert call(**changed)[0] == -3, call(**changed)      # EXB_ERR_CUDA: there is none


@pytest.mark.parametrize("call,changed,code", [
    (select, dict(dtype=1), BAD), (select, dict(sentences=-1), BAD), (select, dict(beams=0), BAD), (select, dict(V=0), BAD), (select, dict(select=0), BAD),
    (select, dict(beams=33), UNSUPPORTED), (select, dict(select=33), UNSUPPORTED), (select, dict(sentences=1 << 31), UNSUPPORTED), (select, dict(V=(1 << 30) + 1, stride=1 << 31), UNSUPPORTED),
    (select, dict(scale=0.0), BAD), (select, dict(scale=-1.0), BAD), (select, dict(scale=float("nan")), BAD), (select, dict(scale=float("inf")), BAD),
    (select, dict(end_token=-1), BAD), (select, dict(end_token=1000), BAD), (select, dict(stride=999), BAD), (select, dict(workspace_bytes=8 * 12 * 9 - 1), BAD),
    *[(select, {k: None}, BAD) for k in ("logits", "scores", "out", "parents", "tokens")],
    (select, dict(logits=A + 1), BAD), (select, dict(scores=S + 2), BAD), (select, dict(out=O + 1), BAD), (select, dict(tokens=T + 2), BAD), (select, dict(workspace=W + 4), BAD),
    (select, dict(out=S), BAD), (select, dict(parents=A + 8), BAD), (select, dict(tokens=P + 4), BAD), (select, dict(workspace=A + 16), BAD), (select, dict(workspace=O), BAD),
    (select, dict(out=N), BAD),
    (reorder, dict(sentences=-1), BAD), (reorder, dict(beams=0), BAD), (reorder, dict(n_states=-1), BAD), (reorder, dict(outer=-1), BAD), (reorder, dict(bytes=-1), BAD),
    (reorder, dict(beams=33), UNSUPPORTED), (reorder, dict(n_states=(1 << 20) + 1), UNSUPPORTED), (reorder, dict(sentences=1 << 40), UNSUPPORTED),
    (reorder, dict(parents=None), BAD), (reorder, dict(states=(A, None)), BAD), (reorder, dict(parents=P + 2), BAD), (reorder, dict(lengths=L + 1), BAD),
    (reorder, dict(states=(A, A)), BAD), (reorder, dict(states=(A, A + 63)), BAD), (reorder, dict(states=(A + 8 * 3 * 16 * 64 - 1, A)), BAD),
    (reorder, dict(states=(A, A + 32), row_stride=3 * 16 * 128, outer_stride=16 * 128, position_stride=128), BAD),
    (reorder, dict(row_stride=0), BAD), (reorder, dict(position_stride=32), BAD), (reorder, dict(outer_stride=100), BAD), (reorder, dict(row_stride=-64), BAD),
    (reorder, dict(parents=A + 64), BAD), (reorder, dict(lengths=A + 4), BAD),
])
def test_bad_calls_are_refused(call, changed, code):
    assert call(**changed)[0] == code, changed


@pytest.mark.skipif(not _no_gpu(), reason="the addresses are not real")
def test_a_call_needs_a_workspace_or_none():
    """(The device is looked for first: what this machine cannot show, the selection's own tests do.)"""
    assert select(workspace=None, workspace_bytes=0)[0] == -3


def test_empty_calls_are_no_error():
    assert select(sentences=0, logits=None)[0] == 0
    for empty in ("sentences", "n_states", "outer", "positions", "bytes"):
        assert reorder(parents=None, **{empty: 0})[0] == 0


def test_states_meet_where_bytes_do():
    """The library's answer for states at every distance, in layouts of unlike order, against sets of bytes."""
    for outer, positions, size, row, out, pos in [(2, 3, 4, 24, 12, 4), (2, 3, 4, 48, 4, 8), (2, 2, 2, 7, 2, 100), (3, 1, 2, 9, 3, 0), (1, 3, 1, 11, 0, 3)]:
        def bytes_at(first):
            return {first + r * row + o * out + p * pos + b for r in range(4) for o in range(outer) for p in range(positions) for b in range(size)}
        far = max(bytes_at(0)) + 3
        for d in range(-far, far + 1):
            rc, said = reorder(states=(A, A + d), lengths=None, sentences=2, beams=2, outer=outer, positions=positions, bytes=size, row_stride=row, outer_stride=out,
                               position_stride=pos)
            assert (rc == BAD and "share" in said) == bool(bytes_at(0) & bytes_at(d)), (outer, positions, size, row, out, pos, d)


def test_the_binding_refuses_tensors_that_do_not_fit(monkeypatch):
    import torch
    from excalibur_b200 import capi
    capi._torch()
    monkeypatch.setattr(capi, "_stream", lambda: None)
    ctx = Fake()

    def z(*shape, dtype=torch.float16):
        return torch.zeros(shape, dtype=dtype)
    f32, i32 = torch.float32, torch.int32
    logits, scores = z(6, 50), z(2, 3, dtype=f32)
    for args, kw in [((logits, z(2, 3)), {}), ((logits, z(6, dtype=f32)), {}), ((logits, z(3, 3, dtype=f32)), {}), ((logits, z(3, 2, dtype=f32).t()), {}),
                     ((z(6, 50, 1), scores), {}), ((z(50, 6).t(), scores), {}), ((logits, scores), dict(ended=z(2, 3))), ((logits, scores), dict(ended=z(6, dtype=torch.bool))),
                     ((logits, scores), dict(ended=z(3, 2, dtype=torch.bool).t())), ((logits, scores), dict(select=0)), ((logits, scores), dict(select=33)),
                     ((logits, scores), dict(select=-1)), ((logits, scores), dict(scale=0.0)), ((z(6, 50, dtype=i32), scores), {}),
                     ((logits, scores), dict(ended=z(2, 3, dtype=torch.bool), end_token=50))]:
        with pytest.raises(capi.ExbError):
            capi.beam_select(ctx, *args, **kw)
    parents, state, lengths = z(2, 3, dtype=i32), z(6, 4, 8, 16), z(2, dtype=i32)
    for args, kw in [((state, z(6, dtype=i32)), {}), ((state, z(2, 3)), {}), ((state, z(3, 2, dtype=i32).t()), {}), ((z(5, 4, 8, 16), parents), {}), ((z(), parents), {}),
                     ((state, parents), dict(lengths=z(3, dtype=i32))), ((state, parents), dict(lengths=z(2))), ((z(6, 16), parents), dict(lengths=lengths)),
                     ((z(6, 4, 16, 8).transpose(2, 3), parents), dict(lengths=lengths)), ((z(6, 1, 16).expand(6, 8, 16), parents), {}), ((z(1, 16).expand(6, 16), parents), {}),
                     ((z(6, 4, 5, 8, 16).transpose(1, 2), parents), dict(lengths=lengths)), (([state, state], parents), {}), (([state, state[:, :2]], parents), {}),
                     (([state, z(6, 0)], parents.to(torch.int64)), {})]:
        with pytest.raises(capi.ExbError):
            capi.reorder_beams(ctx, *args, **kw)


def test_layouts_of_states():
    """Sizes and strides in bytes that the library is told, by what they address."""
    import torch
    from excalibur_b200 import capi
    capi._torch()
    whole = torch.arange(6 * 4 * 8 * 16, dtype=torch.int16).view(6, 4, 8, 16)
    for state, by_length in [(whole, False), (whole, True), (whole.transpose(1, 2), True), (whole[:, 1:3], True), (whole[:, :, 2:6], True), (whole[..., 4:8], True),
                             (whole[..., :1], True), (whole[:, :, :1], True), (whole[:, 2], True), (whole.view(6, 2, 2, 8, 16), True), (whole[:, 0, 0], False),
                             (whole[:, 0, 0, 0], False), (whole[:, :, 0, 0], False), (whole[:, :, 0], False), (whole[::2], True), (whole[:1], True),
                             (whole.transpose(0, 1).contiguous().transpose(0, 1), True)]:
        o, p, size, row, out, pos = capi._state_layout(state, state.shape[0], by_length)
        base = (state.data_ptr() - whole.data_ptr()) if state.data_ptr() >= whole.data_ptr() and state.data_ptr() < whole.data_ptr() + whole.numel() * 2 else None
        at = {r * row + i * out + j * pos + b for r in range(state.shape[0]) for i in range(o) for j in range(p) for b in range(0, size, 2)}
        want = set()
        for index in torch.cartesian_prod(*[torch.arange(n) for n in state.shape]).view(-1, state.dim()).tolist():
            want.add(2 * sum(i * s for i, s in zip(index, state.stride())))
        assert at == want, (state.shape, state.stride(), base)
        if by_length:
            assert p == state.shape[-2]
