"""What the recurrent policy's entry points refuse before anything is launched, and their records' C sizes: no GPU needed."""
import ctypes as C
import os
import subprocess

import pytest
import torch

import rl_gan_amd as R
from rl_gan_amd import _lib
from rl_gan_amd._lib import lib
from rl_gan_amd.tensors import own_elements

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ARG, DIMS, KIND, ALIGN = -1, -2, -3, -5


def test_records_have_the_c_sizes(tmp_path):
    recs = {"rlgan_seq_t": _lib.SeqRef, "rlgan_scan_t": _lib.Scan, "rlgan_policy_t": _lib.Policy, "rlgan_adamw_tensor_t": _lib.AdamWTensor,
            "rlgan_adamw_t": _lib.AdamWState}
    src = tmp_path / "sz.c"
    body = "".join(f'  printf("{n} %zu\\n", sizeof({n}));\n' for n in recs)
    src.write_text(f'#include <stdio.h>\n#include "rlgan_amd.h"\nint main(void) {{\n{body}  printf("chunk %d\\nscalars %d\\n", RLGAN_ADAMW_CHUNK, RLGAN_ADAMW_SCALARS);\n  return 0;\n}}\n')
    exe = tmp_path / "sz"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    assert int(out.pop("chunk")) == _lib.ADAMW_CHUNK and int(out.pop("scalars")) == 32
    for name, size in out.items():
        assert C.sizeof(recs[name]) == int(size), name


def test_packed_records_are_the_records():
    seq = (11, 12, 13)
    s = _lib.Scan(1, 2, 3, 2, _lib.SeqRef(*seq), _lib.SeqRef(21, 22, 23), 31, 32, 33, 34, 35)
    assert bytes(s) == _lib.PACK_SCAN(1, 2, 3, 2, *seq, 21, 22, 23, 31, 32, 33, 34, 35)
    values = list(range(1, 25))
    p = _lib.Policy(*values)
    packed = _lib.PACK_POLICY(*values)
    assert len(packed) == C.sizeof(p)
    back = _lib.Policy.from_buffer_copy(packed)
    for name, _ in _lib.Policy._fields_:                        # (the padding's bytes may be anything)
        assert getattr(back, name) == getattr(p, name), name


def _scan(**change):
    s = _lib.Scan(2, 3, 4, 0, _lib.SeqRef(64, 12, 4), _lib.SeqRef(64, 12, 4), None, None, 0, 0, None)
    for k, v in change.items():
        setattr(s, k, v)
    return s


def test_scan_refusals():
    seq, none = _lib.SeqRef(64, 12, 4), _lib.SeqRef(None, 0, 0)
    fwd = lambda s, h=seq, last=64: lib.rlgan_gated_scan_forward(C.byref(s), h, last, None, None)
    assert lib.rlgan_gated_scan_forward(None, seq, 64, None, None) == ARG
    assert fwd(_scan(batch=0)) == ARG and fwd(_scan(length=-1)) == ARG and fwd(_scan(width=0)) == ARG
    assert fwd(_scan(type=3)) == KIND and fwd(_scan(z=none)) == ARG and fwd(_scan(x=none)) == ARG
    assert fwd(_scan(), none) == ARG and fwd(_scan(), seq, None) == ARG
    assert fwd(_scan(batch=1 << 30, width=4)) == DIMS and fwd(_scan(batch=1 << 16, width=1 << 15)) == DIMS
    assert fwd(_scan(length=(1 << 30) + 1)) == DIMS
    bwd = lambda s, h=seq, dh=seq, dz=seq, dx=seq, ds=64: lib.rlgan_gated_scan_backward(C.byref(s), h, dh, None, dz, dx, ds, None, None)
    assert bwd(_scan(), h=none) == ARG and bwd(_scan(), dh=none) == ARG and bwd(_scan(), dz=none) == ARG
    assert bwd(_scan(), dx=none) == ARG and bwd(_scan(), ds=None) == ARG and bwd(_scan(type=-1)) == KIND
    n = C.c_int64()
    assert lib.rlgan_gated_scan_workspace(2, 3, 4, 0, 0, None) == ARG and lib.rlgan_gated_scan_workspace(0, 3, 4, 0, 0, C.byref(n)) == ARG
    assert lib.rlgan_gated_scan_workspace(2, 3, 4, 7, 0, C.byref(n)) == KIND


def test_step_refusals():
    ok = [0, 2, 4, 64, 4, 64, 4, 64, None, 0, 64, None]
    for at, value, want in ((0, 3, KIND), (1, 0, ARG), (2, -1, ARG), (3, None, ARG), (5, None, ARG), (7, None, ARG), (10, None, ARG)):
        args = list(ok)
        args[at] = value
        assert lib.rlgan_gated_step(*args) == want, at


def test_scan_workspace_is_wanted():
    """A long sequence of few units is cut, and its call wants the workspace that the size function names."""
    n = C.c_int64()
    for backward in (0, 1):
        assert lib.rlgan_gated_scan_workspace(1, 100000, 64, 0, backward, C.byref(n)) == 0
        if n.value:
            s, seq = _scan(batch=1, length=100000, width=64), _lib.SeqRef(64, 0, 64)
            if backward:
                assert lib.rlgan_gated_scan_backward(C.byref(s), seq, seq, None, seq, seq, 64, None, None) == ARG
            else:
                assert lib.rlgan_gated_scan_forward(C.byref(s), seq, 64, None, None) == ARG


def _policy(**change):
    p = _lib.Policy(rows=3, vocab=5, type=0, logits=64, ld=5, actions=64, action_bytes=4, old_logp=64, advantages=64, weights=None, ref_logp=None,
                    legal=None, ld_legal=0, clip_low=0.2, clip_high=0.2, kl_coef=0, entropy_coef=0, temperature=1.0, loss=64, logp=64, entropy=64,
                    kl=64, dlogits=None, ld_d=0)
    for k, v in change.items():
        setattr(p, k, v)
    return p


def test_policy_refusals():
    call = lambda p, ws=64: lib.rlgan_policy_loss(C.byref(p), ws, None)
    assert lib.rlgan_policy_loss(None, 64, None) == ARG
    for k in ("logits", "actions", "old_logp", "advantages", "loss", "logp", "entropy", "kl"):
        assert call(_policy(**{k: None})) == ARG, k
    assert call(_policy(), None) == ARG
    assert call(_policy(rows=0)) == ARG and call(_policy(rows=1 << 31)) == ARG and call(_policy(vocab=0)) == ARG
    assert call(_policy(type=3)) == KIND and call(_policy(action_bytes=2)) == KIND
    assert call(_policy(ld=4)) == ALIGN and call(_policy(dlogits=64, ld_d=4)) == ALIGN and call(_policy(legal=64, ld_legal=3)) == ALIGN
    assert call(_policy(vocab=(1 << 30) + 1, ld=1 << 31)) == DIMS
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-39):
        assert call(_policy(temperature=t)) == ARG
    n = C.c_int64()
    assert lib.rlgan_policy_loss_workspace(0, 5, 0, C.byref(n)) == ARG and lib.rlgan_policy_loss_workspace(3, 5, 9, C.byref(n)) == KIND


def test_adamw_refusals():
    begin = (C.c_int64 * 3)(0, 1, 2)
    grads, types = (C.c_void_p * 2)(64, 64), (C.c_uint8 * 2)(0, 0)

    def state(**change):
        a = _lib.AdamWState(2, 32, 64, 64, C.addressof(begin), 64, 64, None, None, 64, 64, 64, 0.9, 0.999, 1e-8, 0.0)
        for k, v in change.items():
            setattr(a, k, v)
        return a
    call = lambda a, g=grads, t=types: lib.rlgan_adamw_step(C.byref(a), g, t, None, None, None)
    assert lib.rlgan_adamw_step(None, grads, types, None, None, None) == ARG
    assert call(state(), None) == ARG and call(state(), grads, None) == ARG and call(state(n_tensors=0)) == ARG
    for k in ("tensors", "chunks", "chunk_begin", "first", "second", "lr", "step", "scalars"):
        assert call(state(**{k: None})) == ARG, k
    assert call(state(state_bits=16)) == KIND and call(state(state_bits=8)) == ARG
    assert call(state(beta1=1.0)) == ARG and call(state(beta2=-0.1)) == ARG and call(state(eps=float("nan"))) == ARG
    assert call(state(), (C.c_void_p * 2)(64, None)) == ARG and call(state(), grads, (C.c_uint8 * 2)(0, 3)) == KIND
    backwards = (C.c_int64 * 3)(0, 2, 1)
    assert call(state(chunk_begin=C.addressof(backwards))) == DIMS
    for fn, args in ((lib.rlgan_adamw_decode, [64, 64, 64, 64, 64, 64, 64]), (lib.rlgan_adamw_encode, [64, 64, 64, 64, 64, 64, 64])):
        at = 4 if fn is lib.rlgan_adamw_decode else 2
        for n, want in ((0, ARG), (-64, ARG), (63, ALIGN)):
            assert fn(*args[:at], n, *args[at + 1:], None) == want
        for i in range(7):
            if i != at:
                bad = list(args)
                bad[i] = None
                assert fn(*bad, None) == ARG


def test_there_is_no_cpu_path():
    t = torch.zeros(2, 3, 4)
    v = torch.zeros(2)
    for call in (lambda: R.gated_scan(t, t), lambda: R.gated_step(t[0], t[0], t[0]), lambda: R.gated_scan_backward(t, t, t, t),
                 lambda: R.policy_loss(t[0], v.long(), v, v), lambda: R.AdamW([v])):
        with pytest.raises(ValueError):
            call()


def test_elements_that_share_memory():
    t = torch.zeros(4, 6)
    for ok in (t, t.t(), t[:, 1:3], t[::2], t[:0], t[1:2].expand(1, 6), t.view(2, 2, 6).transpose(0, 2)):
        own_elements(ok, "t")
    for bad in (t[:1].expand(4, 6), t.as_strided((4, 6), (3, 1)), t.as_strided((3, 3), (1, 1))):
        with pytest.raises(ValueError):
            own_elements(bad, "t")
