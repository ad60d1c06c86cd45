"""CPU checks of the training operators' C ABI: struct layouts and refusals
before any GPU work."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

from sandmuon_amd import _native

ROOT = Path(__file__).resolve().parents[1]
P = ctypes.c_void_p(256)


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc missing")
def test_qk_struct_layouts_match_header(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "sandmuon_amd.h"', "int main(void){"]
    for cname, cls in (("smx_qk_side", _native.QkSide), ("smx_qk_desc", _native.QkDesc)):
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["return 0;}"]))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(tmp_path / "layout.c"), "-o", str(exe)], check=True)
    got = dict(line.rsplit(" ", 1) for line in
               subprocess.run([str(exe)], capture_output=True, text=True).stdout.split("\n") if line)
    for cname, cls in (("smx_qk_side", _native.QkSide), ("smx_qk_desc", _native.QkDesc)):
        assert int(got[cname]) == ctypes.sizeof(cls)
        for f, _ in cls._fields_:
            assert int(got[f"{cname}.{f}"]) == getattr(cls, f).offset, (cname, f)


def test_act8_refusals():
    lib = _native.lib()
    ok = dict(dtype=1, rows=4, cols=40, stride=40, fmt=0, pitch=64)

    def encode(x=P, codes=P, scales=P, **kw):
        a = dict(ok, **kw)
        return lib.smx_act8_encode(x, a["dtype"], a["rows"], a["cols"], a["stride"], a["fmt"], codes, scales,
                                   a["pitch"], None)

    assert encode(dtype=3) == -3
    assert encode(fmt=2) == -1
    assert encode(rows=-1) == -2 and encode(stride=39) == -2
    assert encode(pitch=40) == -2 and encode(pitch=96) == -2
    assert encode(x=None) == -1 and encode(codes=None) == -1
    assert encode(codes=ctypes.c_void_p(8)) == -4
    assert encode(rows=0, x=None) == 0 and encode(cols=0, pitch=0, x=None) == 0
    assert lib.smx_act8_decode(P, P, 0, 4, 40, 64, None, 1, 40, None) == -1
    assert lib.smx_act8_gelu(P, 1, 4, 40, 40, 0, P, 40, P, P, P, None, 64, None) == -1
    assert lib.smx_act8_gelu_backward(P, 1, 4, 40, 40, None, P, 0, 64, P, 40, None) == -1
    need = lib.smx_act8_wgrad_workspace_bytes(4, 8, 40, 1)
    assert need >= 0 and lib.smx_act8_wgrad_workspace_bytes(-1, 8, 40, 1) == -1

    def wgrad(delta=P, dtype=1, rows=4, n=8, stride=8, fmt=0, k=40, pitch=64, dw=P, out=0):
        return lib.smx_act8_wgrad(delta, dtype, rows, n, stride, P, P, fmt, k, pitch, dw, None, out, P, need, None)

    assert wgrad(dtype=3) == -3 and wgrad(out=7) == -3 and wgrad(fmt=-1) == -1
    assert wgrad(stride=7) == -2 and wgrad(pitch=32) == -2 and wgrad(n=-1) == -2
    assert wgrad(delta=None) == -1 and wgrad(dw=None) == -1
    assert b"dw" in lib.smx_last_error()
    assert wgrad(n=0) == 0


def test_qk_refusals():
    lib = _native.lib()

    def desc(**kw):
        side = dict(x=256, y=256, heads=2, dy=256)
        side.update({k: kw.pop(k) for k in ("x", "y", "weight_dtype", "dw", "dy", "weight") if k in kw})
        fields = dict(cos=256, sin=256, table_rows=8, batch=1, seq=2, dim=64, rot=64, eps=1e-6, dtype=1, style=0)
        fields.update(kw)
        d = _native.QkDesc(**fields)
        d.q, d.k = _native.QkSide(**side), _native.QkSide(heads=0)
        return d

    call = lambda **kw: lib.smx_qk_norm_rotary(desc(**kw), None)
    assert call(dtype=5) == -3 and call(style=2) == -1 and call(eps=-1.0) == -1
    assert call(rot=63) == -2 and call(rot=66) == -2 and call(dim=0) == -2 and call(dim=1 << 20) == -2
    assert call(cos=None) == -1 and call(x=None) == -1 and call(weight=256, weight_dtype=9) == -3
    assert call(batch=1 << 16, seq=1 << 16) == -2
    assert lib.smx_qk_norm_rotary(None, None) == -1
    assert call(batch=0) == 0
    back = lambda **kw: lib.smx_qk_norm_rotary_backward(desc(**kw), None, 0, None)
    assert back(dy=None) == -1 and back(dw=256) == -1
    assert back(dw=256, weight=256) == -5
    assert lib.smx_qk_workspace_bytes(0) == -1


def test_loss_refusals():
    lib = _native.lib()

    def logprobs(z=P, dtype=1, batch=2, seq=3, vocab=50, bs=150, rs=50, targets=P, out=P):
        return lib.smx_token_logprobs(z, dtype, batch, seq, vocab, bs, rs, targets, None, out, None, None)

    assert logprobs(dtype=3) == -3 and logprobs(vocab=0) == -2 and logprobs(rs=49) == -2 and logprobs(batch=-1) == -2
    assert logprobs(z=None) == -1 and logprobs(targets=None) == -1 and logprobs(out=None) == -1
    assert logprobs(batch=1 << 20, seq=1 << 20) == -2
    assert logprobs(batch=0, z=None) == 0

    def policy(low=.2, high=.2, reduction=0, loss=P, work=P, bytes_=1 << 20, adv=P):
        return lib.smx_policy_loss(P, 1, 2, 3, 50, 150, 50, P, None, None, None, adv, 1, 0, low, high, 0.0, reduction,
                                   1.0, loss, P, P, work, bytes_, None)

    assert policy(low=-.1) == -1 and policy(low=1.1) == -1 and policy(high=-1.0) == -1 and policy(reduction=2) == -1
    assert policy(loss=None) == -1 and policy(adv=None) == -1 and policy(work=None) == -5 and policy(bytes_=4) == -5
    assert lib.smx_policy_loss_workspace_bytes(-1, 2) == -1
    assert lib.smx_preference_loss(P, P, None, 2, 3, .1, 1.5, P, P, P, None) == -1
    assert lib.smx_preference_loss(P, None, None, 2, 3, .1, 0.0, P, P, P, None) == -1
    assert lib.smx_preference_loss(P, P, None, -1, 3, .1, 0.0, P, P, P, None) == -2
    assert lib.smx_scale(P, 4, 1, P, None) == -3 and lib.smx_scale(None, 1, 1, P, None) == -1
    assert lib.smx_scale(None, 1, 0, None, None) == 0


def test_loss_stats_alignment():
    lib = _native.lib()
    assert lib.smx_token_logprobs(P, 1, 2, 3, 50, 150, 50, P, None, P, 260, None) == -4
    assert lib.smx_token_logprobs_backward(P, 1, 2, 3, 50, 150, 50, P, None, 260, P, 3, 1, None, P, None) == -4


def test_policy_loss_coef_refusals():
    lib = _native.lib()

    def call(z=P, low=.2, reduction=0, loss=P, adv=P, stats=P, coef=P, work=P, bytes_=1 << 20, batch=2):
        return lib.smx_policy_loss_coef(z, 2, batch, 3, 50, 150, 50, P, None, None, None, adv, 1, 0, low, .2, 0.0, reduction,
                                        1.0, loss, P, stats, coef, work, bytes_, None)

    assert call(z=None) == -1 and call(low=-.1) == -1 and call(reduction=2) == -1 and call(loss=None) == -1
    assert call(adv=None) == -1 and call(stats=None) == -1 and call(coef=None) == -1 and call(stats=ctypes.c_void_p(260)) == -4
    assert call(work=None) == -5 and call(bytes_=4) == -5 and call(batch=-1) == -2
    assert b"policy_loss_coef" in lib.smx_last_error()


def test_weight_gradient_of_no_outputs():
    lib = _native.lib()
    for k in (0, 40, 4096):
        for dtype in (0, 1, 2):
            assert lib.smx_act8_wgrad_workspace_bytes(4, 0, k, dtype) == 0
    assert lib.smx_act8_wgrad_workspace_bytes(4, 8, 0, 1) >= 0 and lib.smx_act8_wgrad_workspace_bytes(0, 8, 40, 1) >= 0
    # more features than a call takes: refused before the plan's products overflow
    for n, k in ((1 << 21, 8), (8, 1 << 21), (1 << 40, 1 << 40)):
        assert lib.smx_act8_wgrad_workspace_bytes(4, n, k, 1) == -2
