"""Refusals of the 8-bit products and of drawing tokens: every bad size, type,
stride or alignment is answered with SKB_ERR_ARG before anything touches a GPU,
so they are checked without one."""

from __future__ import annotations

import subprocess
import sys
import types

import pytest
import torch

A = 1 << 20  # stands for a 256-byte aligned device address; nothing reads it


@pytest.fixture(scope="module")
def lib():
    from soraku_tts_b200 import _lib
    from soraku_tts_b200.build import build

    build()
    return _lib


F32, BF16, F16, I8 = range(4)
QUANT = dict(x=A, x_type=F32, ldx=100, rows=3, K=100, norm_weight=A, eps=1e-6, q=A, ldq=112, scale=A, stream=None)
HEAD = dict(x=A, x_type=F32, ldx=100, x_scale=None, norm_weight=A, eps=1e-6, T=3, K=100)
TAIL = dict(out=A, out_type=F32, ldo=40, workspace=A, workspace_bytes=1 << 40, stream=None)
LINEAR = dict(HEAD, w=A, ldw=112, w_scale=A, N=40, bias=A, residual=A, ldr=40, **TAIL)
SWIGLU = dict(HEAD, gate=A, ldg=112, gate_scale=A, up=A, ldu=112, up_scale=A, I=40, **TAIL)
SAMPLE = dict(logits=A, type=F32, ld=100, rows=3, V=100, uniform=A, temperatures=None, temperature=1.0, top_ks=None, top_k=0,
              top_ps=None, top_p=1.0, min_ps=None, min_p=0.0, tokens=A, logprob=A, stream=None)

CODES = dict(x_type=I8, ldx=112, x_scale=A, norm_weight=None)
BAD_ROWS = [dict(x=None), dict(x_type=-1), dict(K=0), dict(K=-5), dict(K=131072, ldx=1 << 18, ldq=1 << 18, ldw=1 << 18, ldg=1 << 18,
            ldu=1 << 18), dict(ldx=99), dict(x=A + 2), dict(x=A + 1, x_type=BF16), dict(norm_weight=A + 2), dict(eps=-1.0),
            dict(eps=float("nan")), dict(eps=float("inf"))]
BAD_X = [dict(T=-1), dict(x_type=4), dict(x_scale=A), dict(CODES, x_scale=None), dict(CODES, norm_weight=A), dict(CODES, ldx=104),
         dict(CODES, ldx=96), dict(CODES, x=A + 8), dict(out=None), dict(out_type=I8), dict(out_type=-1), dict(ldo=39), dict(out=A + 2),
         dict(out=A + 1, out_type=BF16)]


def refused(lib, entry, args, change):
    args = dict(args, **{k: v for k, v in change.items() if k in args})
    assert getattr(lib.lib(), "skb_" + entry)(*args.values()) == lib.SKB_ERR_ARG
    assert entry in lib.last_error()


@pytest.mark.parametrize("change", BAD_ROWS + [dict(rows=-1), dict(x_type=I8), dict(q=None), dict(scale=None), dict(q=A + 8),
                                               dict(ldq=104), dict(ldq=96), dict(scale=A + 2)])
def test_quantize_rows_refuses(lib, change):
    refused(lib, "quantize_rows", QUANT, change)


@pytest.mark.parametrize("change", BAD_ROWS + BAD_X + [dict(w=None), dict(w_scale=None), dict(N=0), dict(N=-1), dict(w=A + 8),
                                                       dict(ldw=104), dict(ldw=96), dict(w_scale=A + 1), dict(ldr=39),
                                                       dict(residual=A + 2), dict(bias=A + 2)])
def test_int8_linear_refuses(lib, change):
    refused(lib, "int8_linear", LINEAR, change)


@pytest.mark.parametrize("change", BAD_ROWS + BAD_X + [dict(gate=None), dict(up=None), dict(gate_scale=None), dict(up_scale=None),
                                                       dict(I=0), dict(gate=A + 4), dict(up=A + 4), dict(ldg=104), dict(ldu=96),
                                                       dict(up_scale=A + 1)])
def test_int8_swiglu_refuses(lib, change):
    refused(lib, "int8_swiglu", SWIGLU, change)


@pytest.mark.parametrize("change", [dict(workspace=None), dict(workspace=A + 8), dict(workspace_bytes=16)])
def test_products_of_many_tokens_need_their_workspace(lib, change):
    sizes = dict(T=500, K=1000, ldx=1000)
    assert lib.lib().skb_int8_workspace(500, 1000, F32) > 0
    assert lib.lib().skb_int8_workspace(500, 1000, I8) == 0
    refused(lib, "int8_linear", LINEAR, dict(sizes, ldw=1008, **change))
    refused(lib, "int8_swiglu", SWIGLU, dict(sizes, ldg=1008, ldu=1008, **change))


@pytest.mark.parametrize("change", [dict(logits=None), dict(uniform=None), dict(tokens=None), dict(logprob=None), dict(type=I8),
                                    dict(type=-1), dict(rows=-1), dict(rows=1 << 28), dict(V=0), dict(V=(1 << 18) + 1, ld=1 << 19),
                                    dict(ld=99), dict(logits=A + 2), dict(uniform=A + 2), dict(temperatures=A + 1),
                                    dict(top_ks=A + 2), dict(top_ps=A + 2), dict(min_ps=A + 2), dict(tokens=A + 4),
                                    dict(logprob=A + 2)])
def test_sample_tokens_refuses(lib, change):
    refused(lib, "sample_tokens", SAMPLE, change)


@pytest.mark.parametrize("entry,args", [("quantize_rows", dict(QUANT, rows=0)), ("int8_linear", dict(LINEAR, T=0)),
                                        ("int8_swiglu", dict(SWIGLU, T=0)), ("sample_tokens", dict(SAMPLE, rows=0))])
def test_no_rows_is_no_work(lib, entry, args):
    assert getattr(lib.lib(), "skb_" + entry)(*args.values()) == lib.SKB_OK


def test_python_layer_refuses_cpu_tensors():
    from soraku_tts_b200 import kernels as K

    x, w = torch.zeros(2, 32), K.Int8Rows(torch.zeros(4, 32, dtype=torch.int8), torch.zeros(4))
    for call in (lambda: K.quantize_rows(x), lambda: K.int8_linear(x, w), lambda: K.int8_swiglu(x, w, w),
                 lambda: K.sample_tokens(x, torch.zeros(2)), lambda: K.int8_linear(w, w), lambda: K.int8_linear(None, w)):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------- the short way from Python
def cut_off(monkeypatch):
    """As if the extension module had not been built."""
    import soraku_tts_b200
    from soraku_tts_b200 import _lib

    monkeypatch.setattr(_lib, "_bind", None)
    monkeypatch.delattr(soraku_tts_b200, "_bind", raising=False)
    monkeypatch.setitem(sys.modules, "soraku_tts_b200._bind", None)


def test_without_the_short_way_calls_go_through_ctypes(lib, monkeypatch):
    from soraku_tts_b200 import kernels as K

    cut_off(monkeypatch)
    with pytest.warns(RuntimeWarning, match="_bind"):
        short = lib.bind()
    assert short.product(*range(9)) is None and short.quantize(1, 2, 3) is None and short.sample(*range(6)) is None
    with pytest.raises(ValueError, match="CUDA"):
        K.quantize_rows(torch.zeros(2, 32))


def test_the_short_way_is_not_taken_with_another_torch(lib, monkeypatch):
    from soraku_tts_b200 import build

    assert lib.bind().built_for == build.bind_key()
    monkeypatch.setattr(lib, "_bind", None)
    monkeypatch.setattr(torch, "__version__", "1.0.0")
    with pytest.warns(RuntimeWarning, match="torch 1.0.0"):
        assert lib.bind().product(*range(9)) is None


def test_the_short_way_is_not_taken_when_it_does_not_say_what_it_was_built_for(lib, monkeypatch):
    import soraku_tts_b200

    monkeypatch.setattr(lib, "_bind", None)
    monkeypatch.setattr(soraku_tts_b200, "_bind", types.ModuleType("_bind"), raising=False)
    with pytest.warns(RuntimeWarning, match="unknown"):
        assert lib.bind().product(*range(9)) is None


@pytest.mark.parametrize("change", [dict(CXX="other-g++"), dict(torch="9.9.9"), dict(file="elsewhere"), dict(stamp=None), dict(fail=1)])
def test_the_short_way_is_built_again_when_what_it_was_built_for_changes(lib, monkeypatch, tmp_path, change):
    from soraku_tts_b200 import build

    runs = []

    def run(cmd, **kw):
        runs.append(cmd)
        if "fail" not in change:
            open(cmd[cmd.index("-o") + 1], "w").close()
        return subprocess.CompletedProcess(cmd, 1 if "fail" in change else 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", run)
    monkeypatch.setattr(build, "HERE", str(tmp_path))
    monkeypatch.setattr(build, "BIND", str(tmp_path / "_bind.x.so"))
    monkeypatch.setattr(build, "BIND_STAMP", str(tmp_path / "bind.txt"))
    (tmp_path / "_bind.so").touch()  # of a build that gave it no ABI
    if "fail" in change:  # what was there before is not loaded
        with pytest.raises(RuntimeError):
            build._build_bind(False)
        assert not list(tmp_path.iterdir())
        return
    build._build_bind(False)
    build._build_bind(False)
    assert len(runs) == 1 and not (tmp_path / "_bind.so").exists()
    if "CXX" in change:
        monkeypatch.setattr(build, "CXX", change["CXX"])
    elif "torch" in change:
        monkeypatch.setattr(torch, "__version__", change["torch"])
    elif "file" in change:
        monkeypatch.setattr(torch, "__file__", str(tmp_path / change["file"] / "__init__.py"))
    else:
        (tmp_path / "bind.txt").unlink()
    build._build_bind(False)
    build._build_bind(False)
    assert len(runs) == 2


def test_the_library_is_built_without_the_short_way(lib, monkeypatch):
    from soraku_tts_b200 import build

    def fails(force):
        raise RuntimeError("no headers")

    monkeypatch.setattr(build, "_build_bind", fails)
    with pytest.warns(RuntimeWarning, match="longer way"):
        assert build.build() == build.LIB
