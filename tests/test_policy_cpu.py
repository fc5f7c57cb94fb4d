"""What the operators of ``multigrid_amd.policy`` refuse, checked without a GPU: through the C entry points, whose checks come
before anything is launched, and through the Python functions."""
import ctypes
import os

import pytest

torch = pytest.importorskip("torch")

from multigrid_amd import _lib, policy  # noqa: E402
from multigrid_amd._lib import MgAdjust, MgEmbed, MgLogits  # noqa: E402

needs_lib = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="libmgrid_hip.so not built")
P = ctypes.c_void_p(4096)  # an address that nothing reads: every call below is refused first, or has no rows


def embed_spec(**more):
    e = MgEmbed(n=4, fields=3, dim=8, ids_type=_lib.U8, dtype=_lib.F32, ids_stride=3, field_stride=1, row_stride=8, scale=1.0)
    e.sizes[:3] = (11, 6, 7)
    for k, v in more.items():
        if k == "size0":
            e.sizes[0] = v
        else:
            setattr(e, k, v)
    return e


@needs_lib
@pytest.mark.parametrize("more,word", [
    (dict(n=-1), "n -1"), (dict(n=1 << 31), "n 2147483648"), (dict(fields=0), "fields"), (dict(fields=9), "fields"), (dict(dim=0), "dim"),
    (dict(dim=(1 << 20) + 1), "dim"), (dict(ids_type=3), "type"), (dict(dtype=3), "type"), (dict(ids_stride=-1), "stride"), (dict(row_stride=-1), "stride"),
    (dict(field_stride=-1), "stride"), (dict(size0=0), "field 0"), (dict(size0=-5), "field 0"), (dict(size0=(1 << 30)), "rows"), (dict(reserved0=1), "reserved0")])
def test_embed_refuses(more, word):
    L = _lib.lib()
    e = embed_spec(**more)
    for rc in (L.mg_embed(ctypes.byref(e), P, P, P, None), L.mg_embed_grad(ctypes.byref(e), P, P, P, P, 1 << 40, None),
               L.mg_embed_grad_workspace(ctypes.byref(e))):
        assert rc == -1 and word in L.mg_last_error(None).decode()


@needs_lib
def test_embed_refuses_missing_pointers_and_workspaces():
    L = _lib.lib()
    e = ctypes.byref(embed_spec())
    assert L.mg_embed(None, P, P, P, None) == -1 and L.mg_embed_grad(None, P, P, P, P, 0, None) == -1 and L.mg_embed_grad_workspace(None) == -1
    for args in ((None, P, P), (P, None, P), (P, P, None)):
        assert L.mg_embed(e, *args, None) == -1 and b"null" in L.mg_last_error(None)
        assert L.mg_embed_grad(e, *args, P, 1 << 40, None) == -1 and b"null" in L.mg_last_error(None)
    assert L.mg_embed(ctypes.byref(embed_spec(n=0)), None, None, None, None) == 0  # nothing to do
    for big in (dict(n=100000), dict(n=100000, size0=5000), dict(n=5000, size0=5000, fields=1)):
        e = embed_spec(**big)
        need = L.mg_embed_grad_workspace(ctypes.byref(e))
        assert need >= 0
        if need:
            assert L.mg_embed_grad(ctypes.byref(e), P, P, P, P, need - 1, None) == -1 and b"workspace" in L.mg_last_error(None)
            assert L.mg_embed_grad(ctypes.byref(e), P, P, P, None, need, None) == -1 and b"workspace" in L.mg_last_error(None)
            assert L.mg_embed_grad(ctypes.byref(e), P, P, P, ctypes.c_void_p(4100), need, None) == -1 and b"workspace" in L.mg_last_error(None)


def adjust_spec(**more):
    a = MgAdjust(n=4, k=9, dtype=_lib.F32, logits_stride=9, out_stride=9, grad_stride=9, history_dev=4096, history_stride=5, history_type=_lib.I64, t=5,
                 repetition=1.0)
    for k, v in more.items():
        setattr(a, k, v)
    return a


@needs_lib
@pytest.mark.parametrize("more,word", [
    (dict(n=-1), "n -1"), (dict(k=0), "k 0"), (dict(k=(1 << 24) + 1), "k "), (dict(dtype=7), "type"), (dict(t=-1), "history"), (dict(history_type=3), "history"),
    (dict(t=(1 << 24) + 1), "history"), (dict(mask_kind=3), "mask"), (dict(mask_kind=1), "mask"), (dict(mask_kind=2), "mask"), (dict(logits_stride=-9), "stride"), (dict(mask_stride=-1), "stride"),
    (dict(bias_stride=-1), "stride"), (dict(history_stride=-1), "stride"), (dict(grad_stride=-1), "stride"), (dict(out_stride=8), "overlap"), (dict(repetition=0.0), "repetition"),
    (dict(repetition=-1.0), "repetition"), (dict(repetition=float("nan")), "repetition"), (dict(repetition=float("inf")), "repetition")])
def test_adjust_refuses(more, word):
    L = _lib.lib()
    a = adjust_spec(**more)
    for rc in (L.mg_adjust_logits(ctypes.byref(a), P, P, None), L.mg_adjust_logits_grad(ctypes.byref(a), P, P, P, None)):
        assert rc == -1 and word in L.mg_last_error(None).decode()


@needs_lib
def test_adjust_refuses_missing_pointers():
    L = _lib.lib()
    assert L.mg_adjust_logits(None, P, P, None) == -1 and L.mg_adjust_logits_grad(None, P, P, P, None) == -1
    a = ctypes.byref(adjust_spec())
    assert L.mg_adjust_logits(a, None, P, None) == -1 and L.mg_adjust_logits(a, P, None, None) == -1
    for args in ((None, P, P), (P, None, P), (P, P, None)):
        assert L.mg_adjust_logits_grad(a, *args, None) == -1 and b"null" in L.mg_last_error(None)
    assert L.mg_adjust_logits(ctypes.byref(adjust_spec(n=0)), None, None, None) == 0


def logits_spec(**more):
    l = MgLogits(n=4, k=9, dtype=_lib.F32, stride=9, temperature=1.0, tokens_type=_lib.I64)
    for k, v in more.items():
        setattr(l, k, v)
    return l


@needs_lib
@pytest.mark.parametrize("more,word", [
    (dict(n=-1), "n -1"), (dict(n=1 << 31), "n "), (dict(k=0), "k 0"), (dict(k=(1 << 24) + 1), "k "), (dict(dtype=3), "type"), (dict(tokens_type=3), "tokens"),
    (dict(tokens_type=_lib.U8, k=256), "tokens"), (dict(stride=-1), "stride"), (dict(temperature=0.0), "temperature"), (dict(temperature=1e-40), "temperature"), (dict(temperature=-1.0), "temperature"),
    (dict(temperature=float("nan")), "temperature"), (dict(temperature=float("inf")), "temperature")])
def test_draw_and_logprobs_refuse(more, word):
    L = _lib.lib()
    l = logits_spec(**more)
    r = ctypes.byref(l)
    for rc in (L.mg_draw(r, P, P, _lib.F32, P, P, P, 1 << 40, None), L.mg_token_logprobs(r, P, P, P, P, P, P, 1 << 40, None),
               L.mg_token_logprobs_grad(r, P, P, P, P, 1, P, 1, P, None), L.mg_draw_workspace(r), L.mg_token_logprobs_workspace(r)):
        assert rc == -1 and word in L.mg_last_error(None).decode()


@needs_lib
def test_draw_and_logprobs_refuse_missing_pointers():
    L = _lib.lib()
    r = ctypes.byref(logits_spec())
    assert L.mg_draw(None, P, P, 0, P, P, P, 0, None) == -1 and L.mg_token_logprobs(None, P, P, P, P, P, P, 0, None) == -1
    assert L.mg_draw(r, None, P, 0, P, P, P, 0, None) == -1 and L.mg_draw(r, P, P, 0, None, P, P, 0, None) == -1
    assert L.mg_draw(r, P, P, _lib.BF16, P, P, P, 0, None) == -1 and b"uniform" in L.mg_last_error(None)
    assert L.mg_token_logprobs(r, None, P, P, P, P, P, 0, None) == -1 and L.mg_token_logprobs(r, P, None, P, P, P, P, 0, None) == -1
    assert L.mg_token_logprobs(r, P, P, P, P, ctypes.c_void_p(4104), P, 1 << 40, None) == -1 and b"aligned" in L.mg_last_error(None)
    long = ctypes.byref(logits_spec(k=33, stride=33))
    for args in ((None, P, P, P, 1, P, 1, P), (P, None, P, P, 1, P, 1, P), (P, P, P, P, 1, P, 1, None),
                 (P, P, ctypes.c_void_p(4104), P, 1, P, 1, P), (P, P, P, P, -1, P, 1, P), (P, P, P, P, 1, P, -1, P)):
        assert L.mg_token_logprobs_grad(r, *args, None) == -1
        assert L.mg_token_logprobs_grad(long, *args, None) == -1
    assert L.mg_token_logprobs_grad(long, P, P, None, P, 1, P, 1, P, None) == -1
    none = ctypes.byref(logits_spec(n=0))
    assert L.mg_draw(none, None, None, 0, None, None, None, 0, None) == 0
    assert L.mg_token_logprobs(none, None, None, None, None, None, None, 0, None) == 0
    for more in (dict(k=200000), dict(k=200000, n=1), dict(k=70000, n=3, dtype=_lib.F16)):
        l = logits_spec(**more)
        for size, call in ((L.mg_draw_workspace, lambda w, b: L.mg_draw(ctypes.byref(l), P, P, 0, P, P, w, b, None)),
                           (L.mg_token_logprobs_workspace, lambda w, b: L.mg_token_logprobs(ctypes.byref(l), P, P, P, P, P, w, b, None))):
            need = size(ctypes.byref(l))
            assert need >= 0
            if need:
                for w, b in ((P, need - 1), (None, need), (ctypes.c_void_p(4100), need)):
                    assert call(w, b) == -1 and b"workspace" in L.mg_last_error(None)


def test_tensors_on_the_cpu_are_refused():
    x, ids = torch.zeros((4, 7)), torch.zeros((4,), dtype=torch.int64)
    for call in (lambda: policy.embed(ids, x), lambda: policy.embed_grad(x, ids, 5), lambda: policy.adjust_logits(x), lambda: policy.draw(x),
                 lambda: policy.token_logprobs(x, ids), lambda: policy.adjust_logits(x, out=x)):
        with pytest.raises(ValueError, match="on a GPU"):
            call()


def test_the_structures_are_the_header_s():
    """Sizes and a few offsets of the ctypes structures, as the C compiler lays the header's out."""
    import subprocess
    import tempfile
    text = "#include <stdio.h>\n#include <stddef.h>\n#include \"mgrid.h\"\nint main(void) { printf(\"%zu %zu %zu %zu %zu %zu %zu\\n\", sizeof(MgEmbed), " \
           "offsetof(MgEmbed, sizes), sizeof(MgAdjust), offsetof(MgAdjust, repetition), offsetof(MgAdjust, mask_stride), sizeof(MgLogits), offsetof(MgLogits, tokens_type)); }\n"
    with tempfile.TemporaryDirectory() as d:
        src = os.path.join(d, "a.c")
        open(src, "w").write(text)
        subprocess.check_call(["gcc", "-I", _lib.INCLUDE_DIR, src, "-o", os.path.join(d, "a")])
        got = [int(v) for v in subprocess.check_output([os.path.join(d, "a")]).split()]
    assert got == [ctypes.sizeof(MgEmbed), MgEmbed.sizes.offset, ctypes.sizeof(MgAdjust), MgAdjust.repetition.offset, MgAdjust.mask_stride.offset,
                   ctypes.sizeof(MgLogits), MgLogits.tokens_type.offset]
