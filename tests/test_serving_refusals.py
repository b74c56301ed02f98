"""What the C entries of the scoring and paged-cache operators refuse, without a GPU: every bad argument is answered on the host,
with a code and a message, before anything is launched; and the tensor wrappers refuse CPU tensors."""
import ctypes
import math

import pytest
import torch

from ttts_amd import lib as l
from ttts_amd import ops
from ttts_amd.lib import TttsError

EINVAL = -1


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as ge
    ge.build()
    return l.get()


def _p(n=1 << 20):
    """A non-null 16-byte aligned address that nothing looks at."""
    return ctypes.c_void_p(n)


def _call(lib, fn, good, **change):
    args = dict(good, **change)
    return getattr(lib, fn)(*args.values())


def _refused(lib, fn, good, word, **change):
    assert _call(lib, fn, good, **change) == EINVAL, change
    msg = lib.ttts_last_error().decode()
    assert word in msg, (change, msg)


FWD = dict(logits=_p(), dtype=0, ldl=16, tokens=_p(), logp=_p(), entropy=_p(), stats=_p(), top_logp=_p(), top_idx=_p(), R=4, C=10, top_k=3,
           temperature=1.0, ws=_p(), nbytes=1 << 30, stream=None)
BWD = dict(logits=_p(), dtype=1, ldl=16, tokens=_p(), stats=_p(), entropy=_p(), g_logp=_p(), g_entropy=None, dlogits=_p(), ldd=16, R=4, C=10,
           Cd=16, temperature=1.0, stream=None)
DFWD = dict(logits=_p(), dtype=2, ldl=16, idx=_p(), val=_p(), loss=_p(), stats=_p(), R=4, C=10, K=3, temperature=1.0, tail=1, ws=_p(),
            nbytes=1 << 30, stream=None)
DBWD = dict(logits=_p(), dtype=0, ldl=16, idx=_p(), val=_p(), stats=_p(), g=_p(), dlogits=_p(), ldd=16, R=4, C=10, Cd=16, K=3, temperature=1.0,
            tail=0, accumulate=0, stream=None)


@pytest.mark.parametrize("fn,good", [("ttts_token_logprobs_fwd", FWD), ("ttts_token_logprobs_bwd", BWD), ("ttts_distill_fwd", DFWD),
                                     ("ttts_distill_bwd", DBWD)])
def test_row_operators_refuse(lib, fn, good):
    name = fn[len("ttts_"):]
    for change in (dict(dtype=3), dict(dtype=-1), dict(R=-1), dict(C=0), dict(C=17), dict(C=l.SCORE_MAX_CLASSES + 1, ldl=1 << 22),
                   dict(temperature=0.0), dict(temperature=-2.0), dict(temperature=math.inf), dict(temperature=math.nan), dict(temperature=1e-39),
                   dict(logits=None), dict(logits=_p((1 << 20) + 1))):
        _refused(lib, fn, good, name, **change)
    for key in good:
        if isinstance(good[key], ctypes.c_void_p) and key != "ws":
            _refused(lib, fn, good, "null", **{key: None})
    if "Cd" in good:
        _refused(lib, fn, good, "Cd", Cd=9)
        _refused(lib, fn, good, "Cd", ldd=15)
    if "K" in good:
        _refused(lib, fn, good, "K", K=0)
        _refused(lib, fn, good, "K", K=l.DISTILL_MAX_K + 1)
    if "top_k" in good:
        _refused(lib, fn, good, "top_k", top_k=-1)
        _refused(lib, fn, good, "top_k", top_k=l.SCORE_MAX_TOP + 1)
    assert _call(lib, fn, good, R=0) == 0                  # no rows: nothing is launched


def test_workspaces_are_checked(lib):
    """Where a call needs scratch, a missing, short or misaligned one is refused; the sizes grow with the rows."""
    for fn, good, need in (("ttts_token_logprobs_fwd", dict(FWD, C=300000, ldl=300000), lambda R: lib.ttts_token_logprobs_workspace_bytes(R, 300000, 3)),
                           ("ttts_distill_fwd", dict(DFWD, C=300000, ldl=300000), lambda R: lib.ttts_distill_workspace_bytes(R, 300000)),
                           ("ttts_attn_paged_decode", ATT, lambda M: lib.ttts_attn_paged_decode_workspace_bytes(M, 4, 2, 64, 16, ATT["width"]))):
        n = need(4)
        if n == 0:
            continue
        assert n % 16 == 0
        _refused(lib, fn, good, "workspace", nbytes=n - 1)
        _refused(lib, fn, good, "workspace", ws=None)
        _refused(lib, fn, good, "workspace", ws=_p((1 << 20) + 8))


ATT = dict(q=_p(), qm=256, qh=64, k=_p(), v=_p(), table=_p(), ts=500, lens=_p(), out=_p(), om=256, oh=64, lse=_p(), dtype=1, M=4, H=4, Hkv=2, dh=64,
           page=16, P=9, width=500, scale=0.125, ws=_p(), nbytes=1 << 30, stream=None)
WRITE = dict(k=_p(), v=_p(), ksn=128, ksh=64, vsn=128, vsh=64, kp=_p(), vp=_p(), slots=_p(), dtype=2, N=4, H=2, dh=64, page=16, P=9, stream=None)


@pytest.mark.parametrize("fn,good", [("ttts_attn_paged_decode", ATT), ("ttts_kv_page_write", WRITE)])
def test_paged_operators_refuse(lib, fn, good):
    name = fn[len("ttts_"):]
    heads = "Hkv" if "Hkv" in good else "H"
    for change in (dict(dtype=0), dict(dtype=5), dict(dh=48), dict(dh=256), dict(page=8), dict(page=48), dict(page=2048), dict(P=0), {heads: 0}):
        _refused(lib, fn, good, name, **change)
    for key in good:
        if isinstance(good[key], ctypes.c_void_p) and key != "ws":
            _refused(lib, fn, good, "null", **{key: None})
            if key not in ("table", "lens", "lse", "slots"):
                _refused(lib, fn, good, "aligned", **{key: _p((1 << 20) + 2)})
    for key in ("qm", "qh", "om", "oh", "ksn", "ksh", "vsn", "vsh"):
        if key in good:
            _refused(lib, fn, good, "strides", **{key: good[key] + 4})
    if "M" in good:
        for change in (dict(M=-1), dict(H=5), dict(H=0), dict(width=0), dict(ts=499), dict(width=1 << 28, ts=1 << 28), dict(scale=math.inf), dict(scale=math.nan)):
            _refused(lib, fn, good, name, **change)
        assert _call(lib, fn, good, M=0) == 0
    else:
        _refused(lib, fn, good, name, N=-1)
        assert _call(lib, fn, good, N=0) == 0


def test_wrappers_refuse_cpu_tensors():
    x, tok = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64)
    i, t, v = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3), torch.zeros(2)
    kp = torch.zeros(2, 1, 16, 32, dtype=torch.bfloat16)
    k = torch.zeros(2, 1, 32, dtype=torch.bfloat16)
    calls = [lambda: ops.token_logprobs_fwd(x, tok), lambda: ops.token_logprobs_bwd(x, tok, torch.zeros(2, 2), v, v), lambda: ops.distill_fwd(x, i, t),
             lambda: ops.distill_bwd(x, i, t, torch.zeros(2, 3), v), lambda: ops.kv_page_write(k, k, kp, kp, tok),
             lambda: ops.attn_paged_decode(k, kp, kp, torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 1.0)]
    for f in calls:
        with pytest.raises(TttsError, match="must live on the GPU"):
            f()


def test_more_than_one_launch_holds(lib):
    """2^32 threads of one launch, or more: refused by name, nothing is launched."""
    big = 1 << 30
    _refused(lib, "ttts_token_logprobs_fwd", FWD, "one launch", R=big)
    _refused(lib, "ttts_token_logprobs_bwd", BWD, "one launch", R=(1 << 31) - 1, C=16)
    _refused(lib, "ttts_distill_fwd", DFWD, "one launch", R=big)
    _refused(lib, "ttts_distill_bwd", DBWD, "one launch", R=big)
    _refused(lib, "ttts_kv_page_write", WRITE, "one launch", N=big, H=64, ksn=4096, vsn=4096)
    _refused(lib, "ttts_attn_paged_decode", ATT, "one launch", M=big, width=4)


@pytest.mark.parametrize("units", range(1, 10))
def test_a_split_sequence_has_no_more_parts_than_its_join_holds(lib, units):
    """The parts of the longest tables (2^30 keys), read off the workspace: the join keeps the weights of 2048 of them."""
    for M, Hkv in {(units, 1), (1, units)}:
        for log_page in (4, 7, 10):
            for keys in [1 << n for n in range(12, 31)] + [2048 * 4096 + 1024, 5 * 10 ** 7, 10 ** 9]:
                width = keys >> log_page
                n = lib.ttts_attn_paged_decode_workspace_bytes(M, Hkv, Hkv, 32, 1 << log_page, width)
                assert n // (M * Hkv * (32 + 2) * 4) <= 2048, (M, Hkv, keys)


@pytest.mark.parametrize("fn,good", [("ttts_token_logprobs_fwd", FWD), ("ttts_token_logprobs_bwd", BWD), ("ttts_distill_fwd", DFWD),
                                     ("ttts_distill_bwd", DBWD)])
def test_temperatures_whose_reciprocal_in_bits_overflows(lib, fn, good):
    """1 / temperature times log2 e is the exponents' factor: where that is not finite every exponent of a row's maximum would be NaN."""
    for T in (3.4e-39, 4.0e-39, 4.2e-39):
        _refused(lib, fn, good, "temperature", temperature=T)
    assert _call(lib, fn, good, R=0, temperature=5.0e-39) == 0


@pytest.mark.parametrize("scale", [2.4e38, -2.4e38, 3.4e38])
def test_scales_that_overflow_in_bits(lib, scale):
    """scale times log2 e multiplies the scores: infinite, a score of 0 would be NaN."""
    _refused(lib, "ttts_attn_paged_decode", ATT, "scale", scale=scale)
    assert _call(lib, "ttts_attn_paged_decode", ATT, M=0, scale=2.3e38 if scale > 0 else -2.3e38) == 0


def test_workspaces_that_are_needed_are_asked_for(lib):
    """The three calls whose scratch is checked above do need some (more for more rows; the attention splits more sequences into fewer parts);
    calls that one launch answers need none."""
    for need in (lambda n: lib.ttts_token_logprobs_workspace_bytes(n, 300000, 3), lambda n: lib.ttts_distill_workspace_bytes(n, 300000)):
        assert 0 < need(4) and need(8) == 2 * need(4)
    assert lib.ttts_attn_paged_decode_workspace_bytes(4, 4, 2, 64, 16, ATT["width"]) > 0
    assert lib.ttts_token_logprobs_workspace_bytes(4, 2048, 3) == lib.ttts_distill_workspace_bytes(4, 2048) == 0
    assert lib.ttts_attn_paged_decode_workspace_bytes(4, 4, 2, 64, 16, 40) == 0
