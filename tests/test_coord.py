"""The coordinator-side operators without a GPU: what their entries refuse is refused before anything is launched, calls of
no rows are nothing, and the 64-bit references the GPU tests use agree with the CPU checker and with closed forms."""
import ctypes as C

import numpy as np
import pytest

import b1_oracle as O
import coord_reference as R
from mimo26f_afd_amd import _lib, coord

P = 0x10000  # an address nothing is read from: every call below returns before a launch


def join_call(plan, rows=1, h=P, planes=(P,), h_out=P, **more):
    coord.Join(**plan)(rows, h, planes, h_out, **more)


def refused(fn, *args, **kw):
    with pytest.raises(coord.CoordError) as e:
        fn(*args, **kw)
    assert e.value.code == 1


GOOD = dict(cols=64, pre_weight=P)


@pytest.mark.parametrize("change", [dict(cols=0), dict(cols=-8), dict(cols=16385), dict(planes=0), dict(planes=5), dict(eps=0.0), dict(eps=-1e-6),
                                    dict(eps=float("nan")), dict(eps=float("inf")), dict(scale=float("nan")), dict(scale=float("inf")),
                                    dict(plane_pitch=63), dict(h_pitch=63), dict(norm_pitch=63), dict(gate_cols=2), dict(gate_cols=64, gate_pitch=63),
                                    dict(gate_cols=1, gate_pitch=-1), dict(pre_weight=None), dict(pre_weight=P + 2), dict(post_weight=P + 1)])
def test_join_refuses_bad_plans(change):
    plan = dict(GOOD, **change)
    refused(join_call, plan, planes=(P,) * plan.get("planes", 1) if plan.get("planes", 1) <= 4 else (P,) * 5, norm=P, gate=P)


def test_join_refuses_bad_calls():
    refused(join_call, GOOD, rows=-1)
    refused(join_call, GOOD, h=None)
    refused(join_call, GOOD, h=P + 2)
    refused(join_call, GOOD, planes=(None,))
    refused(join_call, GOOD, planes=(P + 1,))
    refused(join_call, GOOD, planes=(P, P))                          # two planes under a plan of one
    refused(join_call, GOOD, h_out=None)                             # nothing to write
    refused(join_call, GOOD, norm=P + 1)
    refused(join_call, GOOD, payload=P)                              # codes without scales
    refused(join_call, GOOD, scales=P)
    refused(join_call, dict(GOOD, cols=48), payload=P, scales=P)     # not whole blocks
    refused(join_call, dict(GOOD, payload_pitch=63), payload=P, scales=P)
    refused(join_call, dict(GOOD, cols=128, scales_pitch=3), payload=P, scales=P)
    refused(join_call, dict(GOOD, gate_cols=64))                     # a gate is announced and missing
    refused(join_call, dict(GOOD, gate_cols=1), gate=P + 2)
    join_call(GOOD, rows=0)                                          # no rows: nothing to do


def test_w4_refuses_bad_weights_and_calls():
    for args in ((None, P, 16, 64), (P, None, 16, 64), (P, P, 0, 64), (P, P, 16, 0), (P, P, 16, 48), (P + 8, P, 16, 64), (P, P, -4, 64),
                 (P, P, 1 << 27, 32), (P, P, 16, 1 << 25)):
        refused(coord.Weights4, *args)
    lib = _lib.load()
    assert lib.m26c_w4_matvec(None, P, 64, 1, P, 0, 64, None) == 1
    assert lib.m26c_w4_matvec_fp8(None, P, 64, P, 2, 1, P, 0, 64, None) == 1
    assert lib.m26c_w4_new(P, P, 16, 64, None, None, None, 0) == 1
    lib.m26c_w4_free(None)


def logprob_call(logits=P, bf16=False, rows=2, vocab=100, pitch=100, given=P, n_given=1, given_logprob=P, entropy=P, top=3, top_ids=P,
                 top_logprob=P, workspace=P, workspace_bytes=1 << 30, scale=1.0):
    coord.token_logprobs(logits, bf16, rows, vocab, pitch, given, n_given, given_logprob, entropy, top, top_ids, top_logprob, workspace,
                         workspace_bytes, scale=scale)


@pytest.mark.parametrize("change", [dict(logits=None), dict(logits=P + 2), dict(logits=P + 1, bf16=True), dict(rows=-1), dict(vocab=0), dict(pitch=99),
                                    dict(given=None), dict(given_logprob=None), dict(n_given=-1), dict(given=P + 2), dict(entropy=P + 1), dict(top=-1),
                                    dict(top=33), dict(top=4, vocab=3), dict(top_ids=None), dict(top_logprob=None), dict(scale=0.0), dict(scale=-1.0),
                                    dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=2.0 ** 20 * (1 + 2.0 ** -20)),
                                    dict(vocab=(1 << 30) + 1, pitch=1 << 31), dict(n_given=(1 << 30) + 1), dict(rows=1, vocab=131072, pitch=131072, workspace=None),
                                    dict(rows=1, vocab=131072, pitch=131072, workspace=P + 8),
                                    dict(rows=1, vocab=131072, pitch=131072, workspace_bytes=16)])
def test_logprobs_refuse(change):
    refused(logprob_call, **change)


@pytest.mark.parametrize("past", [1 << 32, -(1 << 32)])
def test_sizes_past_an_int_are_refused_not_wrapped(past):
    """A size that C's int does not hold would come through as another one, and a part of the rows be answered."""
    for change in (dict(rows=past + 2), dict(vocab=past + 100, pitch=1 << 33), dict(n_given=past + 1), dict(top=past + 3)):
        refused(logprob_call, **change)
    assert coord.token_logprobs_workspace(past + 1, 131072, 5) == 0 and coord.token_logprobs_workspace(1, past + 131072, 5) == 0
    for change in (dict(cols=past + 64, plane_pitch=1 << 33, h_pitch=1 << 33, norm_pitch=1 << 33), dict(planes=past + 1), dict(gate_cols=past)):
        refused(join_call, dict(GOOD, **change), norm=P, gate=P)
    weights = coord.Weights4.__new__(coord.Weights4)                  # no handle: nothing would run
    weights._h, weights.n, weights.k = C.c_void_p(), 16, 64
    ran = []
    weights._bf16 = weights._fp8 = lambda *a: ran.append(a) or 0
    refused(weights.matvec, P, past + 1, P)
    refused(weights.matvec_fp8, P, P, past + 1, P)
    assert not ran


def test_logprobs_of_no_rows_and_their_workspace():
    logprob_call(rows=0)
    assert coord.token_logprobs_workspace(0, 1000, 5) == 0 and coord.token_logprobs_workspace(-1, 1000, 5) == 0
    assert coord.token_logprobs_workspace(1, 100, 5) == 0
    need = coord.token_logprobs_workspace(1, 131072, 32)
    assert 0 < need < 1 << 20
    assert coord.token_logprobs_workspace(1, 131072, 33) == 0 and coord.token_logprobs_workspace(1, 131072, -1) == 0


def test_logprobs_workspace_bound_for_any_call():
    """What the header promises, so that a program can set one workspace aside for batches of any size."""
    sizes = sorted({max(1, (1 << b) + d) for b in range(0, 31) for d in (-1, 0, 1) if (1 << b) + d <= 1 << 30} | {50003, 9000, 8193, 200000, 262144})
    for vocab in sizes:
        for rows in (*range(1, 700, 7), 1024, 4096, 8191, 8192, 8193, 1 << 20, (1 << 31) - 1):
            for top in (0, 1, 32):
                assert coord.token_logprobs_workspace(rows, vocab, top) <= 8192 * (16 + 8 * top), (rows, vocab, top)


def test_join_plan_layout_matches_the_header():
    """The ctypes structure has the header's fields in the header's order."""
    import os
    import re
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "m26c_coord.h")).read()
    body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct m26c_join \{(.*?)\} m26c_join;", text, re.S).group(1), flags=re.S)
    names = [w for decl in body.split(";") for w in re.findall(r"(\w+)\s*(?:,|$)", re.sub(r"^\s*(?:const\s+)?\w+\s*\**", "", decl.strip()))]
    assert names == [n for n, _ in coord._JoinPlan._fields_]
    assert C.sizeof(coord._JoinPlan) == 2 * 4 + 3 * 8 + 2 * 8 + (4 + 4) + 8 + 2 * 4 + 2 * 8  # gate_cols is padded to eight bytes


def test_references_agree_with_the_checker():
    rng = np.random.default_rng(1)
    payload = rng.integers(0, 256, (5, 32), dtype=np.uint8)
    scales = rng.integers(2, 250, (5, 2), dtype=np.uint8)
    w = R.w4_weights(payload, scales)
    assert np.array_equal(w, np.asarray(O.mxfp4_rows(payload, scales), np.float64).reshape(5, 64))
    x = (rng.standard_normal((3, 128)) * 4).astype(np.float32)
    p, s = O.q0_quantize(x)
    back = R.wire_values(p, s)
    assert np.max(np.abs(back - x) / np.maximum(np.abs(x), np.repeat(np.abs(x).reshape(3, 4, 32).max(-1), 32, -1).reshape(3, 128) * 2.0 ** -9)) <= 2 * R.UE4M3


def test_logprob_reference_closed_forms():
    x = np.zeros((2, 8))
    x[1] = -np.inf
    x[1, 3] = 5.0
    g, h, ids, lp, *_ = R.logprobs(x, np.array([[0, 9], [3, 0]]), 3, 2.0)
    assert np.allclose(g[0, 0], -np.log(8)) and np.isnan(g[0, 1]) and g[1, 0] == 0 and g[1, 1] == -np.inf
    assert np.allclose(h, [np.log(8), 0]) and ids.tolist() == [[0, 1, 2], [3, -1, -1]] and lp[1].tolist() == [0, -np.inf, -np.inf]
