"""The decoder-attention operators without a GPU: the prompt planner's schedule,
refusals at the C boundary, and the 64-bit forms the GPU tests compare with."""
import ctypes

import numpy as np
import pytest

import bsp
import decoder_ref as ref


def inspect(ql, kl, heads, kv_heads, d=128, causal=True, **opts):
    p = bsp.inspect_prompt_plan(ql, kl, heads, kv_heads, d, causal, bsp.make_opts(**opts))
    return p, p["unit_table"], p["cta_begin"]


CASES = [([1], [1], 1, 1), ([37], [37], 8, 2), ([2048, 513, 1, 0, 96], [2048, 700, 600, 5, 96], 32, 8),
         ([5, 300], [2, 100], 6, 2), ([4000], [4000], 5, 1), ([7] * 300, [7] * 300, 64, 1), ([3], [0], 4, 2)]


@pytest.mark.parametrize("ql,kl,heads,kv_heads", CASES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("max_ctas", [0, 5])
def test_prompt_units_cover_every_row_and_key_once(ql, kl, heads, kv_heads, causal, max_ctas):
    plan, units, cta = inspect(ql, kl, heads, kv_heads, causal=causal, max_ctas=max_ctas, group_rows=-1)
    packed = plan["packed_heads"]
    assert (units[:, 9] == 1).all() and plan["workspace_bytes"] == 0
    tokens = 128 // packed
    assert (heads // kv_heads) % packed == 0 and cta[0] == 0 and cta[-1] == len(units) and (np.diff(cta) > 0).all()
    starts_q, starts_k = np.concatenate([[0], np.cumsum(ql)]), np.concatenate([[0], np.cumsum(kl)])
    seen = np.zeros((sum(ql), heads), int)
    for q0, q_end, kv0, kv_len, sees, head0, na, nb, two, *_ in units:
        s = int(np.searchsorted(starts_q, q0, side="right")) - 1
        assert (q_end, kv0, kv_len) == (starts_q[s + 1], starts_k[s], kl[s]) and head0 % packed == 0
        # all heads of a tile share one key/value head
        assert head0 // (heads // kv_heads) == (head0 + packed - 1) // (heads // kv_heads)
        for t in range(2 if two else 1):
            a, b = q0 + t * tokens, min(q0 + (t + 1) * tokens, q_end)
            assert a < b
            seen[a:b, head0:head0 + packed] += 1
            i = np.arange(a, b) - starts_q[s]
            need = np.clip(kl[s] - ql[s] + i + 1, 0, kl[s]) if causal else np.full(b - a, kl[s])
            assert (na, nb)[t] == -(-int(need.max()) // 128)
            if causal:
                assert sees + t * tokens == kl[s] - ql[s] + i[0] + 1
        assert two or nb == 0
    assert (seen == 1).all()
    # no CTA has more than the average and one unit above the best possible
    cost = 32 * units[:, 6:8].max(1) + units[:, 6:8].min(1) + 32
    loads = [cost[a:b].sum() for a, b in zip(cta[:-1], cta[1:])]
    assert max(loads) <= cost.sum() / len(loads) + cost.max()


@pytest.mark.parametrize("ql,kl,heads,kv_heads", CASES + [([16], [32768], 32, 8), ([2, 1], [600, 30000], 4, 2),
                                                          ([300, 1], [200, 131072], 5, 1)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("max_ctas", [0, 5])
def test_prompt_cut_units_join_to_the_whole(ql, kl, heads, kv_heads, causal, max_ctas):
    """The parts of a unit that is cut are the whole plan's unit: the same rows,
    its steps one after the other, each with a workspace slot of its own."""
    whole = inspect(ql, kl, heads, kv_heads, causal=causal, max_ctas=max_ctas, group_rows=-1)[1]
    plan, units, cta = inspect(ql, kl, heads, kv_heads, causal=causal, max_ctas=max_ctas)
    assert cta[0] == 0 and cta[-1] == len(units) and (np.diff(cta) > 0).all()
    rows = {}
    for u in units.tolist():
        rows.setdefault((u[0], u[5]), []).append(u)
    assert sorted(rows) == sorted((u[0], u[5]) for u in whole.tolist())
    slots = []
    for w in whole.tolist():
        parts = sorted(rows[w[0], w[5]], key=lambda u: u[10])
        assert [u[10] for u in parts] == list(range(len(parts))) and all(u[9] == len(parts) for u in parts)
        at = 0
        for u in parts:
            assert u[:2] + [u[5], u[8]] == w[:2] + [w[5], w[8]]
            assert (u[2], u[3], u[4]) == (w[2] + 128 * at, w[3] - 128 * at, w[4] - 128 * at)
            assert [min(max(n - at, 0), max(u[6:8])) for n in w[6:8]] == u[6:8]
            at += max(u[6:8])
            if len(parts) > 1:
                assert u[11] == parts[0][11] and max(u[6:8]) > 0
                slots += [u[11] + 2 * u[10], u[11] + 2 * u[10] + 1]
        assert at == max(w[6:8])
    assert sorted(slots) == list(range(len(slots)))
    assert plan["workspace_bytes"] == len(slots) * 128 * (128 + 2) * 4
    if (ql, kl) == ([16], [32768]) and max_ctas == 0:
        assert plan["ctas"] > 100


def test_prompt_plan_refusals():
    for args in (([1], [1], 3, 2, 128), ([1], [1], 4, 2, 80), ([-1], [1], 4, 2, 128), ([1], [-1], 4, 2, 128),
                 ([2 ** 31 - 1, 2 ** 31 - 1], [1, 1], 4, 2, 64), ([1], [1], 0, 1, 64)):
        with pytest.raises(bsp.BspError):
            inspect(args[0], args[1], args[2], args[3], args[4])


def test_calls_without_a_device_are_refused():
    L = bsp.lib()
    assert L.bsp_rope_table(None, 4, 16, 1e4, None, None, None) == bsp.BSP_ERR_INVALID_ARG
    assert L.bsp_rope(None, None, 0, 0, None, None, 0, 1, 1, 16, 16, 0, 0, 0, None, 0, 0, None) == bsp.BSP_ERR_INVALID_ARG
    assert L.bsp_kv_append(None, None, None, 0, 0, None, 0, 0, 0, 0, None, None, None, 0, 0, None, 0, 0, 0, None, 0, 0,
                           0, None, 0, 0, None, 0, 0, None) == bsp.BSP_ERR_INVALID_ARG
    h = ctypes.c_void_p(1)
    assert L.bsp_prompt_plan_create(None, 0, None, None, 1, 1, 64, 1, None, ctypes.byref(h)) == bsp.BSP_ERR_INVALID_ARG
    assert not h.value
    assert L.bsp_decode_plan_create(None, 1, 1, 1, 64, 16, None, ctypes.byref(h)) == bsp.BSP_ERR_INVALID_ARG
    assert L.bsp_prompt_execute(None, None, 0, 0, None, 0, 0, None, 0, 0, 1.0, None, 0, 0, None, None) == bsp.BSP_ERR_INVALID_ARG
    assert L.bsp_decode_execute(None, None, None, 0, 0, 0, None, None, 0, 0, 1.0, None, 0, 0, None, None) == bsp.BSP_ERR_INVALID_ARG
    assert L.bsp_prompt_plan_destroy(None) == L.bsp_decode_plan_destroy(None) == bsp.BSP_OK


def test_codes_of_the_64_bit_form():
    """e4m3 of the plain form: every value is its own code, halves go to even,
    and the scale's exponent is the smallest that fits."""
    v = ref.VALUES
    own = ref.e4m3(v[np.isfinite(v)])
    assert np.array_equal(v[own], v[np.isfinite(v)])
    mid = (ref._GRID[:-1] + ref._GRID[1:]) / 2
    assert (ref.e4m3(mid) % 2 == 0).all()
    assert ref.e4m3(np.array([1e9, -1e9, np.nan])).tolist() == [126, 254, 127]
    for a in (1e-45, 1.0, 448.0, 448.0001, 3.3e38):
        e = ref.exponent(a)
        assert a <= 448 * 2.0 ** e or e == 119
        assert e == -100 or a > 448 * 2.0 ** (e - 1)
