"""The ragged decode operators' refusals and plain restatements where there is
no GPU: nothing here reaches a device."""
import ctypes as C
import math

import numpy as np
import pytest

import ragged_ref as ref
import specdec_b200 as sd

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lib():
    return sd.load_library()


@pytest.mark.parametrize("cfg", [(6, 4, 64, 128, 16, 1), (4, 4, 48, 128, 16, 1), (4, 4, 64, 256, 16, 1), (4, 4, 64, 32, 64, 1),
                                 (4, 4, 64, 128, 8, 1), (4, 4, 64, 128, 48, 1), (4, 4, 64, 128, 16, 5000), (4, 4, 64, 128, 16, -1),
                                 (0, 0, 64, 128, 16, 1)])
def test_create_refuses_a_bad_geometry_before_a_device_is_needed(lib, cfg):
    c, h = sd._KV8Config(*cfg), C.c_void_p()
    assert lib.specdec_kv8_create(C.byref(c), 0, C.byref(h)) == 1
    assert not h.value and lib.specdec_kv8_last_error(None)


def test_null_arguments(lib):
    c, h = sd._KV8Config(4, 4, 64, 128, 16, 1), C.c_void_p()
    assert lib.specdec_kv8_create(None, 0, C.byref(h)) == 1
    assert lib.specdec_kv8_create(C.byref(c), 0, None) == 1
    assert lib.specdec_kv8_destroy(None) in (0, 1)
    assert lib.specdec_kv8_check(None, None) == 1
    assert lib.specdec_kv8_attend(None, None, None, None, 0, 0, 0, 0, None, 0, 0, None, 1, 1.0, 0, None) == 1


def test_sample_refuses(lib):
    f = lambda **k: lib.specdec_sample(*(dict(l=None, dtype=sd.F32, rows=1, vocab=8, stride=8, T=None, k=None, p=None, m=None,
                                              u=None, tok=None, prob=None, st=None) | k).values())
    assert f() == 1 and b"null" in lib.specdec_last_error(None)
    for bad in (dict(dtype=9), dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 20) + 1), dict(rows=2, stride=7)):
        assert f(**bad) == 1
    assert f(rows=0) == 0  # no rows: nothing to do


def test_binding_refuses_host_tensors(lib):
    codes, scales = torch.zeros(2, 1, 16, 16, dtype=torch.int8), torch.zeros(2, 1, 1)
    with pytest.raises(ValueError):
        sd.KV8Layer(codes, codes, scales, scales)
    with pytest.raises(ValueError):
        sd.KV8Layer(codes[0], codes[0], scales, scales)
    z = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        sd.KV8Batch(torch.zeros(1, 1, dtype=torch.int32), z[:1], z)
    with pytest.raises(ValueError):
        sd.sample(torch.zeros(1, 8), torch.zeros(1), z[:1])


# ---- the restatements against formulas that need no cache ---------------------------

@pytest.mark.parametrize("seed", range(5))
def test_plan_hands_out_each_page_once(seed):
    rng = np.random.default_rng(seed)
    B, P, cols = 6, 16, 5
    table, ring, state = np.full((B, cols), -1, np.int32), rng.permutation(B * cols).astype(np.int32), (int(rng.integers(B * cols)), B * cols)
    held = np.zeros(B, np.int64)
    for _ in range(40):
        keep = np.where(rng.random(B) < 0.2, 0, held - rng.integers(0, 1 + np.minimum(held, 4)))
        q = rng.integers(0, 1 + np.minimum(20, cols * P - keep))
        table, ring, state, held, cu, req, pos, slots, status = ref.plan(held, keep, q, table, ring, state, P, int(q.sum()) + 2)
        assert status == 0 and np.array_equal(held, keep + q) and cu[-1] == q.sum()
        used = [table[b, c] for b in range(B) for c in range(-(-held[b] // P))]
        free = [ring[(state[0] + i) % len(ring)] for i in range(state[1])]
        assert sorted(used + free) == list(range(B * cols))
        for t in range(cu[-1]):
            assert slots[t] == table[req[t], pos[t] // P] * P + pos[t] % P and held[req[t]] - q[req[t]] <= pos[t] < held[req[t]]
        assert (req[cu[-1]:] == -1).all() and (slots[cu[-1]:] == -1).all()


def test_append_in_pieces_stays_near_the_rows():
    rng = np.random.default_rng(2)
    H, P, t, D, n = 2, 32, 16, 8, 50
    x = rng.normal(0, 1, (n, H, D)).astype(np.float32)
    codes, scales = np.zeros((2, H, P, D), np.int8), np.full((2, H, P // t), 9.0, np.float32)
    table, at = np.array([[1, 0]], np.int32), 0
    for q in (1, 4, 11, 1, 20, 13):
        codes, scales = ref.append(codes, scales, table, [at + q], [0, q], x[at:at + q], P, t)
        at += q
    for p in range(n):
        got = codes[table[0, p // P], :, p % P] * scales[table[0, p // P], :, p % P // t][:, None]
        # half a step when written, half a step for each time that the block's scale grew: at most 3 pieces a block
        assert np.all(np.abs(got - x[p]) <= scales[table[0, p // P], :, p % P // t][:, None] * 2.001)


def test_attend_is_plain_attention():
    rng = np.random.default_rng(3)
    H, Hkv, D, P, t, L, q = 4, 2, 8, 16, 16, 40, 3
    codes = [rng.integers(-127, 128, (4, Hkv, P, D)).astype(np.int8) for _ in range(2)]
    scales = [rng.uniform(0.01, 0.02, (4, Hkv, 1)).astype(np.float32) for _ in range(2)]
    table = np.array([[2, 0, 3]], np.int32)
    x = rng.normal(0, 1, (q, H, D)).astype(np.float32)
    for window in (0, 7):
        out, lse, _ = ref.attend(x, *codes, *scales, table, [L], [0, q], P, t, 0.3, window)
        k, v = (torch.tensor((c.astype(np.float64) * s.astype(np.float64).repeat(P, 2)[..., None])[table[0]].transpose(0, 2, 1, 3)
                             .reshape(-1, Hkv, D)[:L]).repeat_interleave(2, 1) for c, s in zip(codes, scales))
        s = 0.3 * torch.einsum("ihd,jhd->hij", torch.tensor(x).double(), k)
        i, j = torch.arange(q)[:, None] + L - q, torch.arange(L)[None]
        s = s.masked_fill((j > i) | ((j <= i - window) if window else torch.zeros(q, L, dtype=torch.bool)), -math.inf)
        assert np.allclose(out, torch.einsum("hij,jhd->ihd", s.softmax(2), v).numpy(), rtol=1e-12, atol=1e-12)
        assert np.allclose(lse, s.logsumexp(2).T.numpy(), rtol=1e-12)


def test_sample_row_filters():
    l = np.log(np.array([0.05, 0.4, 0.05, 0.3, 0.2])).astype(np.float32)
    keep = lambda *a: np.nonzero(ref.sample_row(l, *a)[1])[0].tolist()
    assert keep(1, 0, 1, 0) == [0, 1, 2, 3, 4]
    assert keep(1, 2, 1, 0) == [1, 3]
    assert keep(1, 4, 1, 0) == [0, 1, 3, 4]       # of two equal ones the first
    assert keep(1, 0, 0.71, 0) == [1, 3, 4]
    assert keep(1, 0, 0.0, 0) == [1]              # the likeliest stays
    assert keep(1, 0, 1, 0.45) == [1, 3, 4]
    assert keep(1, 3, 0.75, 0.6) == [1, 3]
