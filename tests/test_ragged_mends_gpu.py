"""The ragged decode operators on the GPU where they once went wrong.
Restatements are those of ragged_ref.py or stand here; tolerances are
test_ragged_gpu.py's."""
import ctypes as C
import math

import numpy as np
import pytest

import ragged_ref as ref
import specdec_b200 as sd
from test_ragged_gpu import (WIDE, check_attend, check_sample, cu, make_cache, make_table, run_append, run_attend, run_plan,
                             run_sample)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# ---------------------------------------------------------------------------
# block tables

@pytest.mark.parametrize("head,count,status", [(-1, 5, 2), (24, 5, 2), (3, -1, 2), (3, 25, 2), (1 << 30, 1 << 30, 2),
                                               (3, 23, 2), (3, 22, 0), (3, 1, 1)])
def test_plan_says_what_is_wrong_with_a_ring(gpu_lib, head, count, status):
    """A head or count outside the ring, or a tail that would come round to pages of this step's head, is a bad ring (2), too
    few pages are 1: a caller who frees pages and tries again on 1 must not do so on 2."""
    P, cap = 16, 24
    held, keep, q = [40, 0, 48], [40, 0, 5], [30, 8, 0]  # takes 2 and 1 pages, gives 2 of 3 back
    table = np.array([[20, 21, 22, -1, -1], [-1] * 5, [17, 18, 19, -1, -1]], np.int32)
    ring = np.arange(cap, dtype=np.int32)[::-1].copy()
    got = run_plan(held, keep, q, table, ring, (head, count), P, 40)
    assert got[8] == status
    if status:  # nothing moved
        want = (table, ring, (head, count), held, [0] * 4, [-1] * 40, [-1] * 40, [-1] * 40, status)
    else:
        want = ref.plan(held, keep, q, table, ring, (head, count), P, 40)
    for g, w in zip(got, want):
        assert np.array_equal(g, w)


# ---------------------------------------------------------------------------
# cache write

@pytest.mark.parametrize("old", [-0.03, -0.002, -1e-39, 0.03, 0.002, 0.0])
def test_append_over_a_block_of_any_scale(gpu_lib, old):
    """Older values keep their sign and size, to half a step of the new scale, where their block came with a scale below 0
    (a cache that another program filled); the new scale is the larger of the two sizes."""
    P, t, D, H = 32, 16, 16, 2
    rng = np.random.default_rng(25)
    cache = make_cache(rng, 1, H, P, D, t)
    codes = [c.copy() for c in cache[:2]]
    codes[0][0, 0, 0, :3] = [127, -127, 1]
    scales = [np.full_like(s, old) for s in cache[2:]]
    x = rng.normal(0, 0.3, (4, H, D)).astype(np.float32)
    (k, v, ks, vs), *_ = run_append([x, -2 * x], [*codes, *scales], np.zeros((1, 1), np.int32), [13], [0, 4], P, t, "f32", H, D)
    for c, s, was, rows in ((k, ks, codes[0], x), (v, vs, codes[1], -2 * x)):
        new = np.maximum(np.float32(abs(old)), np.abs(rows).max((0, 2)) * (np.float32(1) / np.float32(127)))  # [H]
        assert np.array_equal(s[0, :, 0], new) and np.array_equal(s[0, :, 1], np.full(H, old, np.float32))
        value = c[0].astype(np.float64) * new.astype(np.float64)[:, None, None]
        assert np.all(np.abs(value[:, :9] - was[0, :, :9].astype(np.float64) * np.float32(old)) <= new[:, None, None] * 0.50001)
        assert np.all(np.abs(value[:, 9:13] - rows.transpose(1, 0, 2)) <= new[:, None, None] * 0.50001)
        assert np.array_equal(c[0, :, 13:], was[0, :, 13:])


# ---------------------------------------------------------------------------
# sampling

@pytest.mark.parametrize("V", [2049, 4100, 8193, 16385])
def test_blocks_of_short_slices_meet_before_they_write(gpu_lib, V):
    """Blocks with next to nothing to load must not write to one that has not started: the maximum of every block's slice
    arrives, launch after launch, beside other work that delays blocks."""
    at = np.linspace(0, V - 1, 16).astype(np.int64)
    l = np.full((len(at), V), -2.0, np.float32)
    l[np.arange(len(at)), at] = 3.0
    rows, u = cu(l), torch.full((1,), 0.5, device="cuda")
    tok, prob = torch.zeros(len(at), 40, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, device="cuda")
    side, a = torch.cuda.Stream(), torch.randn(2048, 2048, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    zero = torch.zeros(1, device="cuda")
    for j in range(40):
        with torch.cuda.stream(side):
            a @ a
        for i in range(len(at)):
            sd.sample(rows[i:i + 1], u, tok[i, j], prob, temperature=zero,
                      stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert tok[:, :, 0].cpu().numpy().tolist() == np.repeat(at[:, None], 40, 1).tolist()
    T, k = np.ones(len(at), np.float32), np.full(len(at), 5)
    check_sample(l, np.full(len(at), 0.3, np.float32), T, k, T, 0 * T, *run_sample(l, np.full(len(at), 0.3), k=k))


@pytest.mark.parametrize("groups", [((0.0, 2000), (-0.05, 100)), ((0.0, 1500), (-0.3, 1500), (-2.0, 3000)),
                                    ((0.0, 30000), (-1e-3, 2000), (-4.0, 20000))])
def test_top_p_cut_at_the_edge_of_many_equal_weights(gpu_lib, groups):
    """Cuts just below, at and just above the mass of a group of equal logits: within what shifted sums leave open
    (2^-18 of it, 64 steps of a 24-bit top_p) the group's bin and the next one's both stay possible."""
    z = np.array([g[0] for g in groups], np.float32)
    n = np.array([g[1] for g in groups])
    l = np.random.default_rng(1).permutation(np.repeat(z, n))[None]
    w = np.floor(np.exp(z.astype(np.float64)) * 2.0 ** 31)
    edges = np.cumsum(n * w)[:-1] / (n * w).sum()
    p = np.concatenate([np.rint(e * 2 ** 24) + np.arange(-80, 81) for e in edges]).clip(1, 2 ** 24 - 1) / 2.0 ** 24
    B = len(p)
    u = np.where(np.arange(B) % 2, 1 - 2.0 ** -24, 0.5).astype(np.float32)
    one, zero = np.ones(B, np.float32), np.zeros(B, np.float32)
    p = p.astype(np.float32)
    rows = np.broadcast_to(l, (B, l.shape[1]))
    tok, prob = run_sample(rows, u, p=p)
    check_sample(rows, u, one, zero.astype(int), p, zero, tok, prob)
    k = np.full(B, int(n.sum()) - 1)  # the same cuts, top-k on as well
    check_sample(rows, u, one, k, p, zero, *run_sample(rows, u, k=k, p=p))


@pytest.mark.parametrize("V", [40, 33000, 400003])
def test_sample_at_an_infinite_temperature(gpu_lib, V):
    # every finite logit becomes 0 and draws alike; tokens at -infinity stay out whatever the filters
    l = np.random.default_rng(28).normal(0, 3, (5, V)).astype(np.float32)
    l[:, ::3] = -np.inf
    l[0, 4] = np.nan
    l[4, 7] = np.inf
    allowed = [np.flatnonzero(np.isfinite(r)) for r in l[:4]]
    u, T = np.array([0, 0.3, 0.7, 1 - 2.0 ** -24, 0.9], np.float32), [np.inf] * 5
    for k, p in ((0, 1.0), (9, 1.0), (0, 0.5), (10, 0.5), (V - 1, 1.0)):
        tok, prob = run_sample(l, u, T=T, k=[k] * 5, p=[p] * 5)
        for b, a in enumerate(allowed):
            n = min(k, len(a)) if k else len(a)
            n = -(-math.floor(p * n * 2 ** 31) // 2 ** 31)
            assert tok[b] == a[int(np.float64(u[b]) * 2 ** 24) * n >> 24] and abs(prob[b] * n - 1) < 1e-6
        assert tok[4] == 7 and prob[4] == 1


def test_sample_refuses_logits_of_the_host(gpu_lib):
    # the call runs on the logits' device, which it asks for: memory that has none is refused before any launch
    l, u, tok = np.zeros((1, 9), np.float32), torch.zeros(1, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    rc = gpu_lib.specdec_sample(l.ctypes.data, sd.F32, 1, 9, 9, None, None, None, None, u.data_ptr(), tok.data_ptr(), None, None)
    assert rc == 1 and b"device memory" in gpu_lib.specdec_last_error(None)


# ---------------------------------------------------------------------------
# attention

@pytest.mark.parametrize("dtype,max_q,spare", [("f32", 1, 1), ("f32", 9, 1), ("bf16", 1, 1), ("bf16", 9, 1), ("bf16", 64, WIDE)])
@pytest.mark.parametrize("D", [64, 128])
def test_attend_one_position_far_above_a_long_tail(gpu_lib, dtype, max_q, spare, D):
    """The first position stands 14 to 22 nats above 100,000 others of equal weight, whose values share a sign: what is
    lost of their weights adds up.  Requests share their pages and are many, so that a block has a whole request and the
    first position's warp a quarter of its tail: at 17 nats 7e-5 of the largest value with steps of 2^-24 of the largest
    weight."""
    Hkv, G, P, t, L, B = 8, 8 if max_q == 64 else 1, 128, 128, 100_000, 64
    H = Hkv * G
    rng = np.random.default_rng(21)
    table, n_pages = make_table(rng, [L], P, spare_cols=spare)
    k = np.zeros((n_pages, Hkv, P, D), np.int8)
    k[table[0, 0], :, 0, 0] = 127
    v = np.clip(np.rint(rng.normal(20, 30, k.shape)), -127, 127).astype(np.int8)
    ks = np.full((n_pages, Hkv, 1), 16 / 127, np.float32)
    vs = np.full((n_pages, Hkv, 1), 0.02, np.float32)
    x = np.zeros((1, H, D), np.float32)
    x[0, :, 0] = np.repeat([14, 16, 17, 17.5, 18, 18.5, 20, 22], G) / 16
    want = ref.attend(x, k, v, ks, vs, table, [L], [0, 1], P, t, 1.0, 0)
    got = run_attend(np.repeat(x, B, 0), (k, v, ks, vs), np.repeat(table, B, 0), [L] * B, np.arange(B + 1), H, Hkv, D, P, t,
                     dtype, 1.0, 0, max_q=max_q)
    check_attend(*got, *(np.repeat(w, B, 0) for w in want), dtype)


def test_attend_long_tails_of_uneven_weights(gpu_lib):
    # keys that spread the tail over 30 nats, some of it above the first position: the maximum moves on the way
    H, Hkv, D, P, t, L = 4, 1, 64, 64, 16, 60_000
    rng = np.random.default_rng(22)
    lens, q = [L, 20_000], [1, 3]
    table, n_pages = make_table(rng, lens, P)
    k = np.clip(np.rint(rng.normal(0, 40, (n_pages, Hkv, P, D))), -127, 127).astype(np.int8)
    k[table[:, 0], :, 0, :] = 50
    v = np.clip(np.rint(rng.normal(20, 30, k.shape)), -127, 127).astype(np.int8)
    ks = rng.uniform(0.01, 0.02, (n_pages, Hkv, P // t)).astype(np.float32)
    vs = rng.choice([0, 1e-3, 0.02, 0.5], (n_pages, Hkv, P // t)).astype(np.float32)
    x = (rng.normal(0, 1, (4, H, D)) + 0.5).astype(np.float32)
    want = ref.attend(x, k, v, ks, vs, table, lens, [0, 1, 4], P, t, 0.7, 0)
    check_attend(*run_attend(x, (k, v, ks, vs), table, lens, [0, 1, 4], H, Hkv, D, P, t, "f32", 0.7, 0), *want, "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,P,t,G,q", [(128, 128, 64, 1, 1), (128, 16, 16, 2, 5), (64, 32, 16, 1, 9), (64, 64, 64, 4, 1), (32, 128, 16, 2, 1),
                                       (16, 16, 16, 1, 3)])
def test_attend_maxima_that_keep_growing(gpu_lib, dtype, D, P, t, G, q):
    """Scores that climb by 20 nats along a cache, step after step with some noise, in items that a block does whole and
    several of: sums of earlier runs meet later maxima, and no item finds another's."""
    Hkv, B, L = 8, 64, 9_001
    H = Hkv * G
    rng = np.random.default_rng(24)
    table, n_pages = make_table(rng, [L], P)
    k, v, ks, vs = make_cache(rng, n_pages, Hkv, P, D, t)
    climb = np.rint(np.linspace(-127, 127, table.shape[1] * P)[:L])
    for p in range(L):
        k[table[0, p // P], :, p % P, 0] = climb[p]
    ks[:] = 0.02
    x = rng.normal(0, 0.5, (q, H, D)).astype(np.float32)
    x[:, :, 0] = rng.uniform(2, 6, (q, H))
    x = np.asarray(torch.tensor(x).to(torch.float32 if dtype == "f32" else torch.bfloat16).float())
    lens = [L, L - 4000, L - 7500]  # three lengths, one after the other
    want = [ref.attend(x, k, v, ks, vs, table, [n], [0, q], P, t, 1.0, 0) for n in lens]
    got = run_attend(np.tile(x, (B, 1, 1)), (k, v, ks, vs), np.repeat(table, B, 0), [lens[b % 3] for b in range(B)],
                     np.arange(B + 1) * q, H, Hkv, D, P, t, dtype, 1.0, 0, max_q=min(q, 60 // G))
    check_attend(*got, *(np.concatenate([want[b % 3][i] for b in range(B)]) for i in range(3)), dtype)


class _Words:
    """Device memory at an address as 32-bit words."""

    def __init__(self, address, n):
        self.__cuda_array_interface__ = dict(shape=(n,), typestr="<i4", data=(address, False), version=3)


@pytest.mark.parametrize("max_q,spare", [(1, 1), (64, WIDE)])
def test_check_makes_a_handle_whole_again(gpu_lib, max_q, spare):
    """A block that gives up leaves the arrivals of its split items counted and the error word set; check reports it once
    and the next calls merge as before."""
    H, Hkv, D, P, t = 32, 2, 64, 64, 16
    rng = np.random.default_rng(23)
    lens, q = [9000, 500], [2, 4]
    table, n_pages = make_table(rng, lens, P, spare_cols=spare)
    cache = make_cache(rng, n_pages, Hkv, P, D, t)
    cuq = np.array([0, 2, 6])
    x = np.asarray(torch.tensor(rng.normal(0, 1, (6, H, D))).bfloat16().float())
    want = ref.attend(x, *cache, table, lens, cuq, P, t, 0.125, 0)
    h = sd.KV8(H, Hkv, D, page_tokens=P, block_tokens=t, max_batch=2)
    # specdec_kv8: 12 words of geometry, device, multiprocessors, a string of 32 bytes, then part, ticket, err_word
    sms = C.cast(h.h.value + 52, C.POINTER(C.c_int32))[0]
    ticket, err = C.cast(h.h.value + 96, C.POINTER(C.c_uint64))[:2]
    assert sms == torch.cuda.get_device_properties(0).multi_processor_count and err == ticket + 3 * sms * 4
    words = torch.as_tensor(_Words(ticket, 3 * sms + 1), device="cuda")
    h.check()
    assert not words.any()
    words.fill_(1)
    with pytest.raises(sd.SpecDecError, match="did not end"):
        h.check()
    for _ in range(2):
        check_attend(*run_attend(x, cache, table, lens, cuq, H, Hkv, D, P, t, "bf16", 0.125, 0, max_q=max_q, handle=h), *want,
                     "bf16")
    assert not words.any()
    h.check()


def test_a_new_handle_is_ready_for_any_stream(gpu_lib):
    # its workspace is cleared on the default stream, which other streams need not wait for: create does
    sd.KV8(4, 4, 64).close()
    torch.cuda.synchronize()
    busy = torch.cuda.Event()
    torch.cuda._sleep(200_000_000)  # a tenth of a second of the default stream
    busy.record()
    assert not busy.query()
    h = sd.KV8(4, 4, 64)
    assert busy.query()
    h.close()


@pytest.mark.parametrize("dtype,max_q,spare", [("f32", 1, 1), ("f32", 9, 1), ("bf16", 1, 1), ("bf16", 9, 1), ("bf16", 64, WIDE)])
@pytest.mark.parametrize("large", [float(torch.finfo(torch.bfloat16).max), 1.6e38, 1e30])
def test_attend_queries_at_the_end_of_their_type(gpu_lib, dtype, max_q, spare, large):
    # values up to the largest bf16, with a scale that leaves scores of ordinary size
    H, Hkv, D, P, t = 8, 2, 64, 64, 16
    rng = np.random.default_rng(26)
    lens, q = [400, 70], [1, 3]
    table, n_pages = make_table(rng, lens, P, spare_cols=spare)
    cache = make_cache(rng, n_pages, Hkv, P, D, t)
    x = np.clip(rng.normal(0, 0.1, (4, H, D)), -1, 1)
    x[:, :, 3], x[1:, :, 5] = 1, -1
    x = np.asarray(torch.tensor(x * large).to(torch.float32 if dtype == "f32" else torch.bfloat16).float())
    scale = float(np.float32(4 / large))
    want = ref.attend(x, *cache, table, lens, [0, 1, 4], P, t, scale, 0)
    check_attend(*run_attend(x, cache, table, lens, [0, 1, 4], H, Hkv, D, P, t, dtype, scale, 0, max_q=max_q), *want, dtype)


@pytest.mark.parametrize("max_q,spare", [(1, 1), (9, 1), (64, WIDE)])
def test_attend_windows_that_cut_nothing_off(gpu_lib, max_q, spare):
    # windows up to the largest integer, beside rows that stand before their request's first position
    H, Hkv, D, P, t = 8, 2, 64, 16, 16
    rng = np.random.default_rng(27)
    lens, q = [3, 40, 0, 100], [6, 2, 3, 70]
    table, n_pages = make_table(rng, lens, P, spare_cols=spare)
    cache = make_cache(rng, n_pages, Hkv, P, D, t)
    cuq = np.concatenate([[0], np.cumsum(q)])
    x = np.asarray(torch.tensor(rng.normal(0, 1, (sum(q), H, D))).bfloat16().float())
    want = ref.attend(x, *cache, table, lens, cuq, P, t, 0.125, 0)
    cap = table.shape[1] * P
    for window in (100, cap - 1, cap, cap + 1, 2 ** 31 - 5, 2 ** 31 - 1):
        got = run_attend(x, cache, table, lens, cuq, H, Hkv, D, P, t, "bf16", 0.125, window, max_q=max_q)
        check_attend(*got, *want, "bf16")
