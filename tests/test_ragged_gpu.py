"""The ragged decode operators on the GPU against plain restatements
(tests/ragged_ref.py): block tables and slot maps, cache write and read,
attention over the 8-bit cache, sampling.

Tolerances.  Attention in fp32: scores, exponentials and sums carry 24 bits and
products of up to 128 terms, so a weight is off by at most about 2^-17
relatively for scores below 2^4, and an output by that times the largest |v|
(2^-16 allowed).  bf16 rows: weights and queries enter the products with at
least 11 bits (2^-11 of the largest |v|) and the output is rounded to 8 bits
(2^-8 of itself).  Log-sum-exps are fp32 sums: 2^-16.
"""
import math

import numpy as np
import pytest

import ragged_ref as ref
import specdec_b200 as sd

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def cu(x, dtype=None):
    t = torch.as_tensor(np.ascontiguousarray(x))
    return (t if dtype is None else t.to(dtype)).cuda()


def i32(x):
    return cu(np.asarray(x, np.int32))


def make_cache(rng, n_pages, Hkv, P, D, t, scale=(0.005, 0.03)):
    codes = [np.clip(np.rint(rng.normal(0, 40, (n_pages, Hkv, P, D))), -127, 127).astype(np.int8) for _ in range(2)]
    scales = [rng.uniform(*scale, (n_pages, Hkv, P // t)).astype(np.float32) for _ in range(2)]
    return codes[0], codes[1], scales[0], scales[1]


def make_table(rng, lens, P, extra=2, spare_cols=1):
    need = [-(-n // P) for n in lens]
    n_pages = sum(need) + extra
    perm, cols = rng.permutation(n_pages), max(need + [1]) + spare_cols
    table, at = np.full((len(lens), cols), -1, np.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, n_pages


# ---------------------------------------------------------------------------
# block tables and slot maps

def run_plan(held, keep, q, table, ring, state, P, T, stream=0):
    B = len(held)
    h = sd.KV8(1, 1, 64, page_tokens=P, block_tokens=16, max_batch=max(1, B))
    z = dict(dtype=torch.int32, device="cuda")
    d = dict(table=cu(table), kv_len=torch.zeros(B, **z), cu_q=torch.zeros(B + 1, **z), tok_req=torch.zeros(T, **z),
             tok_pos=torch.zeros(T, **z), slots=torch.zeros(T, dtype=torch.int64, device="cuda"),
             status=torch.zeros(1, **z))
    r, out = cu(ring), torch.zeros(2, **z)
    h.plan(sd.KV8Batch(**d), i32(held), i32(keep), i32(q), r, i32(state), out, stream)
    torch.cuda.synchronize()
    g = {k: v.cpu().numpy() for k, v in d.items()}
    return (g["table"], r.cpu().numpy(), tuple(out.cpu().tolist()), g["kv_len"], g["cu_q"], g["tok_req"], g["tok_pos"],
            g["slots"], int(g["status"][0]))


def plan_case(rng, B, P, cols, qmax, T_pad=0):
    cap = cols * P
    held = rng.integers(0, cap + 1, B)
    keep = np.where(rng.random(B) < 0.2, 0, rng.integers(0, held + 1))
    q = np.minimum(rng.integers(0, qmax + 1, B), cap - keep)
    have = -(-held // P)
    n_pages = B * cols + 3
    perm = rng.permutation(n_pages).astype(np.int32)
    table, at = np.full((B, cols), -1, np.int32), 0
    for b in range(B):
        table[b, :have[b]] = perm[at:at + have[b]]
        at += have[b]
    head, count = int(rng.integers(0, n_pages)), n_pages - at
    ring = np.zeros(n_pages, np.int32)
    ring[(head + np.arange(n_pages)) % n_pages] = np.concatenate([perm[at:], perm[:at]])
    return held, keep, q, table, ring, (head, count), P, int(q.sum()) + T_pad


@pytest.mark.parametrize("B,P,cols,qmax,pad", [(1, 128, 1, 1, 0), (3, 16, 7, 40, 5), (33, 128, 5, 9, 1),
                                              (257, 64, 3, 3, 0), (1025, 16, 4, 64, 700), (4096, 32, 2, 2, 3)])
def test_plan(gpu_lib, B, P, cols, qmax, pad):
    c = plan_case(np.random.default_rng(B), B, P, cols, qmax, pad)
    for got, want in zip(run_plan(*c), ref.plan(*c)):
        assert np.array_equal(got, want)


def test_plan_nothing_to_do_and_no_rows(gpu_lib):
    c = ([0, 200, 0], [0, 200, 0], [0, 0, 0], np.array([[-1, -1], [4, 2], [-1, -1]], np.int32),
         np.arange(5, dtype=np.int32), (2, 3), 128, 0)
    for got, want in zip(run_plan(*c), ref.plan(*c)):
        assert np.array_equal(got, want)


@pytest.mark.parametrize("what,status", [("pages", 1), ("keep", 2), ("negative", 2), ("long", 2), ("rows", 4)])
def test_plan_moves_nothing_on_a_bad_step(gpu_lib, what, status):
    held, keep, q, table, ring, (head, count), P, T = plan_case(np.random.default_rng(5), 9, 16, 6, 30)
    if what == "pages":
        count = 0
        q = np.minimum(q + 16, 6 * 16 - keep)
        T = int(q.sum())
    elif what == "keep":
        keep[4] = held[4] + 1
    elif what == "negative":
        q[2] = -1
    elif what == "long":
        q[8] = 6 * 16 - keep[8] + 1
    else:
        T = int(q.sum()) - 1
    c = (held, keep, q, table, ring, (head, count), P, T)
    want = ref.plan(*c)
    assert want[-1] & status
    for got, w in zip(run_plan(*c), want):
        assert np.array_equal(got, w)


# ---------------------------------------------------------------------------
# cache write and read

def run_append(x, cache, table, lens, cuq, P, t, dtype, H, D, pad_stride=0, offset=0):
    """Returns (codes k, v, scales k, v) after the write; rows may sit in wider, shifted buffers."""
    h = sd.KV8(H, H, D, page_tokens=P, block_tokens=t, max_batch=len(lens))
    dev = [cu(a) for a in cache]
    layer = sd.KV8Layer(*dev)
    T = x[0].shape[0]
    rows = []
    for a in x:
        wide = torch.full((offset + T * (H * D + pad_stride) + 1,), 7.0, dtype=DT[dtype], device="cuda")
        r = wide[offset:offset + T * (H * D + pad_stride)].view(T, -1)[:, :H * D].view(T, H, D)
        r.copy_(cu(a))
        rows.append(r)
    batch = sd.KV8Batch(i32(table), i32(lens), i32(cuq))
    h.append(layer, batch, *rows)
    torch.cuda.synchronize()
    return [d.cpu().numpy() for d in dev], h, layer, dev


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("P,t,D,H", [(128, 16, 128, 2), (64, 64, 64, 3), (128, 128, 128, 1), (16, 16, 16, 5), (32, 16, 32, 2)])
@pytest.mark.parametrize("pad,offset", [(0, 0), (24, 1)])
def test_append_and_gather(gpu_lib, dtype, P, t, D, H, pad, offset):
    rng = np.random.default_rng(P + t + D)
    q = [1, 0, 5, 2 * t + 3, 1, t, 7]
    lens = [1, 40, t, 5 * t, 3 * t + 1, 4 * t, P + 3]
    cuq = np.concatenate([[0], np.cumsum(q)])
    table, n_pages = make_table(rng, lens, P)
    cache = make_cache(rng, n_pages, H, P, D, t)
    x = [np.asarray(torch.tensor(rng.normal(0, 1, (sum(q), H, D)) * rng.choice([0.01, 1, 50], (sum(q), 1, 1))).to(DT[dtype]).float()) for _ in range(2)]
    (k, v, ks, vs), h, layer, dev = run_append(x, cache, table, lens, cuq, P, t, dtype, H, D, pad, offset)
    for got, gs, c0, s0, rows in ((k, ks, cache[0], cache[2], x[0]), (v, vs, cache[1], cache[3], x[1])):
        want, ws = ref.append(c0, s0, table, lens, cuq, rows, P, t)
        assert np.array_equal(got, want) and np.array_equal(gs, ws)
        # a new row's value is within half a step of the row
        for b in range(len(lens)):
            for i in range(q[b]):
                p = lens[b] - q[b] + i
                step = gs[table[b, p // P], :, p % P // t].astype(np.float64)
                val = got[table[b, p // P], :, p % P].astype(np.float64) * step[:, None]
                assert np.all(np.abs(val - rows[cuq[b] + i]) <= step[:, None] * 0.50001)
    slots = [int(table[b, p // P]) * P + p % P for b in range(len(lens)) for p in range(lens[b])] + [-1, n_pages * P]
    out = [torch.full((len(slots), H, D), 3.0, dtype=DT[dtype], device="cuda") for _ in range(2)]
    h.gather(layer, cu(np.array(slots, np.int64)), *out)
    for o, c, s in ((out[0], k, ks), (out[1], v, vs)):
        for n, slot in enumerate(slots):
            want = np.zeros((H, D), np.float32)
            if 0 <= slot < n_pages * P:
                want = c[slot // P, :, slot % P].astype(np.float32) * s[slot // P, :, slot % P // t][:, None]
            assert torch.equal(o[n].cpu(), torch.tensor(want).to(DT[dtype]))
    only_v = torch.zeros_like(out[1])
    h.gather(layer, cu(np.array(slots, np.int64)), None, only_v)
    assert torch.equal(only_v, out[1])


def test_append_zero_tiny_and_non_finite_rows(gpu_lib):
    P, t, D, H = 16, 16, 32, 1
    x = np.zeros((6, H, D), np.float32)
    x[1] = 1e-39  # its scale is below the smallest normal number
    x[2, 0, :3] = [np.inf, -np.inf, np.nan]
    x[2, 0, 3:] = 2.0
    x[3, 0, 0] = np.nan  # nothing finite but zeros
    x[4] = 3e38
    x[5, 0, 1] = np.inf
    lens, q = [1, 1, 1, 1, 1, 1], [1] * 6
    table = np.arange(6, dtype=np.int32)[:, None]
    cache = make_cache(np.random.default_rng(0), 6, H, P, D, t)
    (k, v, ks, vs), *_ = run_append([x, x], cache, table, lens, np.arange(7), P, t, "f32", H, D)
    want, ws = ref.append(cache[0], cache[2], table, lens, np.arange(7), x, P, t)
    assert np.array_equal(k, want) and np.array_equal(ks, ws)
    assert ks[0, 0, 0] == 0 and ks[1, 0, 0] == 0 and ks[3, 0, 0] == 0 and not k[[0, 1, 3], 0, 0].any()
    assert k[2, 0, 0, :4].tolist() == [127, -127, 0, 127] and np.isfinite(ks).all()


def test_append_keeps_what_a_bad_table_or_length_names(gpu_lib):
    P, t, D, H = 16, 16, 16, 1
    rng = np.random.default_rng(1)
    cache = make_cache(rng, 2, H, P, D, t)
    x = rng.normal(0, 1, (3, H, D)).astype(np.float32)
    # a page past the pool, a negative page, more rows than the request is long
    (k, v, ks, vs), *_ = run_append([x, x], cache, np.array([[9], [-4], [1]], np.int32), [1, 1, 0], [0, 1, 2, 3], P, t, "f32", H, D)
    for a, b in zip((k, v, ks, vs), cache):
        assert np.array_equal(a, b)


# ---------------------------------------------------------------------------
# attention

def run_attend(q, cache, table, lens, cuq, H, Hkv, D, P, t, dtype, scale, window, max_q=None, q_pad=0, out_pad=0,
               handle=None, stream=None, lse=True):
    T = q.shape[0]
    h = handle or sd.KV8(H, Hkv, D, page_tokens=P, block_tokens=t, max_batch=len(lens))
    layer = sd.KV8Layer(*[cu(a) for a in cache])
    wide = torch.zeros(T, H * D + q_pad, dtype=DT[dtype], device="cuda")
    rows = wide[:, q_pad:].view(T, H, D)
    rows.copy_(cu(q))
    out = torch.full((T, H * D + out_pad), 5.0, dtype=DT[dtype], device="cuda")
    o = out[:, :H * D].view(T, H, D)
    ls = torch.full((T, H), 5.0, device="cuda") if lse else None
    batch = sd.KV8Batch(i32(table), i32(lens), i32(cuq))
    m = max([cuq[b + 1] - cuq[b] for b in range(len(lens))] + [0]) if max_q is None else max_q
    torch.cuda.synchronize()
    with torch.cuda.stream(stream) if stream else torch.cuda.stream(torch.cuda.current_stream()):
        h.attend(layer, batch, rows, o, lse=ls, max_q=int(m), scale=scale, window=window,
                 stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert out_pad == 0 or bool((out[:, H * D:] == 5).all())
    return o.float().cpu().numpy().astype(np.float64), None if ls is None else ls.cpu().numpy().astype(np.float64)


def check_attend(got, lse, want, wlse, big, dtype):
    rel, absolute = (2.0 ** -16, 2.0 ** -16) if dtype == "f32" else (2.0 ** -8, 2.0 ** -11)
    assert np.isfinite(got).all()
    err = np.abs(got - want)
    assert np.all(err <= rel * np.abs(want) + absolute * big[..., None]), float((err - rel * np.abs(want)).max())
    empty = np.isneginf(wlse)
    assert np.array_equal(np.isneginf(lse), empty)
    assert np.all(np.abs(lse - wlse)[~empty] <= 2.0 ** -16 * np.maximum(1, np.abs(wlse[~empty])))


def poison(cache, table, lens, P, t):
    """Scales that no visible position uses become NaN or infinity."""
    k, v, ks, vs = (a.copy() for a in cache)
    used = np.zeros((ks.shape[0], ks.shape[2]), bool)
    for b, n in enumerate(lens):
        for p in range(0, n, t):
            if 0 <= table[b, p // P] < ks.shape[0]:
                used[table[b, p // P], p % P // t] = True
    for s, bad in ((ks, np.nan), (vs, np.inf)):
        s[np.broadcast_to(~used[:, None], s.shape)] = bad
    return k, v, ks, vs


SHAPES = [  # heads, kv heads, dim, page, block, q per request, lengths, window
    (4, 4, 64, 128, 16, [1, 1, 1, 1], [1, 15, 128, 300], 0),
    (2, 2, 128, 128, 16, [5, 5, 3, 1], [5, 129, 384, 257], 0),
    (8, 2, 128, 64, 32, [1, 2, 0, 4], [700, 2, 9, 64], 0),
    (8, 1, 64, 32, 32, [3, 1], [33, 1000], 0),
    (24, 8, 32, 16, 16, [1, 2, 1], [17, 16, 250], 0),
    (6, 2, 16, 16, 16, [2, 7], [40, 7], 0),
    (4, 1, 128, 128, 128, [16, 9], [200, 9], 0),
    (8, 2, 128, 128, 64, [70, 33, 1], [70, 400, 513], 0),
    (2, 1, 64, 128, 64, [150], [150], 0),
    (4, 2, 128, 128, 16, [1, 5, 40], [500, 260, 300], 33),
    (4, 4, 64, 64, 16, [1, 130], [130, 200], 1),
    (3, 3, 32, 128, 32, [4], [1500], 700),
    (12, 12, 64, 128, 16, [1] * 20, list(range(1, 21)), 0),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attend(gpu_lib, dtype, shape):
    H, Hkv, D, P, t, q, lens, window = SHAPES[shape]
    rng = np.random.default_rng(100 + shape)
    table, n_pages = make_table(rng, lens, P)
    cache = poison(make_cache(rng, n_pages, Hkv, P, D, t), table, lens, P, t)
    cuq = np.concatenate([[0], np.cumsum(q)])
    x = np.asarray(torch.tensor(rng.normal(0, 1, (sum(q), H, D))).to(DT[dtype]).float())
    scale = 1 / math.sqrt(D)
    want = ref.attend(x, *cache, table, lens, cuq, P, t, scale, window)
    got = run_attend(x, cache, table, lens, cuq, H, Hkv, D, P, t, dtype, scale, window)
    check_attend(*got, *want, dtype)
    # the hint only selects the kernel; other strides; another stream; no lse
    other = run_attend(x, cache, table, lens, cuq, H, Hkv, D, P, t, dtype, scale, window, max_q=1 if max(q) > 1 else 500,
                       q_pad=3, out_pad=5, stream=torch.cuda.Stream())
    check_attend(*other, *want, dtype)
    again = run_attend(x, cache, table, lens, cuq, H, Hkv, D, P, t, dtype, scale, window, lse=False)
    assert np.array_equal(again[0], got[0])


@pytest.mark.parametrize("max_q", [1, 64])
def test_attend_rows_that_see_nothing(gpu_lib, max_q):
    H, Hkv, D, P, t = 4, 2, 64, 32, 16
    rng = np.random.default_rng(3)
    lens, q = [0, 3, 64, 40, 0], [1, 5, 1, 2, 0]  # an empty cache, more rows than positions, missing pages
    table, n_pages = make_table(rng, lens, P)
    table[2] = [-1, n_pages + 5] + [-1] * (table.shape[1] - 2)
    table[3, 0] = -7
    cuq = np.concatenate([[0], np.cumsum(q)])
    cache = poison(make_cache(rng, n_pages, Hkv, P, D, t), table, lens, P, t)
    x = rng.normal(0, 1, (sum(q) + 2, H, D)).astype(np.float32)
    want = ref.attend(x, *cache, table, lens, cuq, P, t, 0.125, 0)
    got, lse = run_attend(x, cache, table, lens, cuq, H, Hkv, D, P, t, "f32", 0.125, 0, max_q=max_q)
    check_attend(got[:sum(q)], lse[:sum(q)], want[0][:sum(q)], want[1][:sum(q)], want[2][:sum(q)], "f32")
    assert not got[[0, 1, 2, 6]].any() and np.isneginf(lse[[0, 1, 2, 6]]).all()
    assert (got[sum(q):] == 5).all() and (lse[sum(q):] == 5).all()  # rows of no request


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("max_q", [1, 64])
def test_attend_scales_of_every_size(gpu_lib, dtype, max_q):
    # value scales from 0 and 1e-30 to 1e4 in one cache, key scales that leave single positions standing
    H, Hkv, D, P, t = 4, 2, 128, 128, 16
    rng = np.random.default_rng(8)
    lens, q = [1000, 77], [2, 3]
    table, n_pages = make_table(rng, lens, P)
    k, v, ks, vs = make_cache(rng, n_pages, Hkv, P, D, t)
    vs[:] = rng.choice([0, 1e-30, 1e-6, 1e-2, 1, 1e4], vs.shape)
    ks[:] = rng.choice([0, 1e-20, 1e-3, 0.02], ks.shape)
    cuq = np.concatenate([[0], np.cumsum(q)])
    x = np.asarray(torch.tensor(rng.normal(0, 1, (sum(q), H, D))).to(DT[dtype]).float())
    want = ref.attend(x, k, v, ks, vs, table, lens, cuq, P, t, 0.0884, 0)
    check_attend(*run_attend(x, (k, v, ks, vs), table, lens, cuq, H, Hkv, D, P, t, dtype, 0.0884, 0, max_q=max_q),
                 *want, dtype)


@pytest.mark.parametrize("max_q", [1, 64])
def test_attend_queries_of_every_size(gpu_lib, max_q):
    # rows of zeros, 1e-30 and 1e3 (one position takes all the weight): the weights keep their sum
    H, Hkv, D, P, t = 4, 4, 64, 64, 32
    rng = np.random.default_rng(9)
    lens, q = [333], [4]
    table, n_pages = make_table(rng, lens, P)
    cache = make_cache(rng, n_pages, Hkv, P, D, t)
    x = rng.normal(0, 1, (4, H, D)).astype(np.float32) * np.array([0, 1e-30, 1, 16], np.float32)[:, None, None]
    want = ref.attend(x, *cache, table, lens, [0, 4], P, t, 0.125, 0)
    check_attend(*run_attend(x, cache, table, lens, [0, 4], H, Hkv, D, P, t, "f32", 0.125, 0, max_q=max_q), *want, "f32")


def test_attend_one_handle_many_sizes_and_repeats(gpu_lib):
    # the workspace is left ready for the next call whatever its split was; equal inputs give equal bits
    H, Hkv, D, P, t = 8, 2, 128, 128, 16
    h = sd.KV8(H, Hkv, D, page_tokens=P, block_tokens=t, max_batch=40)
    rng = np.random.default_rng(10)
    first = {}
    for n in range(6):
        for c, (lens, q) in enumerate([([9000], [1]), ([100] * 40, [1] * 40), ([5000, 3, 700], [5, 1, 2]), ([3000], [90])]):
            if n == 0:
                table, n_pages = make_table(rng, lens, P)
                cache = make_cache(rng, n_pages, Hkv, P, D, t)
                x = np.asarray(torch.tensor(rng.normal(0, 1, (sum(q), H, D))).bfloat16().float())
                first[c] = [cache, table, x, None]
            cache, table, x, was = first[c]
            cuq = np.concatenate([[0], np.cumsum(q)])
            got = run_attend(x, cache, table, lens, cuq, H, Hkv, D, P, t, "bf16", 0.0884, 0, handle=h)
            if was is None:
                first[c][3] = got
                if c != 0:
                    check_attend(*got, *ref.attend(x, *cache, table, lens, cuq, P, t, 0.0884, 0), "bf16")
            else:
                assert np.array_equal(got[0], was[0]) and np.array_equal(got[1], was[1])


TILES = [  # heads, kv heads, dim, page, block, q per request, lengths, window
    (8, 2, 128, 128, 64, [70, 33, 1, 0], [70, 400, 513, 9], 0),
    (2, 1, 64, 128, 64, [150], [150], 0),
    (4, 2, 128, 128, 16, [1, 5, 40], [500, 260, 300], 33),
    (4, 4, 64, 64, 16, [1, 130], [130, 200], 1),
    (6, 2, 128, 16, 16, [100, 7, 86], [100, 290, 129], 0),
    (5, 1, 64, 32, 32, [51, 52, 3], [640, 52, 3], 200),
    (4, 1, 128, 64, 32, [65, 1, 64], [193, 1, 64], 0),
    (2, 2, 128, 128, 128, [300, 257], [1000, 257], 129),
    (16, 1, 64, 16, 16, [3, 17], [40, 17], 0),
]
WIDE = 8000  # columns of tables with room for far more than there is, as for the longest request that may come


@pytest.mark.parametrize("shape", range(len(TILES)))
def test_attend_many_rows_and_wide_tables(gpu_lib, shape):
    H, Hkv, D, P, t, q, lens, window = TILES[shape]
    rng = np.random.default_rng(200 + shape)
    table, n_pages = make_table(rng, lens, P, spare_cols=WIDE)
    cache = poison(make_cache(rng, n_pages, Hkv, P, D, t), table, lens, P, t)
    cuq = np.concatenate([[0], np.cumsum(q)])
    x = np.asarray(torch.tensor(rng.normal(0, 1, (sum(q), H, D))).bfloat16().float())
    scale = 1 / math.sqrt(D)
    want = ref.attend(x, *cache, table, lens, cuq, P, t, scale, window)
    h = sd.KV8(H, Hkv, D, page_tokens=P, block_tokens=t, max_batch=len(lens))
    got = run_attend(x, cache, table, lens, cuq, H, Hkv, D, P, t, "bf16", scale, window, max_q=500, handle=h)
    check_attend(*got, *want, "bf16")
    other = run_attend(x, cache, table, lens, cuq, H, Hkv, D, P, t, "bf16", scale, window, max_q=500, q_pad=3, out_pad=5,
                       stream=torch.cuda.Stream(), handle=h)
    check_attend(*other, *want, "bf16")
    again = run_attend(x, cache, table, lens, cuq, H, Hkv, D, P, t, "bf16", scale, window, max_q=500, lse=False, handle=h)
    assert np.array_equal(again[0], got[0])
    h.check()


@pytest.mark.parametrize("D", [64, 128])
def test_attend_many_short_prompts(gpu_lib, D):
    # several row tiles a block, one after the other through the same shared memory; equal calls give equal bits
    H, Hkv, P, t = 64, 16, 32, 16
    rng = np.random.default_rng(17)
    q = rng.integers(20, 66, 24).tolist()
    lens = [n + int(rng.integers(0, 3)) * 40 for n in q]
    table, n_pages = make_table(rng, lens, P)
    cache = poison(make_cache(rng, n_pages, Hkv, P, D, t), table, lens, P, t)
    cuq = np.concatenate([[0], np.cumsum(q)])
    x = np.asarray(torch.tensor(rng.normal(0, 1, (sum(q), H, D))).bfloat16().float())
    h = sd.KV8(H, Hkv, D, page_tokens=P, block_tokens=t, max_batch=len(lens))
    got = run_attend(x, cache, table, lens, cuq, H, Hkv, D, P, t, "bf16", D ** -0.5, 0, handle=h)
    check_attend(*got, *ref.attend(x, *cache, table, lens, cuq, P, t, D ** -0.5, 0), "bf16")
    for _ in range(10):
        again = run_attend(x, cache, table, lens, cuq, H, Hkv, D, P, t, "bf16", D ** -0.5, 0, handle=h)
        assert np.array_equal(again[0], got[0]) and np.array_equal(again[1], got[1])
    h.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("spare,max_q", [(1, 1), (1, 9), (WIDE, 500)])
def test_attend_a_bad_block_reaches_only_the_rows_that_see_it(gpu_lib, dtype, spare, max_q):
    # the last row's own position opens a block: its scales, or its query, are not finite
    H, Hkv, D, P, t = 8, 2, 128, 128, 16
    rng = np.random.default_rng(12)
    lens, q = [17, 145, 641, 33], [2, 5, 1, 1]
    table, n_pages = make_table(rng, lens, P, spare_cols=spare)
    k, v, ks, vs = make_cache(rng, n_pages, Hkv, P, D, t)
    cuq = np.concatenate([[0], np.cumsum(q)])
    x = np.asarray(torch.tensor(rng.normal(0, 1, (sum(q), H, D))).to(DT[dtype]).float())
    clean = ref.attend(x, k, v, ks, vs, table, lens, cuq, P, t, 0.0884, 0)
    sound = np.ones(sum(q), bool)
    for b, (where, bad) in enumerate([(vs, np.nan), (ks, np.nan), (vs, np.inf)]):
        where[table[b, (lens[b] - 1) // P], :, (lens[b] - 1) % P // t] = bad
        sound[cuq[b + 1] - 1] = False
    x[-1, :, 5] = np.nan
    sound[-1] = False
    got, lse = run_attend(x, (k, v, ks, vs), table, lens, cuq, H, Hkv, D, P, t, dtype, 0.0884, 0, max_q=max_q)
    check_attend(got[sound], lse[sound], *(w[sound] for w in clean), dtype)
    assert not np.isfinite(got[~sound]).any(axis=2).any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("spare,max_q", [(1, 3), (WIDE, 500)])
def test_attend_negative_scales(gpu_lib, dtype, spare, max_q):
    H, Hkv, D, P, t = 4, 2, 64, 64, 16
    rng = np.random.default_rng(13)
    lens, q = [300, 64], [3, 2]
    table, n_pages = make_table(rng, lens, P, spare_cols=spare)
    k, v, ks, vs = make_cache(rng, n_pages, Hkv, P, D, t)
    ks *= rng.choice([-1, 1], ks.shape).astype(np.float32)
    vs *= rng.choice([-1, 1], vs.shape).astype(np.float32)
    cuq = np.concatenate([[0], np.cumsum(q)])
    x = np.asarray(torch.tensor(rng.normal(0, 1, (sum(q), H, D))).to(DT[dtype]).float())
    for scale in (0.125, -0.125):
        want = ref.attend(x, k, v, ks, vs, table, lens, cuq, P, t, scale, 0)
        got = run_attend(x, (k, v, ks, vs), table, lens, cuq, H, Hkv, D, P, t, dtype, scale, 0, max_q=max_q)
        check_attend(*got, *want, dtype)


@pytest.mark.parametrize("max_q", [1, 64])
def test_attend_over_a_thousand_requests(gpu_lib, max_q):
    H, Hkv, D, P, t = 4, 2, 64, 16, 16
    B = 1100
    rng = np.random.default_rng(14)
    lens, q = rng.integers(0, 40, B), rng.integers(0, 3, B)
    table, n_pages = make_table(rng, lens, P, spare_cols=20)
    cache = make_cache(rng, n_pages, Hkv, P, D, t)
    cuq = np.concatenate([[0], np.cumsum(q)])
    x = np.asarray(torch.tensor(rng.normal(0, 1, (int(cuq[-1]), H, D))).bfloat16().float())
    want = ref.attend(x, *cache, table, lens, cuq, P, t, 0.125, 0)
    check_attend(*run_attend(x, cache, table, lens, cuq, H, Hkv, D, P, t, "bf16", 0.125, 0, max_q=max_q), *want, "bf16")


@pytest.mark.parametrize("max_q", [1, 64])
def test_cache_past_32_bit_offsets(gpu_lib, max_q):
    # a pool of over 2^31 codes; the request lives in its last pages
    H, Hkv, D, P, t = 16, 16, 128, 128, 128
    n_pages = (1 << 31) // (Hkv * P * D) + 6
    rng = np.random.default_rng(11)
    lens, q = [300], [2]
    h = sd.KV8(H, Hkv, D, page_tokens=P, block_tokens=t, max_batch=1)
    k = torch.zeros(n_pages, Hkv, P, D, dtype=torch.int8, device="cuda")
    v = torch.zeros_like(k)
    ks, vs = (torch.zeros(n_pages, Hkv, 1, device="cuda") for _ in range(2))
    table = np.array([[n_pages - 1, n_pages - 3, n_pages - 2]], np.int32)
    layer = sd.KV8Layer(k, v, ks, vs)
    rows = [torch.tensor(rng.normal(0, 1, (300, Hkv, D)).astype(np.float32)).cuda() for _ in range(2)]
    h.append(layer, sd.KV8Batch(i32(table), i32(lens), i32([0, 300])), *rows)
    out = [torch.zeros(300, Hkv, D, device="cuda") for _ in range(2)]
    slots = [int(table[0, p // P]) * P + p % P for p in range(300)]
    h.gather(layer, cu(np.array(slots, np.int64)), *out)
    for o, r in zip(out, rows):
        assert float((o - r).abs().max()) <= float(r.abs().max()) / 127 * 0.50001
    x = rng.normal(0, 1, (2, H, D)).astype(np.float32)
    got, lse = torch.zeros(2, H, D, device="cuda"), torch.zeros(2, H, device="cuda")
    h.attend(layer, sd.KV8Batch(i32(table), i32(lens), i32([0, 2])), cu(x), got, lse=lse, max_q=max_q)
    tail = [a[n_pages - 3:].cpu().numpy() for a in (k, v, ks, vs)]
    want = ref.attend(x, *tail, table - (n_pages - 3), lens, [0, 2], P, t, 1 / math.sqrt(D), 0)
    check_attend(got.cpu().numpy().astype(np.float64), lse.cpu().numpy().astype(np.float64), *want, "f32")


# ---------------------------------------------------------------------------
# sampling

def run_sample(l, u, T=None, k=None, p=None, m=None, dtype="f32", pad=0, stream=0):
    B, V = l.shape
    wide = torch.full((B, V + pad), 1e4, dtype=DT[dtype], device="cuda")
    rows = wide[:, pad:]
    rows.copy_(cu(l.astype(np.float32)))
    f = [None if a is None else cu(np.asarray(a, np.float32)) for a in (T, p, m)]
    tok, prob = torch.zeros(B, dtype=torch.int32, device="cuda"), torch.zeros(B, device="cuda")
    sd.sample(rows, cu(np.asarray(u, np.float32)), tok, prob, temperature=f[0], top_k=None if k is None else i32(k),
              top_p=f[1], min_p=f[2], stream=stream)
    torch.cuda.synchronize()
    return tok.cpu().numpy(), prob.cpu().numpy()


def check_sample(l, u, T, k, p, m, tok, prob):
    """The drawn token is the definition's, or next to it within what the 32-bit exponentials leave open."""
    for b in range(len(l)):
        if T[b] <= 0:
            assert tok[b] == int(np.argmax(np.where(np.isnan(l[b]), -np.inf, l[b]))) and prob[b] == 1
            continue
        z, kept, by = ref.sample_row(l[b], T[b], k[b], p[b], m[b])
        W = kept.sum()
        # an exponential of up to 2^5 in size is off by 2^-22 of itself, a floor by 1; a cut may move by one
        # weight of the edge
        slack = W * 2.0 ** -21 + 2 * len(z) + (0 if p[b] >= 1 else float(kept[by].min()) if len(by) else 0)
        run = np.cumsum(kept)
        target = math.floor(int(np.float32(u[b]) * 2 ** 24) * W / 2 ** 24)
        i = int(tok[b])
        assert run[i] + slack > target >= run[i] - kept[i] - slack, (b, i)
        if kept[i] > 0:
            assert abs(prob[b] - kept[i] / W) <= (slack / W + 2.0 ** -20) * prob[b] + 2.0 ** -30
        else:
            assert p[b] < 1  # only the edge of a top-p cut may differ


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V,B,pad", [(1, 3, 0), (2, 9, 1), (37, 64, 3), (1000, 40, 0), (2048, 33, 0), (32000, 24, 0),
                                    (50257, 9, 1), (131073, 5, 0), (300001, 2, 7), (400003, 2, 1)])
def test_sample(gpu_lib, dtype, V, B, pad):
    rng = np.random.default_rng(V)
    l = rng.normal(0, 3, (B, V)) + (rng.random((B, V)) < 4 / V) * rng.uniform(0, 12, (B, V))
    l[rng.random((B, V)) < 0.02] = -np.inf
    l[rng.random((B, V)) < 0.001] = np.nan
    l[:, rng.integers(0, V)] = 1.5
    l = np.asarray(torch.tensor(l).to(DT[dtype]).float())
    u = rng.random(B).astype(np.float32).clip(0, 1 - 2.0 ** -24)
    u[0] = 0
    T = rng.choice([0, 0.3, 0.7, 1, 1.3], B).astype(np.float32)
    k = rng.choice([0, 1, 2, 40, 500, V, V + 5], B)
    p = rng.choice([0, 0.1, 0.5, 0.9, 0.99, 1], B).astype(np.float32)
    m = rng.choice([0, 0.01, 0.1, 0.9, 2], B).astype(np.float32)
    tok, prob = run_sample(l, u, T, k, p, m, dtype, pad)
    check_sample(l, u, T, k, p, m, tok, prob)
    # one filter at a time
    one, zero, no = np.ones(B, np.float32), np.zeros(B, np.float32), np.zeros(B, np.int64)
    for kw in (dict(), dict(T=one * 0.8), dict(k=k), dict(p=p), dict(m=m)):
        full = dict(T=one, k=no, p=one, m=zero) | kw
        check_sample(l, u, full["T"], full["k"], full["p"], full["m"], *run_sample(l, u, dtype=dtype, **kw))


@pytest.mark.parametrize("V", [5, 4097, 40000, 200003, 500001])
def test_sample_ties_go_to_the_lowest_index(gpu_lib, V):
    # equal logits: every weight is 2^31 exactly, so the token is floor(u n) of the first n kept
    u = np.array([0, 0.25, 0.5, 0.999, 1 - 2.0 ** -24], np.float32)
    l = np.full((5, V), -3.25)
    u24 = (u.astype(np.float64) * 2 ** 24).astype(np.int64)
    for k, p, n in ((0, 1.0, V), (3, 1.0, 3), (0, 0.5, math.ceil(V / 2)), (4, 0.5, 2), (V - 1, 0.75, None)):
        tok, prob = run_sample(l, u, k=[k] * 5, p=[p] * 5)
        if n is None:
            n = -(-math.floor(0.75 * (V - 1) * 2 ** 31) // 2 ** 31)
        assert tok.tolist() == [int(x) * n >> 24 for x in u24]
        assert np.allclose(prob, 1 / n, rtol=1e-6)
    # two groups of equal logits: top-k ends inside the lower one
    l = np.where(np.arange(V) % 5 == 4, 2.0, 0.0)[None]
    n = V // 5
    tok, _ = run_sample(l, [1 - 2.0 ** -24], k=[n + 2], T=[50.0])
    assert tok[0] == max(1, (n * 5 - 1))
    tok, _ = run_sample(l, [0.0], k=[n + 2], T=[50.0])
    assert tok[0] == 0


def test_sample_empty_infinite_and_odd_rows(gpu_lib):
    V = 33000
    l = np.zeros((6, V), np.float32)
    l[0] = -np.inf
    l[1] = np.nan
    l[2, [7, 900]] = np.inf
    l[3] = -np.inf
    l[3, 21] = -1e30
    l[4, :] = -np.finfo(np.float32).max
    l[4, 5] = 0
    l[5, [11, 12]] = np.finfo(np.float32).max
    u = np.array([0.3, 0.3, 0.6, 0.9, 0.9, 0.2], np.float32)
    for kw in ({}, dict(k=[3] * 6, p=[0.9] * 6, m=[0.1] * 6), dict(T=[0.5] * 6)):
        tok, prob = run_sample(l, u, **kw)
        assert tok.tolist() == [-1, -1, 900, 21, 5, 11]
        assert prob.tolist() == [0, 0, 0.5, 1, 1, 0.5]
    tok, prob = run_sample(l, u, T=[0.0, 0, 0, -1, 0, 0])
    assert tok.tolist() == [-1, -1, 7, 21, 5, 11] and prob.tolist() == [0, 0, 1, 1, 1, 1]


def test_sample_extreme_temperatures(gpu_lib):
    # z that all round to one value, or to infinities: ties by index
    V = 5000
    rng = np.random.default_rng(2)
    l = np.sort(rng.normal(0, 1, (4, V)).astype(np.float32), axis=1)
    T = np.array([1e38, 1e30, 1e-38, 1e-20], np.float32)
    u = np.array([0.5, 0.999, 0.5, 0.5], np.float32)
    for kw in (dict(), dict(k=[7] * 4), dict(p=[0.5] * 4), dict(k=[100] * 4, p=[0.3] * 4)):
        full = dict(k=[0] * 4, p=[1.0] * 4) | kw
        tok, prob = run_sample(l, u, T=T, **kw)
        check_sample(l, u, T, full["k"], full["p"], [0] * 4, tok, prob)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sample_flat_rows(gpu_lib, dtype):
    # nearly flat logits put thousands of tokens around every cut
    V, B = 60000, 12
    rng = np.random.default_rng(4)
    l = rng.normal(0, np.array([1e-3, 0.05, 0.5] * 4)[:, None], (B, V))
    l = np.asarray(torch.tensor(l).to(DT[dtype]).float())
    u = rng.random(B).astype(np.float32).clip(0, 1 - 2.0 ** -24)
    k = np.array([0, 30000, 5000, 0] * 3)
    p = np.array([0.5, 1, 0.9, 0.999, 0.03, 0.5] * 2, np.float32)
    one, zero = np.ones(B, np.float32), np.zeros(B, np.float32)
    check_sample(l, u, one, k, p, zero, *run_sample(l, u, one, k, p, zero, dtype))


@pytest.mark.parametrize("V,B", [(320000, 2), (1000000, 1), (320000, 101), (70000, 150)])
def test_sample_nearly_equal_long_rows(gpu_lib, V, B):
    # weights just below the largest fill one bin with the whole row
    rng = np.random.default_rng(V)
    l = rng.uniform(-1e-3, 0, (B, V)).astype(np.float32)
    l[:, 7] = 1e-3
    u = rng.random(B).astype(np.float32).clip(0, 1 - 2.0 ** -24)
    rows = rng.choice(B, min(B, 3), replace=False)
    one, none = np.ones(B, np.float32), np.zeros(B, np.int64)
    for k, p in ((none, one * np.float32(0.5)), (none + V // 3, one), (none + V // 2, one * np.float32(0.9)), (none, one)):
        tok, prob = run_sample(l, u, one, k, p)
        check_sample(l[rows], u[rows], one, k, p, 0 * one, tok[rows], prob[rows])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V,B,pad", [(2049, 150, 1), (32000, 160, 0), (32003, 149, 5), (131075, 130, 3)])
def test_sample_many_rows(gpu_lib, dtype, V, B, pad):
    # a block a row, and rows that each start at another alignment
    rng = np.random.default_rng(V + B)
    l = (rng.standard_normal((B, V), np.float32) * 3).astype(np.float32)
    l[rng.random((B, V), np.float32) < 0.01] = -np.inf
    l[:, ::97] = 2.25
    l = np.asarray(torch.tensor(l).to(DT[dtype]).float())
    u = rng.random(B).astype(np.float32).clip(0, 1 - 2.0 ** -24)
    T = rng.choice([0, 0.7, 1, 1.3], B).astype(np.float32)
    k = rng.choice([0, 1, 50, 300, 5000], B)
    p = rng.choice([0.3, 0.9, 0.99, 1], B).astype(np.float32)
    m = rng.choice([0, 0, 0.02], B).astype(np.float32)
    tok, prob = run_sample(l, u, T, k, p, m, dtype, pad)
    rows = np.concatenate([[0, B - 1], rng.choice(B, 40, replace=False)])
    check_sample(l[rows], u[rows], T[rows], k[rows], p[rows], m[rows], tok[rows], prob[rows])


def test_sample_frequencies(gpu_lib):
    # 4,096 uniforms on a grid draw each token as often as its weight says, within one draw
    p = np.array([0.5, 0.25, 0.125, 0.0625, 0.0625])
    l = np.tile(np.log(p), (4096, 1)).astype(np.float32)
    tok, _ = run_sample(l, (np.arange(4096) + 0.5) / 4096)
    assert np.abs(np.bincount(tok, minlength=5) - 4096 * p).max() <= 1


# ---------------------------------------------------------------------------
# a step's operators together

@pytest.mark.parametrize("heads,kv_heads,dim,slots,pages", [(8, 2, 64, 4, 13), (4, 4, 32, 7, None)])
def test_server(gpu_lib, heads, kv_heads, dim, slots, pages):
    """Greedy requests that share a pool against each request alone in 64 bits without a cache.

    Codes are off by half a step of a block's largest value (about 4 standard deviations / 127), some times over where
    the scale grows: 0.02 of a value's deviation for keys and values each.  Two layers and the output rows keep that
    size, so logits (deviation 1) are off by about 0.06 and two of them by 0.4 at most; the gap of the two largest of
    1,000 logits is 0.3 on average, so most tokens are the largest's own."""
    from specdec_b200.ragged_demo import Model, Server

    model = Model(heads=heads, kv_heads=kv_heads, dim=dim, dtype=torch.float32)
    server = Server(model, slots=slots, max_len=256, pages=pages, page_tokens=32, chunk=20)
    rng = np.random.default_rng(15)
    prompts = [rng.integers(0, model.vocab, n).tolist() for n in [1, 70, 20, 21, 33, 64, 5, 100, 1, 40]]
    out = server.serve(prompts, 12, temperature=0.0)
    n_pages = server.ring.shape[0]
    head, free = server.state[server.turn].tolist()
    assert free == n_pages == server.free and sorted(server.ring.tolist()) == list(range(n_pages))
    double = Model(heads=heads, kv_heads=kv_heads, dim=dim, dtype=torch.float64)
    for name in ("embed", "wo", "wqkv"):  # the same weights
        w = getattr(model, name)
        setattr(double, name, w.double() if name == "embed" else [x.double() for x in w])
    own = 0
    for p, o in zip(prompts, out):
        assert o[:len(p)] == p and len(o) == len(p) + 12

        def attention(layer, q, k, v):
            n, g = len(q), heads // kv_heads
            k, v = (t.repeat_interleave(g, 1) for t in (k, v))
            s = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(dim)
            s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -math.inf)
            return torch.einsum("hij,jhd->ihd", s.softmax(2), v)

        ids = torch.tensor(o, device="cuda")
        logits = double.forward(ids, torch.arange(len(o), device="cuda"), attention)(slice(len(p) - 1, len(o) - 1))
        took = logits.gather(1, ids[len(p):, None])[:, 0]
        best = logits.max(1).values
        assert bool((took >= best - 0.4).all()), float((best - took).max())
        own += int((took == best).sum())
    assert own > 12 * len(prompts) / 2
    # drawn tokens: the same seed gives the same tokens, whatever ran before
    a, b = (server.serve(prompts[:6], 9, seed=3) for _ in range(2))
    assert a == b and all(0 <= t < model.vocab for r in a for t in r)


def test_a_step_in_a_graph(gpu_lib):
    # the four calls captured once and replayed on new lengths, rows and uniforms give what the calls give
    H, Hkv, D, P, t, B, cols = 4, 2, 64, 32, 16, 5, 6
    rng = np.random.default_rng(16)
    h = sd.KV8(H, Hkv, D, page_tokens=P, block_tokens=t, max_batch=B)
    z = dict(dtype=torch.int32, device="cuda")
    T = 16

    def state():
        s = dict(table=torch.full((B, cols), -1, **z), kv_len=torch.zeros(B, **z), cu_q=torch.zeros(B + 1, **z),
                 tok_req=torch.zeros(T, **z), tok_pos=torch.zeros(T, **z), slots=torch.zeros(T, dtype=torch.int64, device="cuda"),
                 status=torch.zeros(1, **z))
        s["batch"] = sd.KV8Batch(**s)
        s["layer"] = sd.KV8Layer(*(torch.zeros(B * cols, Hkv, P, D, dtype=torch.int8, device="cuda") for _ in range(2)),
                                 *(torch.zeros(B * cols, Hkv, P // t, device="cuda") for _ in range(2)))
        s.update(held=torch.zeros(B, **z), keep=torch.zeros(B, **z), q_len=torch.zeros(B, **z),
                 ring=torch.arange(B * cols, **z), at=torch.tensor([0, B * cols], **z), at2=torch.zeros(2, **z),
                 k=torch.zeros(T, Hkv, D, device="cuda"), v=torch.zeros(T, Hkv, D, device="cuda"),
                 q=torch.zeros(T, H, D, device="cuda"), out=torch.zeros(T, H, D, device="cuda"),
                 u=torch.zeros(T, device="cuda"), tok=torch.zeros(T, **z))
        return s

    def run(s):
        st = torch.cuda.current_stream().cuda_stream
        h.plan(s["batch"], s["held"], s["keep"], s["q_len"], s["ring"], s["at"], s["at2"], stream=st)
        h.append(s["layer"], s["batch"], s["k"], s["v"], stream=st)
        h.attend(s["layer"], s["batch"], s["q"], s["out"], max_q=4, stream=st)
        sd.sample(s["out"].view(T, H * D)[:, :200], s["u"], s["tok"], stream=st)
        s["at"].copy_(s["at2"])
        s["held"].copy_(s["kv_len"])

    a, b = state(), state()
    run(b)  # nothing yet; kernels are loaded
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(b)
    held = np.zeros(B, np.int64)
    for step in range(12):
        keep = np.maximum(held - rng.integers(0, 3, B), 0)
        q = rng.integers(0, 4, B)
        new = dict(keep=keep, q_len=q)
        rows = {n: rng.normal(0, 1, tuple(a[n].shape)).astype(np.float32) for n in ("k", "v", "q")}
        rows["u"] = rng.random(T).astype(np.float32).clip(0, 1 - 2.0 ** -24)
        for s in (a, b):
            for n, v in new.items():
                s[n].copy_(i32(v))
            for n, v in rows.items():
                s[n].copy_(cu(v))
        run(a)
        graph.replay()
        torch.cuda.synchronize()
        held = keep + q
        assert int(a["status"][0]) == 0 and a["kv_len"].tolist() == held.tolist()
        for n in ("table", "kv_len", "cu_q", "tok_req", "tok_pos", "slots", "ring", "at", "out", "tok"):
            assert torch.equal(a[n], b[n]), (step, n)
    h.check()


# ---------------------------------------------------------------------------
# refusals

def test_refusals(gpu_lib):
    for bad in (dict(n_heads=6, n_kv_heads=4, head_dim=64), dict(n_heads=4, n_kv_heads=4, head_dim=48),
                dict(n_heads=4, n_kv_heads=4, head_dim=64, page_tokens=256),
                dict(n_heads=4, n_kv_heads=4, head_dim=64, page_tokens=32, block_tokens=64),
                dict(n_heads=4, n_kv_heads=4, head_dim=64, block_tokens=8),
                dict(n_heads=4, n_kv_heads=4, head_dim=64, max_batch=5000), dict(n_heads=0, n_kv_heads=1, head_dim=64)):
        with pytest.raises(sd.SpecDecError) as e:
            sd.KV8(**bad)
        assert e.value.code == 1
    h = sd.KV8(4, 2, 64, max_batch=2)
    rng = np.random.default_rng(0)
    cache = [cu(a) for a in make_cache(rng, 3, 2, 128, 64, 16)]
    layer = sd.KV8Layer(*cache)
    batch = sd.KV8Batch(i32([[0], [1]]), i32([5, 7]), i32([0, 1, 2]))
    q = torch.zeros(2, 4, 64, device="cuda")
    with pytest.raises(ValueError):
        h.attend(layer, batch, q[:, :3], q)
    with pytest.raises(ValueError):
        h.attend(layer, batch, q.half(), q.half())
    with pytest.raises(ValueError):
        h.attend(layer, batch, q, torch.zeros(3, 4, 64, device="cuda"))
    with pytest.raises(ValueError):
        h.attend(layer, batch, q.transpose(1, 2).contiguous().transpose(1, 2), q)
    with pytest.raises(ValueError):
        sd.KV8Layer(cache[0].float(), *cache[1:])
    with pytest.raises(ValueError):
        sd.KV8Layer(cache[0], cache[1], cache[2][:, :, :4].contiguous(), cache[3])
    with pytest.raises(ValueError):
        sd.KV8Batch(i32([[0], [1]]), i32([5]), i32([0, 1, 2]))
    for kw in (dict(max_q=-1), dict(window=-2), dict(scale=float("nan"))):
        with pytest.raises(sd.SpecDecError) as e:
            h.attend(layer, batch, q, torch.zeros_like(q), **kw)
        assert e.value.code == 1
    three = sd.KV8Batch(i32([[0], [1], [2]]), i32([5, 7, 1]), i32([0, 1, 2, 2]))
    with pytest.raises(sd.SpecDecError):
        h.attend(layer, three, q, torch.zeros_like(q))
    with pytest.raises(sd.SpecDecError):  # a plan needs the row arrays
        h.plan(batch, i32([1, 1]), i32([1, 1]), i32([1, 1]), i32([0, 1, 2]), i32([0, 1]), i32([0, 0]))
    state = i32([0, 1])
    full = sd.KV8Batch(i32([[0], [1]]), i32([5, 7]), i32([0, 1, 2]), i32([0] * 4), i32([0] * 4),
                       torch.zeros(4, dtype=torch.int64, device="cuda"), i32([0]))
    with pytest.raises(sd.SpecDecError):  # in and out state in one place
        h.plan(full, i32([1, 1]), i32([1, 1]), i32([1, 1]), i32([0, 1, 2]), state, state)
    l, tok, u = torch.zeros(2, 9, device="cuda"), i32([0, 0]), torch.zeros(2, device="cuda")
    with pytest.raises(ValueError):
        sd.sample(l.half(), u, tok)
    with pytest.raises(ValueError):
        sd.sample(l, u[:1], tok)
    with pytest.raises(ValueError):
        sd.sample(l.T, u, tok)
    with pytest.raises(sd.SpecDecError):
        sd.sample(l[:, :0], u, tok)
    # buffers of the host are never passed on
    host = torch.zeros(2, 4, 64)
    with pytest.raises(ValueError):
        h.attend(layer, batch, host, q)
    with pytest.raises(ValueError):
        h.attend(layer, batch, q, host)
    with pytest.raises(ValueError):
        h.append(layer, batch, host[:, :2], host[:, :2])
    with pytest.raises(ValueError):
        h.gather(layer, torch.zeros(2, dtype=torch.int64, device="cuda"), host[:, :2].contiguous())
    with pytest.raises(ValueError):
        sd.sample(l.cpu(), u, tok)
    with pytest.raises(ValueError):
        sd.KV8Batch(torch.zeros(2, 1, dtype=torch.int32), i32([5, 7]), i32([0, 1, 2]))
    # calls of nothing are calls
    none = sd.KV8Batch(torch.zeros(0, 1, dtype=torch.int32, device="cuda"), i32([]), i32([0]))
    h.attend(layer, none, q[:0], q[:0])
    h.append(layer, none, q[:0, :2], q[:0, :2])
    h.gather(layer, torch.zeros(0, dtype=torch.int64, device="cuda"), q[:0, :2], None)
    sd.sample(l[:0], u[:0], tok[:0])
    torch.cuda.synchronize()
