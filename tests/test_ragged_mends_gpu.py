"""The ragged decode operators on the GPU where they once went wrong.
Restatements are those of ragged_ref.py or stand here; tolerances are
test_ragged_gpu.py's."""
import numpy as np
import pytest

import specdec_b200 as sd
from test_ragged_gpu import check_sample, cu, run_sample

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


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
