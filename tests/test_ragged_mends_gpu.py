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
