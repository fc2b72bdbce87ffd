"""The sampler's weights at the borders that one unit of 2^-43 decides."""
import math

import pytest
import torch

from _served_oracle import choose

pytestmark = pytest.mark.gpu

# A logit below the largest and a whole number that is its weight, round(2^43 exp(x)), or one more than that; min_p of a 2^43th of the number, which
# fp32 holds, keeps the first kind and drops the second.  2^43 exp(x) is 0.2 at least from a half.
BORDERS = [
    ("-0x1.4aa11p-6", 8620366888960, True), ("-0x1.7904c6p-6", 8595993788416, True), ("-0x1.a5802ap-6", 8572687613952, True),
    ("-0x1.2cc324p-5", 8479008358400, True), ("-0x1.5c575ep-4", 8078961934336, True), ("-0x1.010d72p-3", 7758536507392, True),
    ("-0x1.ca2fecp-1", 3594521149440, True), ("-0x1.6f3b42p-6", 8601130237952, True), ("-0x1.dc808ap-6", 8543957155840, True),
    ("-0x1.dde44p-6", 8543232589824, True), ("-0x1.e97312p-6", 8537207996416, True), ("-0x1.11e144p-6", 8650276995072, False),
    ("-0x1.268fd2p-6", 8639364464640, False), ("-0x1.3563a4p-6", 8631549427712, False), ("-0x1.41fdf6p-6", 8624912465920, False),
    ("-0x1.4f7c96p-6", 8617811509248, False), ("-0x1.b64f1ap-6", 8563897401344, False), ("-0x1.d4ff24p-6", 8547872014336, False),
    ("-0x1.e60344p-6", 8538998964224, False), ("-0x1.eda65ap-6", 8535019618304, False), ("-0x1.1c8138p-5", 8495852158976, False),
    ("-0x1.251316p-5", 8486969147392, False), ("-0x1.29e592p-5", 8481974779904, False)]
BORDERS = [(float.fromhex(x), w, kept) for x, w, kept in BORDERS]


@pytest.mark.parametrize("t", [1.0, 4.0, 0.125])
@pytest.mark.parametrize("V", [2, 400, 20000])
def test_weights_at_the_border_of_min_p(cuda_device, V, t):
    """By the list of a small vocabulary and by the sums of a large one; powers of two as temperatures leave the weights as they are."""
    from frankentorch_b200.ops import decode as D
    n = len(BORDERS)
    x = torch.full((n, V), -math.inf, device="cuda")
    x[:, 0] = 0.0
    x[:, V - 1] = torch.tensor([b[0] * t for b in BORDERS], dtype=torch.float64).float()
    least = torch.tensor([b[1] / 2 ** 43 for b in BORDERS], dtype=torch.float64)
    assert torch.equal(least.float().double(), least) and torch.equal(x[:, V - 1].double().cpu() / t, torch.tensor([b[0] for b in BORDERS]).double())
    token, logprob = D.sample(x, torch.ones(n, device="cuda"), temperature=t, min_p=least.float().cuda())      # the last one that is kept
    for r, (v, low, kept) in enumerate(BORDERS):
        want = choose([0.0, v * t], 1.0, t, 0, 1.0, float(least[r]))
        assert want[0] == int(kept)
        assert int(token[r]) == (V - 1 if kept else 0), (r, v, low)
        assert abs(float(logprob[r]) - want[1]) <= 2.0 ** -24 * abs(want[1]) + 1e-9


def test_weights_at_the_border_of_top_p(cuda_device):
    """Two tokens that are kept only as long as less than p of the sum lies before the second: p of 2^43 over the sum, to either side."""
    from frankentorch_b200.ops import decode as D
    rows, p = [], []
    for x, low, kept in BORDERS:
        w = low if kept else low - 1
        share = torch.tensor(2 ** 43 / (2 ** 43 + w), dtype=torch.float64).float()
        for q in (share, torch.nextafter(share, torch.tensor(0.0)), torch.nextafter(share, torch.tensor(1.0))):
            rows.append([0.0, x])
            p.append(float(q))
    token, _ = D.sample(torch.tensor(rows, device="cuda"), torch.ones(len(rows), device="cuda"), top_p=torch.tensor(p, device="cuda"))
    for r, row in enumerate(rows):
        assert int(token[r]) == choose(row, 1.0, 1.0, 0, p[r], 0.0)[0], (row, p[r])
