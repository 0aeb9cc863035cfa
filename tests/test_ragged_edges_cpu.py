"""Edges of the ragged operators on the host: ids of near ties and NaN, bad offsets and entries, the cache's states
after an error, arguments that lie elsewhere."""
import math
import torch
from tinytron_b200 import ops


# ----------------------------------------------------------------------------- token statistics
def test_token_stats_ids_follow_the_logits():
    """Logits that differ by less than a log-prob's rounding are in their own order; a NaN is below every number."""
    x = torch.zeros(4, 50)
    x[0, 40], x[0, 10], x[0, 20] = 18.0, 1e-3, 1e-3 + 1.2e-10
    assert float(x[0, 20]) > float(x[0, 10])
    x[1, 3], x[1, 7] = math.nan, 1.0
    x[2] = -math.inf
    x[2, 5], x[2, 6] = math.nan, 2.0
    x[3, 0], x[3, 1], x[3, 2] = -0.0, math.inf, 1.0
    st = ops.token_stats(x, torch.tensor([40, 7, 6, 1]), top_k=4)
    assert st.top_ids.tolist() == [[40, 20, 10, 0], [7, 0, 1, 2], [6, 0, 1, 2], [1, 2, 0, 3]]
    last = ops.token_stats(x[1:2, :20], torch.tensor([7]), top_k=20).top_ids[0]
    assert int(last[-1]) == 3
