"""attn_paged over batches of another make: thousands of sequences of a few tokens each."""
import numpy as np
import pytest

from paged_ref import Batch
from test_gpu_paged_repair import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("seqs,heads", [(700, (6, 2, 64)), (4096, (6, 1, 16)), (1500, (4, 1, 256))])
def test_thousands_of_short_chunks(device, seqs, heads, i8):
    """Where each sequence's tiles begin takes as much room as queries and keys behind it, which the copy engine then fills."""
    n_q, n_kv, d = heads
    rng = np.random.default_rng(seqs)
    new = [int(n) for n in rng.integers(0, 8, seqs)]
    b = Batch(new, [int(c) for c in rng.integers(0, 20, seqs)], n_q=n_q, n_kv=n_kv, d=d, page=16, i8=i8, pad=3)
    check(device, b)
