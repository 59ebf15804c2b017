"""attn_paged over batches of another make: thousands of sequences of a few tokens each, a prompt beside single tokens, promises of at most so many
new tokens that are not kept, first tokens in front of a window on pages of any size."""
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


@pytest.mark.parametrize("i8", [False, True])
def test_single_tokens_beside_a_prompt(device, i8):
    """Rows of a prompt that fill tiles on average: the single tokens beside it then take tiles of many rows too, behind long contexts."""
    b = Batch([500, 1, 1, 0, 1], [40, 3000, 700, 9, 2999], n_q=8, n_kv=2, d=128, page=16, i8=i8, pad=5)
    assert b.rows * 4 // b.seqs >= 128
    check(device, b)
    check(device, b, window=600, sinks=4)


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("max_new", [1, 2, 20, 64])
def test_more_new_tokens_than_promised(device, max_new, i8):
    """The rows behind those that were promised are left as they were; the others do not see their keys."""
    check(device, Batch([70, 3, 1, 33], [100, 700, 0, 5], n_q=4, n_kv=1, d=64, page=16, i8=i8), max_new=max_new)


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("page", [1, 7, 12, 20, 24])
@pytest.mark.parametrize("window,sinks", [(100, 4), (64, 70), (300, 16), (16, 200)])
def test_first_tokens_in_front_of_a_window_on_any_pages(device, page, window, sinks, i8):
    """Pages in which eight keys need not lie one behind another, ones in which they do, with first tokens in front of the window's."""
    check(device, Batch([140, 3, 20], [900, 1500, 0], n_q=4, n_kv=2, d=64, page=page, i8=i8), window=window, sinks=sinks)
