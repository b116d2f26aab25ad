"""The paged 4-bit cache's operators together, as examples/paged_kv4.py runs them."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

EXAMPLES = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "win-directml-java_b200", "examples")


def test_prompts_samples_drafts_and_compaction():
    """Against dense attention over the held rows.  Those are bf16 roundings of what the cache holds: values (and the
    outputs) up to 4.6 differ by 2^-9 of that, a score (sum over 64 channels of |q k| of at most 60, scaled by 1/8)
    by 60 / 8 * 2^-9 = 0.015, which moves a weighted mean of such values by at most twice that times 4.6."""
    sys.path.insert(0, EXAMPLES)
    import paged_kv4
    s = paged_kv4.main()
    assert s.lens.tolist() == [158, 156, 53, 71, 0, 0]
    assert 0 < s.worst <= 2 * 4.6 * 2 ** -9 + 2 * 0.015 * 4.6
    # no page is lost: the counts are the table's
    table = s.table.cpu().numpy()
    refs = s.refs.cpu().numpy()
    for page in range(refs.size):
        assert refs[page] == (table == page).sum()
    for row, n in enumerate(s.lens.tolist()):
        assert (table[row] >= 0).sum() == -(-n // paged_kv4.PAGE)


def test_every_output_of_the_example_lies_within_its_own_bound():
    """Element by element, from the weights and values that make the output (see Server.compare)."""
    sys.path.insert(0, EXAMPLES)
    import paged_kv4
    s = paged_kv4.main()
    assert 0 < s.worst_of_bound <= 1
