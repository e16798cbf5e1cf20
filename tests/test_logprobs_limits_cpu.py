"""How many segments of logits a call of the log probabilities takes, as its header says."""
import pytest

from evo_hip import native as N
from test_paged_cpu import A
from test_serving_cpu import logprobs

MOST = (1 << 26) - 4  # of rows * ceil(vocab / 2048)


@pytest.mark.parametrize("rows,vocab", [(1 << 20, 1 << 20), (1 << 20, 64 * 2048 + 1),
                                        (MOST // 64 + 1, 64 * 2048), (1 << 17, 1 << 20)])
def test_more_are_refused_by_the_size_too(rows, vocab):
    assert rows * -(-vocab // 2048) > MOST
    assert N.call("evo_hip_token_logprobs_workspace_bytes", rows, vocab, 4) == 0
    with pytest.raises(N.OpError, match="grid too large"):
        logprobs(rows=rows, vocab=vocab, stride=vocab, workspace=A, size=1 << 62)


@pytest.mark.parametrize("rows,vocab", [(MOST // 64, 64 * 2048), ((1 << 17) - 1, 1 << 20),
                                        (1 << 20, 2049)])
def test_up_to_the_limit_there_is_a_size(rows, vocab):
    assert rows * -(-vocab // 2048) <= MOST
    assert N.call("evo_hip_token_logprobs_workspace_bytes", rows, vocab, 4) > 0
