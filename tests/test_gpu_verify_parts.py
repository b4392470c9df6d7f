"""Verification with draft probabilities where the sums of p - q go ways of their own:
one workgroup with more parts than it keeps in LDS, and waves of some workgroups that
take more than one part.  Against the restatement in 64 bits, all equal."""
import pytest
import torch

from test_gpu_verify import TYPES, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("seqs,vocab", [(600, 9001), (520, 20011), (1030, 12000), (200, 60001), (130, 128256), (350, 32003)])
def test_sums_of_what_p_has_over_q(cuda, dtype, seqs, vocab):
    """Parts are 1024 (fp32) or 2048 logits, 8 a workgroup.  Drafts far from the target:
    most sequences draw from p - q."""
    if dtype != torch.float32 and vocab < 20000:
        vocab *= 2
    rows = [1 + s % 2 for s in range(seqs)]
    a = make(rows, vocab, dtype, seqs + vocab, True, 2.0)
    a["probs"] = a["probs"].roll(vocab // 3, 1).contiguous()
    check(a)   # (drafts that q holds for unlikely: few are rejected)
    a["drafts"] = (a["drafts"] + vocab // 3) % vocab
    accepted, _ = check(a)
    two = [n for n, r in zip(accepted, rows) if r == 2]
    assert two.count(0) > len(two) // 2


def test_one_workgroup_where_all_is_in_the_last_part(cuda):
    """The threshold falls past the sums that stay in LDS."""
    seqs, vocab = 600, 12000
    a = make([2] * seqs, vocab, torch.float32, 3, True)
    a["logits"][:, :11500] = -30.0
    a["probs"].zero_()
    a["probs"][:, :100] = 0.01
    a["drafts"].fill_(50)
    _, tokens = check(a)
    assert all(t >= 11500 for t in tokens[::2])
