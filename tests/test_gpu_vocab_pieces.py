"""What a model answers and its gradients where the vocabulary goes by in several pieces.  Bounds as for one piece
(test_gpu_vocab_answers)."""

import pytest
import torch

import npeff_ref_amd as d
from test_gpu_vocab_answers import DTYPES, empty, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("rows, words, n_in", [(600, 60_000, 264), (1300, 40_000, 100), (520, 70_000, 515)])
def test_ties_across_pieces(rows, words, n_in, dt):
    """One embedding many times over, more often than a list holds in the small first piece and in what comes after it: the first of
    them lead, whatever products each piece is formed by."""
    X, E = rand((rows, n_in), dt, 1).float(), rand((words, n_in), dt, 2, 0.05)
    v = rand((1, n_in), "f32", 3)
    X = (X + v).to(DTYPES[dt])
    same = torch.cat([torch.arange(70, 1000, 20), torch.arange(1500, words, 701)]).cuda()
    E[same] = (0.3 * v).to(DTYPES[dt])
    top_words, top_logp = empty(rows, 20, dtype=torch.int32), empty(rows, 20)
    d.op_vocab_probs(X, E, top_words=top_words, top_logp=top_logp)
    z = X.double() @ E.double().T
    z[:, same] = z[:, same[:1]]
    at = z.sort(dim=1, descending=True, stable=True).indices[:, :20]
    assert (at == same[:20]).all(1).double().mean() > 0.9
    assert torch.equal(top_words, at.to(torch.int32))
    assert (top_logp[:, :1] == top_logp)[(at == same[:20]).all(1)].all()
