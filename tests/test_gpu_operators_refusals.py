"""What the operators around the Linear do not take is refused by the library, with its own error, in front of the forward."""
import pytest
import torch

from optimus_dl_amd.modules.logprobs import token_logprobs
from optimus_dl_amd.native import NativeError

pytestmark = pytest.mark.gpu


def zeros(rows, cols, grad):
    return torch.zeros((rows, cols), device="cuda", dtype=torch.bfloat16, requires_grad=grad), torch.zeros(rows, dtype=torch.int64, device="cuda")


@pytest.mark.parametrize("grad", [True, False])
def test_more_rows_than_a_call_takes(grad):
    with pytest.raises(NativeError, match="rows"):
        token_logprobs(*zeros(1 << 22, 1, grad))


def test_more_columns_than_the_backward_takes():
    wide = zeros(1, (1 << 24) + 8, True)
    for n_vocab in (None, 100):
        with pytest.raises(NativeError, match="columns"):
            token_logprobs(*wide, n_vocab=n_vocab)
    with torch.no_grad():                                      # nothing is written to the columns behind the vocabulary: any number of them
        r = token_logprobs(*wide, n_vocab=100)
    assert abs(r.logprobs.item() + 4.6051702) < 1e-5
