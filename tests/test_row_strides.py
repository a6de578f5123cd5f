"""How far apart draft_verify takes the rows of p and q to lie, by the shape in which they come (no GPU needed: the call is caught
before it reaches the library)."""
import pytest


class Caught:
    def __init__(self):
        self.args = None

    def q27h_draft_verify(self, *args):
        self.args = args
        return 0


@pytest.fixture
def strides(q27, monkeypatch):
    import torch

    def of(p, q, T, V):
        c = Caught()
        monkeypatch.setattr(q27.ops, "lib", lambda: c)
        x = torch.zeros(T, dtype=torch.int32)
        q27.ops.draft_verify(p, q, x, None, x, x, x, 2, V, x, x, x, x, 0)
        return c.args[1], c.args[3]

    return of


def test_two_dimensions(strides):
    import torch

    x = torch.zeros(6, 40)
    assert strides(x, None, 6, 40) == (40, 40)
    assert strides(x[:, :33], x[::2, :33], 6, 33) == (40, 80)
    assert strides(x[:1, :33], None, 1, 33) == (33, 33)


def test_sequences_tokens_values(strides):
    import torch

    x = torch.zeros(2, 3, 40)
    assert strides(x, None, 6, 40) == (40, 40)
    assert strides(x[..., :33], x[..., 7:], 6, 33) == (40, 40)
    assert strides(x, x, 6, 33) == (40, 40)  # the values behind V are none of a row
    assert strides(torch.zeros(2, 3, 1, 40)[..., :33], None, 6, 33)[0] == 40
    assert strides(torch.zeros(1, 1, 40)[..., :33], None, 1, 33)[0] >= 33


def test_rows_that_are_not_evenly_apart_are_refused(strides):
    import torch

    x = torch.zeros(2, 4, 40)
    for bad in (x[:, :3], x.transpose(0, 1), x[..., ::2]):
        for p, q in ((bad, None), (x[:, :3].contiguous(), bad)):
            with pytest.raises(ValueError):
                strides(p, q, 6, bad.shape[-1])
