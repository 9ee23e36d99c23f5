"""A fork that fails leaves the stepper as it was."""
import pytest
import torch

import test_zavevik
from jax_llama_amd import SequenceStepper


def test_a_fork_that_fails(monkeypatch):
    model = test_zavevik.build(test_zavevik.cfg_full(), "cpu")[0]
    tok = torch.randint(3, 37, (9,), generator=torch.Generator().manual_seed(2)).tolist()
    st, want = SequenceStepper(model, 12), SequenceStepper(model, 12)
    for s in (st, want):
        s.feed("a", tok[:4])
    cache = type(st._live["a"])

    def broken(self, *args, **kw):
        raise RuntimeError("no copies here")

    for attempt in range(3):
        with monkeypatch.context() as m:
            m.setattr(cache, "copy_rows", broken)
            with pytest.raises(RuntimeError):
                st.fork("a", "b")
        assert st.live() == ["a"] and st.held("b") == 0 and len(st._free) == 1  # (its row is kept for the next)
    st.fork("a", "b")
    assert st.live() == ["a", "b"] and st.held("b") == 4
    assert torch.equal(st.feed("b", tok[4:], [4]), want.feed("a", tok[4:], [4]))

