"""Histories that are empty, begin behind their end, or end at the last place that 32 bits count."""
import pytest
import torch

import oracle_serving as oracle
from jax_llama_amd import ops

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]
I32, LAST = torch.int32, 2 ** 31 - 1
PENALTIES = dict(repetition_penalty=1.3, presence_penalty=0.25, frequency_penalty=0.5)


def check(x, got, **kw):
    want, bound = oracle.process_logits(x, **kw)
    assert bool(((got.double().cpu() - want).abs() <= bound).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("v,n", [(100, 60), (14001, 300), (14001, 600)])  # (in place: few places against the columns, many)
def test_starts_behind_the_end(device, v, n):
    starts = torch.tensor([LAST, LAST - 1, LAST - 500, LAST - 1020, LAST - 4000, n, n + 1, n - 1, -LAST - 1, -5, 0], dtype=I32)
    b = len(starts)
    x, h = torch.randn(b, v), torch.randint(0, v, (b, n), dtype=I32)
    for length in (n, 1, 0):
        kw = dict(start=starts, prompt_len=n // 2, **PENALTIES)
        on = {k: t.to(device) if torch.is_tensor(t) else t for k, t in kw.items()}
        for given in (length, torch.tensor([length], dtype=I32, device=device)):
            got = ops.process_logits(x.to(device), history=h.to(device), length=given, **on)
            check(x, got, history=h, length=length, **kw)
            y = x.to(device)
            assert torch.equal(ops.process_logits(y, history=h.to(device), length=given, out=y, **on), got)
        silent = [i for i in range(b) if int(starts[i]) >= length]
        assert torch.equal(got[silent].cpu(), x[silent])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("length", [-1, -LAST - 1, -LAST + 1000, 61, LAST, LAST - 1000])
def test_device_lengths_outside_the_history(device, length):
    """Nothing below 0, all of it past its end."""
    x, h = torch.randn(3, 100), torch.randint(0, 100, (3, 60), dtype=I32)
    got = ops.process_logits(x.to(device), history=h.to(device), length=torch.tensor([length], dtype=I32, device=device), prompt_len=20, **PENALTIES)
    check(x, got, history=h, length=max(0, min(length, 60)), prompt_len=20, **PENALTIES)


@pytest.mark.gpu
def test_a_history_of_2_to_the_31_places():
    """Its last places, behind a start near the end."""
    v, near = 5000, 3001
    h = torch.empty(1, LAST, dtype=I32, device="cuda:0")
    tail = torch.randint(0, v, (1, near), dtype=I32)
    h[:, LAST - near:] = tail.to("cuda:0")
    x = torch.randn(1, v)
    got = ops.process_logits(x.to("cuda:0"), history=h, length=LAST, start=torch.tensor([LAST - near], dtype=I32, device="cuda:0"),
                             prompt_len=LAST - 1000, **PENALTIES)
    check(x, got, history=tail, length=near, prompt_len=near - 1000, **PENALTIES)
