"""Penalties, biases, grammars, several samples and shared prefixes over vocabulary and head shards: two gloo processes on the CPU choose the
tokens that one process chooses."""
import os
import socket

import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from helpers import build, tiny_config
from jax_llama_amd import GenerationConfig, TokenGrammar

V, B, S, NEW = 256, 2, 7, 10
CFG = dict(num_key_value_heads=2, intermediate_size=128, vocab_size=V)


def prompts(b, s, seed):
    return torch.randint(3, V, (b, s), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)


def grammar():
    """Tokens of both shards in turn: 8 k + state, for 4 states."""
    t = torch.full((4, V), -1)
    for s in range(4):
        t[s, s::8] = (s + 1) % 4
        t[s, V // 2 + s::8] = (s + 2) % 4
    return TokenGrammar(t)


def runs(model):
    ids, head = prompts(B, S, 0), prompts(1, 12, 1)

    def config(**kw):
        return GenerationConfig(**{**dict(max_length=S + NEW, do_sample=False, pad_token_id=2, eos_token_id=-1), **kw})

    free = model.generate(ids, generation_config=config()).sequences
    low, high = [int(t) for t in free[:, S:].reshape(-1) if t < V // 2], [int(t) for t in free[:, S:].reshape(-1) if t >= V // 2]
    bias = torch.linspace(-0.05, 0.05, V)
    prefix = model.encode_prefix(head)
    return dict(free=free, penalised=model.generate(ids, generation_config=config(repetition_penalty=1.5, presence_penalty=0.3, frequency_penalty=0.2)).sequences,
                biased=model.generate(ids, generation_config=config(logit_bias=bias, suppress_tokens=low[:2] + high[:2])).sequences,
                once=model.generate(ids, generation_config=config(presence_penalty=1e4)).sequences,
                grammar=model.generate(ids, generation_config=config(grammar=grammar())).sequences,
                samples=model.generate(ids, generation_config=config(repetition_penalty=1.2, do_sample=True, top_k=4, seed=7), num_return_sequences=3).sequences,
                behind=model.generate(ids, generation_config=config(), prefix=prefix).sequences)


def _worker(rank, world, port, q):
    try:
        os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world), LOCAL_RANK=str(rank))
        from jax_llama_amd.models import LLaMAForCausalLM
        from jax_llama_amd.parallel import TPComm, init_distributed
        ctx = init_distributed(backend="gloo", device_type="cpu")
        ctx.setup_mesh(tp=world)
        cfg = tiny_config(**CFG)
        _, _, _, params = build(cfg, seed=11)
        model = LLaMAForCausalLM(cfg, comm=TPComm.from_context(ctx), _do_init=False).load_params(params)
        q.put(("ok", rank, {k: t.tolist() for k, t in runs(model).items()}))
        dist.barrier()
        dist.destroy_process_group()
    except Exception:  # pragma: no cover - surfaced in the parent
        import traceback
        q.put(("err", rank, traceback.format_exc()))


def test_rules_samples_and_prefixes_under_tensor_parallelism():
    want = {k: t.tolist() for k, t in runs(build(tiny_config(**CFG), seed=11)[0]).items()}
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_worker, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    got = [q.get(timeout=240) for _ in procs]
    for p in procs:
        p.join(timeout=60)
    for status, _, out in got:
        assert status == "ok", out
        assert out == want
    allowed = [set(torch.nonzero(row >= 0).reshape(-1).tolist()) for row in grammar().next_state]
    for row in want["grammar"]:
        state = 0
        for t in row[S:]:
            assert t in allowed[state]
            state = int(grammar().next_state[state, t])
    assert all(len(set(row[S:])) == NEW for row in want["once"])
