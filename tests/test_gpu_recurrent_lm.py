"""The language model of examples/recurrent_lm.py: the operators together, trained and served."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
spec = importlib.util.spec_from_file_location("recurrent_lm", os.path.join(ROOT, "examples", "recurrent_lm.py"))
lm = importlib.util.module_from_spec(spec)
spec.loader.exec_module(lm)


def test_training_brings_the_loss_down_and_the_same_losses_every_time():
    runs = []
    for _ in range(2):
        torch.manual_seed(1)
        runs.append(lm.train(lm.RecurrentLM(32, 64, 4, 2).cuda(), 60))
    assert runs[0][-1] < 0.6 * runs[0][0], runs[0]
    # (the products are torch's; the operators' own gradients have one order)
    assert abs(runs[0][0] - runs[1][0]) < 1e-5


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_packed_prompts_and_single_tokens_give_the_logits_of_the_whole_sequence(dtype):
    torch.manual_seed(2)
    model = lm.RecurrentLM(50, 96, 3, 2, dtype=dtype).cuda()
    sequences = [torch.randint(0, 50, (n,)).cuda() for n in (1, 40, 7, 131)]
    heads = [1, 33, 7, 100]
    rows = torch.tensor([5, 0, 3, 2], dtype=torch.int32, device="cuda")
    cache = model.new_cache(6)
    bounds = torch.tensor([0] + heads).cumsum(0).to(device="cuda", dtype=torch.int32)
    logits = model.prefill(torch.cat([s[:n] for s, n in zip(sequences, heads)]), bounds, cache, rows)
    with torch.no_grad():
        whole = [model(s[None])[0].float() for s in sequences]
    # two layers of a few dozen roundings each: the unit of the type, thirty times over, of the largest logit
    bound = 30 * {torch.float32: 2.0 ** -20, torch.bfloat16: 2.0 ** -8}[dtype] * max(float(w.abs().max()) for w in whole)
    at = list(heads)
    while True:
        for n in range(4):
            assert float((logits[n].float() - whole[n][at[n] - 1]).abs().max()) <= bound, (n, at[n])
        running = [n for n in range(4) if at[n] < len(sequences[n])]
        if not running:
            break
        # requests that are done take no part
        slots = torch.tensor([int(rows[n]) if n in running else -1 for n in range(4)], dtype=torch.int32, device="cuda")
        tokens = torch.stack([sequences[n][min(at[n], len(sequences[n]) - 1)] for n in range(4)])
        step = model.step(tokens, cache, slots)
        for n in running:
            logits[n] = step[n]
            at[n] += 1
