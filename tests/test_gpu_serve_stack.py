"""The example that serves several requests through a stack of attention and
MLP layers: every attention call against the formula in 64 bits on what the
cache gives back, blocks all returned, answers the same each time."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("serve_stack", os.path.join(ROOT, "examples", "serve_stack.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("fmt,heads,dim", [("int8", (8, 2), 128), ("e4m3", (4, 4), 64)])
def test_attention_inside_the_stack(gpu, example, fmt, heads, dim):
    seen = []

    class Checked(example.Stack):
        def attend(self, i, q, step):
            out = super().attend(i, q, step)
            G, scale = q.shape[1] // self.kv_heads, dim ** -0.5
            starts, lens, table = step.q_start.tolist(), step.kv_len.tolist(), step.table.cpu()
            for r, kv in enumerate(lens):
                t0, n = starts[r], starts[r + 1] - starts[r]
                if n == 0:
                    continue
                pos = torch.arange(kv)
                slots = (table[r][pos // 16].long() * 16 + pos % 16).to(gpu)
                got = self.cache[i].read(slots)  # fp16: 2^-11 of the exact values
                hidden = pos.to(gpu)[None] > kv - n + torch.arange(n, device=gpu)[:, None]
                for h in range(q.shape[1]):
                    k, v = (got[x][:, h // G].double() for x in ("k", "v"))
                    x = q[t0: t0 + n, h].double()
                    s = (x @ k.t().contiguous() * scale).masked_fill(hidden, -torch.inf)
                    p = torch.softmax(s, 1)
                    want, spread = p @ v, p @ v.abs()
                    # rounding of the output, the weights and the values read back, 2^-11 each, and of the keys read
                    # back: 2^-11 of a score's summands, in a weight and in the sum of weights
                    slack = (x.abs() @ k.abs().t().contiguous() * scale).masked_fill(hidden, 0).amax(1, keepdim=True)
                    bound = 2.0 ** -11 * want.abs() + 2.0 ** -11 * (2.1 + 2 * slack) * spread + 2.0 ** -20
                    assert ((out[t0: t0 + n, h].double() - want).abs() <= bound).all(), (i, r, h)
            seen.append((q.shape[0], max(lens)))
            return out

    lengths, new, blocks = [70, 5, 1, 33], 4, 30
    torch.manual_seed(0)
    prompts = [torch.randint(512, (n,)) for n in lengths]
    make = dict(layers=2, hidden=1024, intermediate=4096, q_heads=heads[0], kv_heads=heads[1], head_dim=dim, vocab=512, top_k=40,
                blocks=blocks, fmt=fmt, device=gpu)
    answers = []
    for stack in (Checked(**make), example.Stack(**make)):
        batch = example.KvBatch(blocks, 16, max_requests=4, max_blocks=6, q_heads=heads[0], kv_heads=heads[1], head_dim=dim)
        for _ in range(2):  # the blocks that come back are used again
            out, _ = example.serve(stack, prompts, new, 48, batch)
            answers.append(out)
            assert batch.cached.tolist() == [0] * 4 and int(batch.state[1]) == blocks
            assert sorted(batch.ring.tolist()) == list(range(blocks))
    assert all(a == answers[0] for a in answers) and all(len(a) == new for a in answers[0])
    assert max(n for n, _ in seen) >= 48 and min(n for n, _ in seen) <= 2 and max(kv for _, kv in seen) == 70 + new - 1


def test_example_runs(gpu, example, capsys):
    answers, batch = example.main(["--layers", "1", "--hidden", "1024", "--intermediate", "4096", "--heads", "8,2", "--vocab", "512",
                                   "--prompts", "40,1,17", "--new", "3", "--chunk", "32", "--top-k", "40"])
    assert [len(a) for a in answers] == [3, 3, 3]
    assert "free blocks" in capsys.readouterr().out and int(batch.state[1]) == batch.num_blocks
