"""The serving example over the 4-bit cache: attention inside the stack on rotated rows, tokens with their log
probabilities."""
import os

import pytest
import torch

from test_gpu_kv4_edges import formula, within
from test_gpu_serve_stack import example  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,dim", [((8, 2), 128), ((4, 4), 64)])
def test_rotated_attention_and_scores(gpu, example, heads, dim):  # noqa: F811
    seen, scored = [], []

    class Checked(example.Stack):
        def attend(self, i, q, step):
            out = super().attend(i, q, step)
            starts, lens, table = step.q_start.tolist(), step.kv_len.tolist(), step.table.cpu()
            for r, kv in enumerate(lens):
                n = starts[r + 1] - starts[r]
                if n:
                    pos = torch.arange(kv)
                    got = self.cache[i].read((table[r][pos // 16].long() * 16 + pos % 16).to(gpu))
                    rows = slice(starts[r], starts[r] + n)
                    assert within(out[rows], *formula(q[rows], got["k"], got["v"], kv - n), kv), (i, r)
            seen.append(q.shape[0])
            return out

        def next_tokens(self, x):
            got = super().next_tokens(x)
            z = torch.log_softmax(example.lm_head_forward(example.norm(x)[None], self.head)[0].double(), -1)
            assert ((got["logprob"].double() - z.amax(-1)).abs() <= 2.0 ** -16).all()
            assert ((got["entropy"].double() + (z.exp() * z).sum(-1)).abs() <= 2.0 ** -14).all()
            assert torch.equal(z.gather(1, got["token"][:, None])[:, 0], z.amax(-1))
            scored.append(got["logprob"])
            return got

    lengths, new, blocks = [70, 5, 1, 33], 4, 30
    torch.manual_seed(0)
    prompts = [torch.randint(512, (n,)) for n in lengths]
    make = dict(layers=2, hidden=1024, intermediate=4096, q_heads=heads[0], kv_heads=heads[1], head_dim=dim, vocab=512, top_k=40,
                blocks=blocks, fmt="e2m1", device=gpu)
    answers = []
    for stack in (Checked(**make), example.Stack(**make)):
        batch = example.KvBatch(blocks, 16, max_requests=4, max_blocks=6, q_heads=heads[0], kv_heads=heads[1], head_dim=dim)
        scores = []
        out, _ = example.serve(stack, prompts, new, 48, batch, scores)
        answers.append((out, scores))
        assert [len(a) for a in out] == [new] * 4 == [len(s) for s in scores] and all(x < 0 for s in scores for x in s)
        assert int(batch.state[1]) == blocks
    assert answers[0] == answers[1]
    assert max(seen) >= 48 and sum(s.numel() for s in scored) == 4 * new
    # other angles, other answers' probabilities
    other = example.Stack(**make, base=50.0)
    batch = example.KvBatch(blocks, 16, max_requests=4, max_blocks=6, q_heads=heads[0], kv_heads=heads[1], head_dim=dim)
    scores = []
    example.serve(other, prompts, new, 48, batch, scores)
    assert scores != answers[0][1]


def test_example_runs(gpu, example, capsys):  # noqa: F811
    answers, batch = example.main(["--layers", "1", "--hidden", "1024", "--intermediate", "4096", "--heads", "8,2", "--vocab", "512",
                                   "--prompts", "40,1,17", "--new", "3", "--chunk", "32", "--top-k", "40", "--format", "e2m1"])
    assert [len(a) for a in answers] == [3, 3, 3]
    assert "log probability -" in capsys.readouterr().out and int(batch.state[1]) == batch.num_blocks
    assert os.path.basename(example.__file__) == "serve_stack.py"
