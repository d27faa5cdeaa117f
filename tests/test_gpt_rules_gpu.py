"""GPTs whose blocks have a window with first positions that stay visible, a bias by distance bucket and dropout: loss, every gradient, generation,
against the same model in 64 bits (torch on the CPU, masks from tests/attention_rule.py).

Gradients are held to the training path's bar of 1e-4 of a tensor's largest value."""
import numpy as np
import pytest

from gradcraft_b200 import synth
from tests import attention_rule as R
from tests.helpers import assert_grads_close

pytestmark = pytest.mark.gpu
V, T, C, H, L, F, B = 97, 70, 96, 3, 2, 112, 3


class Reference:
    def __init__(self, arch, weights, opt, p=0.0):
        import torch

        self.torch, self.arch, self.opt, self.p = torch, arch, opt, float(np.float32(p))
        self.w = {k: torch.tensor(v, dtype=torch.float64, requires_grad=True) for k, v in weights.items()}
        self.counter = 0
        self.starts = R.bucket_starts(opt["rel_buckets"], opt["rel_reach"]) if opt.get("rel_buckets") else None

    def norm(self, x, name):
        w = self.w
        if self.arch == "lngelu":
            return self.torch.nn.functional.layer_norm(x, (C,), w[name + ".gamma"], w[name + ".beta"], 1e-5)
        return x * w[name + ".gamma"] / (x.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt()

    def linear(self, x, name):
        return x @ self.w[name + ".W"] + self.w[name + ".b"]

    def drop(self, x, training):
        if not training or self.p == 0:
            return x
        keep = R.kept(x.numel(), self.p, self.opt["dropout_seed"], self.counter)
        self.counter += (x.numel() + 3) // 4
        return x * self.torch.from_numpy(keep.reshape(tuple(x.shape))) / (1.0 - self.p)

    def forward(self, tokens, training=False):
        torch, w, opt = self.torch, self.w, self.opt
        n, S = tokens.shape
        x = w["token_embed.embeds"][torch.from_numpy(tokens)] + w["pos_embed.pos_embeds"][:S]
        i = np.arange(S)
        seen = torch.from_numpy(R.visible(i[:, None], i[None, :], opt.get("window", 0), opt.get("sinks", 0)))
        for l in range(L):
            b = "block_%d." % l
            a = self.norm(x, b + "norm1")
            q, k, v = (self.linear(a, b + "attn.%s_proj" % c).view(n, S, H, C // H).transpose(1, 2) for c in "qkv")
            s = q @ k.transpose(2, 3) / (C // H) ** 0.5
            if self.starts is not None:
                bucket = np.maximum(np.searchsorted(self.starts, np.maximum(i[:, None] - i[None, :], 0), side="right") - 1, 0)
                s = s + w[b + "attn.rel_bias"][:, torch.from_numpy(bucket)]
            o = torch.softmax(s.masked_fill(~seen, -np.inf), -1) @ v
            x = x + self.drop(self.linear(o.transpose(1, 2).reshape(n, S, C), b + "attn.out_proj"), training)
            m = self.norm(x, b + "norm2")
            if self.arch == "lngelu":
                m = self.linear(torch.nn.functional.gelu(self.linear(m, b + "mlp.fc1"), approximate="tanh"), b + "mlp.fc2")
            else:
                m = self.linear(torch.nn.functional.silu(self.linear(m, b + "mlp.w1")) * self.linear(m, b + "mlp.w2"), b + "mlp.w3")
            x = x + self.drop(m, training)
        return self.norm(x, "final_norm") @ w["token_embed.embeds"].T

    def loss_and_grads(self, batches):
        torch, total = self.torch, 0.0
        for x, y in batches:
            logp = torch.log_softmax(self.forward(x, training=True).flatten(0, 1), -1)
            mine = logp[torch.arange(y.size), torch.from_numpy(y.reshape(-1))]
            (-mine.mean() / len(batches)).backward()  # the framework's loss adds 1e-5 inside the logarithm, its gradient leaves that out
            total += float(-(mine.detach().exp() + 1e-5).log().mean()) / len(batches)
        return total, {k: v.grad.numpy().astype(np.float64) for k, v in self.w.items()}

    def greedy(self, start, context, most):
        toks = list(start)
        while len(toks) < most:
            row = self.forward(np.array(toks[-context:])[None])[0, -1].detach().numpy()
            top = np.sort(row)[-2:]
            assert top[1] - top[0] > 1e-4 * np.abs(row).max()  # an arg-max that no rounding turns
            toks.append(int(row.argmax()))
        return toks


def make(arch, opt, seed=0):
    from gradcraft_b200.trainer import Trainer

    w = synth.gpt_weights(arch, V, T, C, H, L, F, seed=seed, perturb=True, std=0.1)
    if opt.get("rel_buckets"):
        for l in range(L):
            w["block_%d.attn.rel_bias" % l] = synth.normal(seed, "rel%d" % l, (H, opt["rel_buckets"]), 0.5)
    tr = Trainer(arch, V, T, C, H, L, F, options=opt)
    tr.load(w)
    return tr, w


OPTIONS = [dict(window=16, sinks=2), dict(rel_buckets=16, rel_reach=40), dict(window=24, sinks=3, rel_buckets=8, rel_reach=32), dict(dropout=0.2, dropout_seed=77), dict(window=9, sinks=1, rel_buckets=32, rel_reach=64, dropout=0.1, dropout_seed=5)]


@pytest.mark.parametrize("arch", ["lngelu", "rmsswiglu"])
@pytest.mark.parametrize("opt", OPTIONS, ids=lambda o: "-".join("%s%s" % kv for kv in o.items()))
def test_training_step(arch, opt):
    tr, w = make(arch, opt)
    ref = Reference(arch, w, opt, opt.get("dropout", 0.0))
    batches = [tuple(np.ascontiguousarray(x) for x in b) for b in synth.token_batches(3, 2, B, T, V)]
    tr.zero_grad()
    loss = sum(tr.forward_backward(x, y, accum=2) for x, y in batches)  # the second micro-batch adds to every gradient and draws masks of its own
    want, grads = ref.loss_and_grads(batches)
    assert abs(loss - want) < 1e-5 * want
    got = {k: v.reshape(grads[k].shape) for k, v in tr.get("grad").items()}
    assert_grads_close(got, grads)
    assert tr.dropout_counter() == ref.counter
    tr.set_dropout_counter(0)  # the same masks again
    tr.zero_grad()
    again = sum(tr.forward_backward(x, y, accum=2) for x, y in batches)
    assert again == loss and all((tr.get("grad")[k] == got[k].reshape(-1)).all() for k in got)
    tr.optimizer_step()
    tr.close()


@pytest.mark.parametrize("arch", ["lngelu", "rmsswiglu"])
@pytest.mark.parametrize("opt", OPTIONS[:3] + OPTIONS[4:], ids=lambda o: "-".join("%s%s" % kv for kv in o.items()))
def test_generation(arch, opt):
    """Within the context window and past it; nothing is dropped, and training goes on where it was."""
    tr, w = make(arch, opt, seed=2)
    ref = Reference(arch, w, opt)
    start = [5, 17, 3, 60, 8, 2, 41]
    for context, most, prompt in ((70, 40, start), (20, 33, start), (70, 12, start[:2])):
        before = tr.dropout_counter()
        got = tr.generate(prompt, most, num_sequences=2, context_length=context)
        assert got.tolist() == [ref.greedy(prompt, context, most)] * 2
        assert tr.dropout_counter() == before
    one = tr.generate(start, 30, num_sequences=3, temperature=0.8, top_k=1)  # sampled from the best token alone: the same text
    assert one.tolist() == [ref.greedy(start, 70, 30)] * 3
    tr.close()


def test_a_model_without_options_is_what_it_was():
    from gradcraft_b200.trainer import Trainer

    w = synth.gpt_weights("lngelu", V, T, C, H, L, F, seed=1, perturb=True)
    x, y = (np.ascontiguousarray(a) for a in synth.token_batches(3, 1, B, T, V)[0])
    got = []
    for options in (None, dict(window=0, sinks=4), dict(dropout=0.0)):
        tr = Trainer("lngelu", V, T, C, H, L, F, options=options)
        tr.load(w)
        tr.zero_grad()
        got.append((tr.forward_backward(x, y), tr.get("grad"), tr.generate([1, 2, 3], 20).tolist()))
        tr.close()
    for loss, grads, text in got[1:]:
        assert loss == got[0][0] and text == got[0][2] and all((grads[k] == got[0][1][k]).all() for k in grads)


def test_refusals():
    from gradcraft_b200.trainer import Trainer, TrainerError

    for bad in (dict(window=-1), dict(window=4, sinks=65), dict(rel_buckets=65), dict(rel_buckets=8, rel_reach=0), dict(dropout=1.5), dict(dropout=-0.1)):
        with pytest.raises(TrainerError):
            Trainer("lngelu", V, T, C, H, L, F, options=bad)
    with pytest.raises(TrainerError):  # a head of 160 columns
        Trainer("lngelu", V, T, 160, 1, L, F, options=dict(window=4))
