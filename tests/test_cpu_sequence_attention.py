"""The attention block over un-pooled sequences on the CPU path: alone, and in a model whose sequences come from a table."""
import pytest
import torch

import tensornet_b200 as tn
from tensornet_b200.data import Ragged


@pytest.fixture(autouse=True)
def _cpu_runtime():
    tn.core.shutdown()
    tn.core.config.force_cpu = True
    tn.core.init()
    yield
    tn.core.shutdown()


def _reference(layer, x, lengths, target=None):
    """The block in fp32 without this package's operators, sequence by sequence."""
    D, H, G, dim = layer.head_dim, layer.heads, layer.kv_heads, layer.dim

    def norm(t):
        return torch.nn.functional.layer_norm(t, (dim,), layer.norm.gamma, layer.norm.beta, layer.epsilon)

    def project(t, w, n):
        return t @ w[:, :n].t() + w[:, n]

    outs = []
    for b in range(x.shape[0]):
        n = int(lengths[b])
        seq = norm(x[b, :n])
        asks = x[b] if target is None else target[b].view(-1, dim)
        q = project(norm(asks), layer.query, dim).view(-1, H, D).transpose(0, 1)
        kv = project(seq, layer.key_value, dim)
        k, v = [kv[:, i * G * D:(i + 1) * G * D].view(n, G, D).transpose(0, 1).repeat_interleave(H // G, 0) for i in range(2)]
        m = n if target is None else asks.shape[0]
        s = q[:, :m] @ k.transpose(1, 2) * D ** -0.5
        if layer.cap:
            s = layer.cap * torch.tanh(s / layer.cap)
        place = torch.arange(m).view(-1, 1) + n - m
        if layer.slopes is not None:
            s = s - layer.slopes.view(-1, 1, 1) * (place - torch.arange(n)).abs()
        if layer.causal and target is None:
            s = s.masked_fill(torch.arange(n) > place, -1e30)
        o = (torch.softmax(s, -1) @ v).transpose(0, 1).reshape(m, H * D) if n else torch.zeros(m, H * D)
        y = project(o, layer.output, H * D)
        out = asks.clone()
        out[:m] = asks[:m] + y
        outs.append(out)
    return torch.stack(outs).view(x.shape if target is None else target.shape)


@pytest.mark.parametrize("kw", [dict(heads=2), dict(heads=4, kv_heads=2, head_dim=8, causal=True, distance_bias=True, cap=5.0)])
@pytest.mark.parametrize("shape", [None, (3, 16), (3, 2, 16)])
def test_block(kw, shape):
    torch.manual_seed(0)
    layer = tn.layers.SequenceAttention(16, **kw)
    with torch.no_grad():
        for w, n in ((layer.query, 16), (layer.key_value, 16), (layer.output, layer.heads * layer.head_dim)):
            w[:, n] = torch.randn(w.shape[0]) * 0.1          # biases
    x, lengths = torch.randn(3, 9, 16, requires_grad=True), torch.tensor([9, 0, 4])
    target = None if shape is None else torch.randn(shape, requires_grad=True)
    y = layer(x, lengths, target)
    ref = _reference(layer, x, lengths, target)
    assert y.shape == ref.shape and torch.allclose(y, ref, atol=0.06)          # operands in bf16
    if target is None:
        assert torch.equal(y[2, 4:], x[2, 4:]) and torch.equal(y[1], x[1])
    wrt = [x, layer.query, layer.key_value, layer.output, layer.norm.gamma] + ([] if target is None else [target])
    g = torch.randn_like(y)
    for a, b in zip(torch.autograd.grad(y, wrt, g), torch.autograd.grad(ref, wrt, g)):
        assert float((a - b).norm()) <= 0.03 * float(b.norm()) + 1e-4
    again = tn.layers.SequenceAttention(**layer.get_config())
    assert again.get_config() == layer.get_config()


def test_refusals():
    with pytest.raises(ValueError, match="multiple of 8"):
        tn.layers.SequenceAttention(20, heads=2)
    with pytest.raises(ValueError, match="no multiple"):
        tn.layers.SequenceAttention(48, heads=3, kv_heads=2)
    layer = tn.layers.SequenceAttention(16, heads=2)
    with pytest.raises(ValueError, match="sequences"):
        layer(torch.zeros(2, 16))
    with pytest.raises(ValueError, match="targets"):
        layer(torch.zeros(2, 5, 16), target=torch.zeros(3, 16))
    with pytest.raises(ValueError, match="prefix"):
        layer(torch.zeros(2, 5, 16), prefix=torch.zeros(2, dtype=torch.int32))


def test_nothing_there():
    layer = tn.layers.SequenceAttention(16, heads=2)
    assert layer(torch.zeros(0, 5, 16)).shape == (0, 5, 16)
    t = torch.randn(2, 16)
    assert layer(torch.zeros(2, 0, 16), target=t).shape == (2, 16)


class _Behaviour(tn.model.Model):
    """A candidate item against a user's history."""

    def __init__(self):
        super().__init__()
        cc, ec = tn.feature_column, tn.feature_column.embedding_column
        hist = ec(cc.sequence_category_column(cc.category_column("hist", 512), 6), 16)
        item = ec(cc.category_column("item", 512), 16)
        opt = tn.core.Adam(learning_rate=0.01, initial_scale=0.3)
        self.seq = tn.layers.SequenceEmbeddingFeatures([hist], opt, name="hist")
        self.item = tn.layers.EmbeddingFeatures([item], opt, name="item", is_concat=True)
        self.encode = tn.layers.SequenceAttention(16, heads=2, causal=True, distance_bias=True)
        self.look = tn.layers.SequenceAttention(16, heads=2)
        self.mlp, self.head = tn.layers.MLP(32, [16]), tn.layers.DenseHead(16)

    def forward(self, features):
        x, lengths = self.seq({"hist": features["hist"]}, training=self.training)
        item = self.item({"item": features["item"]}, training=self.training)
        x = self.encode(x, lengths)
        from tensornet_b200.ops import functional as F

        return self.head(self.mlp(F.concat_cast([self.look(x, lengths, item), item])))


def behaviour_batch(B=32, seed=0):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, 7, (B,), generator=g)
    off = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)])
    f = {"hist": Ragged(torch.randint(1, 40, (int(off[-1]),), generator=g), off), "item": torch.randint(1, 40, (B,), generator=g)}
    return f, (f["item"] % 2).float()


def test_in_a_model():
    torch.manual_seed(0)
    m = _Behaviour()
    m.compile(optimizer=tn.optimizer.Optimizer(tn.core.Adam(learning_rate=1e-3)))
    f, y = behaviour_batch()
    before = [p.detach().clone() for p in (m.encode.query, m.look.key_value, m.look.norm.gamma)]
    losses = [float(m.train_on_batch(f, y)) for _ in range(3)]
    assert all(l == l for l in losses)
    assert all(not torch.equal(a, b) for a, b in zip(before, (m.encode.query, m.look.key_value, m.look.norm.gamma)))
    assert torch.as_tensor(m.predict_on_batch(f)).reshape(-1).shape == (32,)
