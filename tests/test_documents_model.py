"""A decoder on packed documents: norms of query and key heads, attention within documents and the loss without logits, as LlamaModel runs
them together."""

from types import SimpleNamespace

import pytest
import torch

from templar_b200.model_factory import get_titan_model_args, titan_to_hf_state_dict
from templar_b200.models.llama import LlamaModel, ModelArgs, build_model
from templar_b200.models.llama_int8 import Int8Llama
from templar_b200.models.llama_tp import TPLlamaModel
from templar_b200.ops import functional as OF

EOS = 2
ARGS = dict(dim=128, n_layers=3, n_heads=2, n_kv_heads=1, vocab_size=260, intermediate_size=256, max_seq_len=256)


def packed_tokens(lens, seed=0, vocab=260):
    g = torch.Generator().manual_seed(seed)
    docs = [torch.cat((torch.randint(3, vocab, (n - 1,), generator=g), torch.tensor([EOS]))) for n in lens]
    return docs, torch.cat(docs)[None]


def model_of(seed=1, device=None, dtype=None, **options):
    m = build_model(ModelArgs(**ARGS, **options), device=device, dtype=dtype, seed=seed)
    for layer in m.layers.values():                              # weights of the norms as training leaves them
        for norm in (layer.attention.q_norm, layer.attention.k_norm):
            if norm is not None:
                with torch.no_grad():
                    norm.weight.mul_(torch.linspace(0.5, 1.5, norm.weight.numel(), device=norm.weight.device).to(norm.weight.dtype))
    return m


@pytest.mark.parametrize("qk_norm", [False, True])
def test_documents_of_a_sequence_are_scored_as_if_alone(qk_norm):
    docs, tokens = packed_tokens((7, 20, 1, 12))
    m = model_of(qk_norm=qk_norm, document_eos=EOS)
    with torch.no_grad():
        together = m(tokens)[0]
        alone = torch.cat([m(d[None])[0] for d in docs])
        across = model_of(qk_norm=qk_norm)(tokens)[0]
    torch.testing.assert_close(together, alone, rtol=1e-4, atol=1e-4)
    assert (across[7:] - together[7:]).abs().max() > 1e-2        # without the option rows look at the document before


def grads(m, tokens, labels, scale=1.0):
    m.zero_grad()
    loss = m.loss(tokens, labels, scale)
    loss.backward()
    return loss.detach(), {n: p.grad.clone() for n, p in m.named_parameters()}


@pytest.mark.parametrize("mode,option", [("none", "op"), ("full", "op"), ("selective", "2"), ("selective", "op")])
def test_fused_loss_and_checkpointing_leave_the_gradients_as_they_are(mode, option):
    _, tokens = packed_tokens((9, 31, 8))
    labels = tokens.roll(-1, 1)
    labels[0, ::5] = -100
    ref = model_of(qk_norm=True, document_eos=EOS)
    want, gw = grads(ref, tokens, labels, 0.5)
    m = model_of(qk_norm=True, document_eos=EOS, fused_loss=True)
    m.activation_checkpointing, m.ac_option = mode, option
    got, gg = grads(m, tokens, labels, 0.5)
    torch.testing.assert_close(got, want)
    assert {"layers.0.attention.q_norm.weight", "layers.2.attention.k_norm.weight"} <= gg.keys() == gw.keys()
    for n in gw:
        torch.testing.assert_close(gg[n], gw[n], rtol=1e-4, atol=1e-6, msg=n)


def test_gradients_against_differences():
    _, tokens = packed_tokens((5, 6), seed=3)
    m = model_of(qk_norm=True, document_eos=EOS, fused_loss=True)
    labels = tokens.roll(-1, 1)
    _, g = grads(m, tokens, labels)
    with torch.no_grad():
        for name, p in m.named_parameters():
            if "q_norm" not in name and "k_norm" not in name and name != "output.weight":
                continue
            d = torch.randn(p.shape, generator=torch.Generator().manual_seed(1))
            h = 1e-2 / d.norm()
            p.add_(h * d)
            up = m.loss(tokens, labels)
            p.sub_(2 * h * d)
            down = m.loss(tokens, labels)
            p.add_(h * d)
            # fp32 losses near 6 a step of 1e-2 apart: 2 * 6 * 2^-23 / 2e-2 of a step of length one, and the third derivative
            slope, want = ((up - down) / 2e-2).item(), (g[name] * d).sum().item() / d.norm().item()
            assert abs(slope - want) <= 1e-3 + 1e-2 * abs(want), (name, slope, want)


def test_names_sizes_and_refusals():
    assert not any("q_norm" in n for n in LlamaModel(ModelArgs(**ARGS)).state_dict())
    a = ModelArgs(**ARGS, qk_norm=True)
    m = LlamaModel(a)
    assert sum(p.numel() for p in m.parameters()) == a.num_params()
    assert m.materialize_param("layers.1.attention.k_norm.weight", "cpu").eq(1).all()
    for option in (dict(qk_norm=True), dict(document_eos=EOS), dict(fused_loss=True)):
        with pytest.raises(ValueError, match="TPLlamaModel"):
            TPLlamaModel(ModelArgs(**ARGS, **option), 0, 1)
    with pytest.raises(ValueError, match="qk_norm"):
        titan_to_hf_state_dict(m.state_dict(), a)
    f = model_of(fused_loss=True)

    class Shards:
        def accumulate(self, *a):
            pass

    f.output.weight.main_grad = Shards()
    with pytest.raises(ValueError, match="fused_loss"):
        f.loss(*(packed_tokens((4,))[1],) * 2)


def test_options_from_hparams():
    hp = SimpleNamespace(model_size="tiny", sequence_length=64, tokenizer=SimpleNamespace(vocab_size=300, eos_token_id=7),
                         model_config=SimpleNamespace(hidden_size=64, num_hidden_layers=1, num_attention_heads=2, intermediate_size=128),
                         torchtitan=SimpleNamespace())
    a = get_titan_model_args(hp)
    assert (a.qk_norm, a.document_eos, a.fused_loss) == (False, -1, False)
    hp.torchtitan = SimpleNamespace(qk_norm=True, document_attention=True, fused_loss=True)
    a = get_titan_model_args(hp)
    assert (a.qk_norm, a.document_eos, a.fused_loss) == (True, 7, True)
    hp.model_size = "8B"
    assert get_titan_model_args(hp).document_eos == 7 and get_titan_model_args(hp).qk_norm
    hp.tokenizer.eos_token_id = None
    with pytest.raises(ValueError, match="document_attention"):
        get_titan_model_args(hp)


def test_int8_model_scores_documents():
    docs, tokens = packed_tokens((12, 30))
    m = model_of(qk_norm=True, document_eos=EOS, fused_loss=True)
    q = Int8Llama(m)
    with torch.no_grad():
        torch.testing.assert_close(q(tokens)[0, 12:], q(docs[1][None])[0], rtol=1e-3, atol=1e-3)
        full = m(tokens)
        assert (q(tokens) - full).norm() < 0.05 * full.norm()
        labels = tokens.roll(-1, 1)
        torch.testing.assert_close(q.loss(tokens, labels), OF.cross_entropy(q(tokens), labels, 1.0, -100), rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("n_heads,mode", [(2, "none"), (1, "none"), (2, "selective"), (2, "full"), (2, "int8")])
def test_training_step_on_packed_documents(n_heads, mode):
    """Heads of 64 and 128, gradients into buffers: against the same model in fp32, whose operators are the formulas in PyTorch."""
    from templar_b200.parallel.flat import FlatParamStore

    args = dict(ARGS, n_heads=n_heads, dim=128)
    args["n_kv_heads"] = 1
    opts = dict(qk_norm=True, document_eos=EOS, fused_loss=True)
    _, tokens = packed_tokens((60, 130, 7, 59), seed=5)
    tokens = torch.cat((tokens, tokens.flip(1)), 0).cuda()
    labels = tokens.roll(-1, 1)
    labels[:, -1] = -100
    m = build_model(ModelArgs(**args, **opts), device="cuda", dtype=torch.bfloat16, seed=4)
    ref = build_model(ModelArgs(**args, **opts), device="cuda", dtype=torch.float32, seed=4)
    ref.load_state_dict({k: v.float() if v.is_floating_point() else v for k, v in m.state_dict().items()})
    want, gw = grads(ref, tokens, labels)
    store = FlatParamStore(m, device=torch.device("cuda"))
    store.zero_grad()
    m.activation_checkpointing, m.ac_option = mode, "op"
    loss = m.loss(tokens, labels)
    loss.backward()
    assert int(OF.status_word("cuda").item()) == 0
    # bf16 activations through three blocks: 20 roundings of 2^-9 on average each, added in squares
    torch.testing.assert_close(loss, want, rtol=1e-2, atol=1e-2)
    for name, p in m.named_parameters():
        g = p.main_grad.float().view_as(gw[name])
        off = (g - gw[name]).norm() / gw[name].norm()
        assert off < (0.06 if mode == "int8" else 0.04), (name, off.item())
    with torch.no_grad():
        alone = m.loss(tokens, labels)
    torch.testing.assert_close(alone, loss.detach(), rtol=1e-3, atol=1e-3)


def window(device, dtype, shard_params, fused_loss, **extra):
    """One window of the engine on packed documents: micro-steps, optimizer step, compression, outer step; the loss before and after."""
    from templar_b200.parallel.window_engine import EngineConfig, WindowEngine

    m = model_of(seed=3, device=device, dtype=dtype, qk_norm=True, document_eos=EOS, fused_loss=fused_loss)
    eng = WindowEngine(m, EngineConfig(topk=8, inner_lr=1e-3, shard_params=shard_params, max_peers=1, **extra), device=device)
    _, tokens = packed_tokens((40, 25, 63), seed=9)
    tokens = tokens.to(device)
    labels = tokens.roll(-1, 1)
    eng.snapshot()
    losses = []
    for _ in range(3):
        eng.zero_grad()
        losses.append(float(eng.micro_step(tokens, labels)))
        eng.optimizer_step(lr=1e-3)
    eng.compress()
    return losses, eng


def same_window(device, dtype, rel):
    """With parameters whole and the loss without logits, and with parameters in shards and the loss from the logits."""
    losses, eng = window(device, dtype, False, fused_loss=True)
    assert "layers.1.attention.q_norm.weight" in [s.name for s in eng.layout.specs]
    assert torch.isfinite(torch.tensor(losses)).all()
    assert losses == pytest.approx(window(device, dtype, True, fused_loss=False)[0], rel=rel)


def test_window_of_packed_documents():
    same_window("cpu", torch.float32, 1e-4)


@pytest.mark.gpu
def test_window_of_packed_documents_gpu():
    same_window("cuda", torch.bfloat16, 1e-2)                    # logits rounded to bf16 on one side
    assert int(OF.status_word("cuda").item()) == 0
