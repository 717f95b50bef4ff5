"""The optimizer step and the 8-bit product where the framework calls them: Trainer and its checkpoints, the verification test, and
a run of them together — a network trained with 8-bit moments, its embeddings scored and its speakers named in 8-bit integers."""
import numpy as np
import pytest
import torch

from titanet_amd import LOSSES, TitaNet, metrics
from titanet_amd.int8 import quantize_rows
from titanet_amd.optim import AdamW, grad_norm
from titanet_amd.train import load_checkpoint, save_checkpoint
from titanet_amd.trainer import Trainer

pytestmark = pytest.mark.gpu


def _model(loss="ce", classes=11, seed=3, dropout=0.0):
    torch.manual_seed(seed)
    return TitaNet(n_mels=80, n_mega_blocks=1, n_sub_blocks=3, encoder_hidden_size=256, encoder_output_size=1536, embedding_size=192,
                   mega_block_kernel_size=3, loss_function=LOSSES[loss](192, classes, device="cuda"), dropout=dropout, device="cuda").train()


def _batch(n=12, classes=11, frames=64, seed=4):
    g = torch.Generator().manual_seed(seed)
    y = torch.randint(0, classes, (n,), generator=g)
    voices = torch.randn(classes, 80, 1, generator=g)
    return (voices[y] + 0.5 * torch.randn(n, 80, frames, generator=g)).cuda(), y.cuda()


@pytest.mark.parametrize("bits", [32, 8])
def test_trainer_steps_like_the_optimizer_on_the_flat_buffer(bits):
    a, b = _model(), _model()
    trainer = Trainer(a, lr=2e-3, weight_decay=0.05, optimizer="adamw", state_bits=bits, max_grad_norm=0.5)
    b._native_forward(*_batch())                     # (makes the gradient buffer)
    flat = b.flat_parameters().detach()
    flat.copy_(a.flat_parameters())
    b._flat["bnbuf"].copy_(a._flat["bnbuf"])
    opt = AdamW([flat], lr=2e-3, weight_decay=0.05, state_bits=bits, max_grad_norm=0.5)
    for k in range(3):
        x, y = _batch(seed=10 + k)
        trainer.step(x, y)
        flat.grad = a.flat_gradients().clone()       # the gradient the trainer stepped with
        opt.step()
        assert torch.equal(flat, a.flat_parameters()) and torch.equal(trainer.last_grad_norm, opt.last_grad_norm), k
    assert all(torch.equal(m, n) for m, n in zip(trainer.adamw.moments(), opt.moments()))


@pytest.mark.parametrize("bits", [32, 8])
def test_trainer_graph_and_eager_agree(bits):
    kw = dict(lr=1e-3, weight_decay=0.05, optimizer="adamw", state_bits=bits, max_grad_norm=1.0)
    a, b = _model(), _model()
    eager, graph = Trainer(a, **kw), Trainer(b, use_graph=True, graph_warmup=1, **kw)
    x, y = _batch()
    for k in range(6):
        eager.lr = graph.lr = 1e-3 / (k + 1)
        la, lb = float(eager.step(x, y)[2]), float(graph.step(x, y)[2])
        torch.cuda.synchronize()
        # the backward pass sums by atomics in places: the two runs agree to float32 rounding, not to the bit; a moment's code may turn with it
        assert abs(la - lb) <= 1e-3 * abs(la) + 1e-4, k
    assert graph._graphs and next(iter(graph._graphs.values()))["graph"] is not None
    assert float(eager.optimizer_state_dict()["state"][0]["step"]) == float(graph.optimizer_state_dict()["state"][0]["step"]) == 6


@pytest.mark.parametrize("bits", [32, 8])
def test_checkpoints_resume_where_they_stopped(tmp_path, bits):
    kw = dict(lr=1e-3, weight_decay=0.05, optimizer="adamw", state_bits=bits, max_grad_norm=1.0)
    a = _model()
    ta = Trainer(a, **kw)
    for k in range(3):
        ta.step(*_batch(seed=k))
    save_checkpoint(a, ta, 3, str(tmp_path / "c.pth"))
    b = _model(seed=9)
    tb = Trainer(b, **kw)
    assert load_checkpoint(b, tb, str(tmp_path / "c.pth"))[0] == 3
    assert torch.equal(a.flat_parameters(), b.flat_parameters()) and tb.step_count == 3
    assert all(torch.equal(m, n) for m, n in zip(ta.adamw.moments(), tb.adamw.moments()))
    sd = ta.optimizer_state_dict()
    ref = torch.optim.AdamW(a.parameters())
    ref.load_state_dict(sd)                          # torch's own takes it
    assert sd["param_groups"][0]["decoupled_weight_decay"] and len(sd["state"]) == len(list(a.parameters()))


def test_trainer_refusals():
    m = _model()
    for kw in (dict(optimizer="sgd"), dict(state_bits=8), dict(max_grad_norm=1.0), dict(optimizer="adamw", state_bits=4)):
        with pytest.raises(ValueError):
            Trainer(m, **kw)
    assert Trainer(m).last_grad_norm is None


def test_scores_of_pairs_in_8_bits():
    g = torch.Generator().manual_seed(6)
    e, gallery = torch.randn(70, 192, generator=g).cuda(), torch.randn(33, 192, generator=g).cuda()
    for args in ((e,), (e, gallery)):
        full, eight = metrics.cosine_scores(*args), metrics.cosine_scores(*args, bits=8)
        # each of 192 factors is off by at most half a step of (row maximum / 127): below 4 sigma / 127 / 2 of a unit row's entries
        assert eight.shape == full.shape and float((full - eight).abs().max()) < 0.02
    unit = gallery / gallery.norm(dim=1, keepdim=True)
    assert torch.equal(metrics.cosine_scores(e, quantize_rows(unit), bits=8), metrics.cosine_scores(e, gallery, bits=8))
    with pytest.raises(ValueError):
        metrics.cosine_scores(e, bits=16)


@pytest.mark.parametrize("loss", ["ce", "arc"])
def test_train_with_8_bit_moments_then_answer_in_8_bits(loss):
    model = _model(loss)
    trainer = Trainer(model, lr=1e-3, weight_decay=0.01, optimizer="adamw", state_bits=8, max_grad_norm=5.0)
    for k in range(30):
        out = trainer.step(*_batch(24, seed=k))
        assert bool(torch.isfinite(out[2]))
    model.eval()
    x, y = _batch(40, seed=99)
    with torch.no_grad():
        emb = model(x)
        head = model.loss_function.int8_head()
        scores = head(emb)
        w = model.loss_function.fc.weight
        want = emb @ (w if loss == "ce" else torch.nn.functional.normalize(w, dim=1)).t() + (model.loss_function.fc.bias if loss == "ce" else 0.0)
    assert scores.shape == (40, 11) and float((scores - want).norm()) < 0.02 * float(want.norm())
    specs, ids = list(x.cpu()), y.tolist()
    (m32, s32, labels), (m8, s8, _) = (metrics.verification_test(model, specs, ids, score_bits=b) for b in (32, 8))
    assert s32.shape == s8.shape == (1600,) and np.abs(s32 - s8).max() < 0.02 and set(m8) == set(m32)
    assert model.training is False


def test_trainer_graphs_of_several_lengths_report_their_own_norm():
    model = _model()
    trainer = Trainer(model, lr=1e-3, optimizer="adamw", max_grad_norm=1.0, use_graph=True, graph_warmup=1)
    for k, frames in enumerate((64, 96, 64, 96, 64, 64, 96, 96, 64)):
        trainer.step(*_batch(frames=frames, seed=20 + k))
        want = float(grad_norm(model.flat_gradients()))
        assert abs(float(trainer.last_grad_norm) - want) <= 2 * 2.0 ** -24 * want, (k, frames)
    assert all(st["graph"] is not None for st in trainer._graphs.values())
