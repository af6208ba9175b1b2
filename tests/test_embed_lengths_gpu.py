"""A padded batch of utterances of different lengths embeds as the utterances alone (engine.embed(lengths=)): packed
attention, the bias by bucket borders and the mean over each utterance's own frames, in the encoder; and
clip_grad_norm_ in a training loop's place."""
import pytest
import torch

from nrse_amd import arch as A, params as PR

pytestmark = pytest.mark.gpu
LENS = [16000, 9000, 12345, 400, 16000, 7777]


def engine(dtype, weight_split=False):
    from nrse_amd.engine import ByolEngine
    arch = A.TINY.deterministic()
    flat = PR.init_byol_flat(PR.byol_layout(arch, 256, 512), 1234)
    return ByolEngine(arch, 256, 512, device="cuda:0", compute_dtype=dtype, init_flat=flat, weight_split=weight_split)


def batch(fill):
    g = torch.Generator().manual_seed(3)
    wav = torch.full((len(LENS), 16000), fill)
    for i, n in enumerate(LENS):
        wav[i, :n] = torch.randn(n, generator=g)
    return wav.cuda()


def alone(eng, wav):
    return torch.cat([eng.embed(wav[i:i + 1, :n].contiguous()) for i, n in enumerate(LENS)])


def rel(a, b):
    return ((a.double() - b.double()).norm(dim=1) / b.double().norm(dim=1)).max().item()


@pytest.mark.parametrize("fill", [0.0, 1e4, float("nan")])
def test_padded_batch_embeds_as_its_utterances_f32(nrse_device, fill):
    eng = engine(torch.float32)
    wav = batch(fill)
    # f32 products and sums in another order, through two layers: the bound of the model's own parity test
    assert rel(eng.embed(wav, lengths=LENS), alone(eng, wav)) < 1e-4
    dev = torch.tensor(LENS, device="cuda")
    assert torch.equal(eng.embed(wav, lengths=dev), eng.embed(wav, lengths=torch.tensor(LENS)))


@pytest.mark.parametrize("split", [False, True], ids=["bf16", "bf16sw"])
def test_padded_batch_embeds_as_its_utterances_bf16(nrse_device, split):
    """Against the f32 embedding: no further from it than the utterances alone are, within the two forms' roundings
    (each value's rounding falls out independently: a factor of 1.5 on a norm of 256 of them)."""
    want = alone(engine(torch.float32), batch(0.0))
    eng = engine(torch.bfloat16, weight_split=split)
    wav = batch(float("nan"))
    one, many = alone(eng, wav), eng.embed(wav, lengths=LENS)
    assert torch.isfinite(many).all()
    assert rel(many, want) <= 1.5 * rel(one, want) + 1e-6


def test_whole_lengths_and_none(nrse_device):
    eng = engine(torch.float32)
    wav = batch(0.0)
    whole = eng.embed(wav, lengths=[16000] * len(LENS))
    assert rel(whole, eng.embed(wav)) < 1e-4
    emb = eng.embed(wav, lengths=[16000, 0, 399, 400, 16000, 1])     # under one frame: zeros
    assert (emb[[1, 2, 5]] == 0).all() and rel(emb[[0, 4]], whole[[0, 4]]) < 1e-4
    assert (emb[3] != 0).any()


def test_lengths_refusals(nrse_device):
    from nrse_amd._lib import NrseError
    eng = engine(torch.float32)
    wav = batch(0.0)
    for bad in ([16000] * 5, [16001] * 6, [-1] * 6, [1.5] * 6, torch.zeros(6, 1, dtype=torch.int64), [True] * 6):
        with pytest.raises(NrseError, match="lengths"):
            eng.embed(wav, lengths=bad)
    fl = eng.frame_lengths(LENS, wav)
    assert fl.tolist() == [max(0, eng.arch.frames(n)) for n in LENS]
    with pytest.raises(NrseError, match="eval-mode"):
        eng.encoder_forward(eng.weights("online"), wav, train=True, flens=fl)


def test_encoder_module(nrse_device):
    from nrse_amd.model import WavLMEncoder
    eng = engine(torch.float32)
    enc = WavLMEncoder(engine=eng)
    wav = batch(0.0)
    assert torch.equal(enc(wav.unsqueeze(1), lengths=LENS), eng.embed(wav, lengths=LENS))
    assert torch.equal(enc(wav), eng.embed(wav))


@pytest.mark.parametrize("C", [256, 512, 768, 1024])
def test_ln_mean_lens(nrse_device, C):
    from nrse_amd import kernels as K
    B, T = 5, 70
    g = torch.Generator(device="cuda").manual_seed(C)
    h = torch.randn(B, T, C, generator=g, device="cuda") * 3 + 1
    gamma, beta = torch.randn(C, generator=g, device="cuda"), torch.randn(C, generator=g, device="cuda")
    lens = torch.tensor([70, 1, 0, 33, 32], dtype=torch.int32, device="cuda")
    for b, n in enumerate(lens.tolist()):
        h[b, n:] = float("nan")
    emb = torch.full((B, C), float("nan"), device="cuda")
    K.ln_mean_lens(h, gamma, beta, lens, emb, 1e-5)
    x = h.double()
    y = (x - x.mean(-1, keepdim=True)) / (x.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt() * gamma.double() + beta.double()
    for b, n in enumerate(lens.tolist()):
        want = y[b, :n].mean(0) if n else torch.zeros(C, dtype=torch.float64, device="cuda")
        # f32: (C + T) terms of size about |gamma| 4 + |beta|
        err = (C + T) * 2.0 ** -24 * (4 * gamma.double().abs() + beta.double().abs())
        assert ((emb[b].double() - want).abs() <= err).all(), (b, n)


# ------------------------------------------------------------------------------------------------ clip_grad_norm_
def test_clip_grad_norm_in_a_loop(nrse_device):
    """As torch.nn.utils.clip_grad_norm_, on a small network's parameters after a backward."""
    from nrse_amd.train import clip_grad_norm_
    torch.manual_seed(5)
    net = torch.nn.Sequential(torch.nn.Linear(64, 96), torch.nn.LayerNorm(96), torch.nn.Linear(96, 7)).cuda()
    unused = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    params = [*net.parameters(), unused]
    (net(torch.randn(32, 64, device="cuda")) ** 2).sum().backward()
    params[0].grad = params[0].grad.t().contiguous().t()      # dense in another order
    before = [p.grad.clone() for p in net.parameters()]
    want = torch.nn.utils.clip_grad_norm_(params, 0.5)
    ref = [p.grad.clone() for p in net.parameters()]
    for p, g in zip(net.parameters(), before):
        p.grad.copy_(g)
    norm = clip_grad_norm_(iter(params), 0.5)
    assert abs(float(norm) / float(want) - 1) < 1e-6
    for p, r in zip(net.parameters(), ref):
        assert float((p.grad - r).norm() / r.norm()) < 1e-6
    assert clip_grad_norm_([unused], 1.0) == 0.0
    params[0].grad[0, 0] = float("inf")
    with pytest.raises(RuntimeError, match="not clipped"):
        clip_grad_norm_(net.parameters(), 1.0, error_if_nonfinite=True)
    with pytest.raises(ValueError):
        clip_grad_norm_(net.parameters(), 1.0, norm_type=1.0)


def test_clip_grad_norm_of_the_model(nrse_device):
    """The drop-in model's flat gradient, in place of torch's call of the reference loop."""
    from nrse_amd.model import BYOLSpeechModel, byol_loss
    from nrse_amd.train import clip_grad_norm_
    cfg = {"model": {"name": "nrse/wavlm-tiny", "ema_decay": 0.99, "projection_dim": 256, "prediction_dim": 512}}
    model = BYOLSpeechModel(cfg, compute_dtype=torch.float32, arch=A.TINY.deterministic())
    model.train()
    wav = batch(0.0)
    p, z = model(wav, wav + 0.1)
    byol_loss(p, z).backward()
    want = float(model.online_flat.grad.double().norm())
    norm = clip_grad_norm_(model.parameters(), 0.5 * want)
    assert abs(float(norm) / want - 1) < 1e-6
    assert abs(float(model.online_flat.grad.double().norm()) / (0.5 * want) - 1) < 1e-5
