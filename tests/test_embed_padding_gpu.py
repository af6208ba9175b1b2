"""What the padding of a padded batch holds does not count anywhere else either."""
import pytest
import torch

from test_embed_lengths_gpu import LENS, alone, batch, engine, rel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fill", [float("nan"), float("inf"), 1e30, -1e4])
def test_padding_in_the_split_weight_mode(nrse_device, fill):
    """No saturation is counted for it (the counters make the exponents move), and the embedding is that of any other
    padding, bit for bit."""
    eng = engine(torch.bfloat16, weight_split=True)
    eng.sat_buf.zero_()
    want = eng.embed(batch(0.0), lengths=LENS)
    assert int(eng.sat_buf.abs().sum()) == 0
    got = eng.embed(batch(fill), lengths=LENS)
    assert int(eng.sat_buf.abs().sum()) == 0
    assert torch.equal(got, want)


def test_device_lengths_are_clamped(nrse_device):
    """Lengths on the device are not read back to be checked: they are taken as clamped to [0, L]."""
    eng = engine(torch.float32)
    wav = batch(0.0)
    over = torch.tensor([16000, 99999, -5, 400, 2 ** 40, 7777], device="cuda")
    assert torch.equal(eng.embed(wav, lengths=over), eng.embed(wav, lengths=[16000, 16000, 0, 400, 16000, 7777]))
    assert rel(eng.embed(wav, lengths=over)[[0]], alone(eng, wav)[[0]]) < 1e-4


@pytest.mark.parametrize("L", [399, 300, 10, 9, 1])
def test_a_batch_without_a_frame(nrse_device, L):
    """Every utterance is shorter than one frame, and so is the batch: zeros, as for one such utterance among others."""
    eng = engine(torch.float32)
    wav = batch(0.0)[:, :L].contiguous()
    emb = eng.embed(wav, lengths=[L, 0, 1, L, L, 0])
    assert emb.shape == eng.embed(batch(0.0)).shape and emb.dtype == torch.float32 and (emb == 0).all()
