"""What cannot run over pages, or draw tokens, is refused before a model is loaded."""
import importlib
import json

import pytest

import float_cases as fc
from conftest import PKG

config = importlib.import_module(PKG + ".float_config")


@pytest.fixture
def unread(monkeypatch):
    """reading a tensor fails the test"""
    R = importlib.import_module(PKG + ".registry")

    def read(self, *a, **kw):
        raise AssertionError("a tensor was read")
    monkeypatch.setattr(R.TensorFiles, "__call__", read)
    return R


def test_a_model_that_pages_do_not_take_is_refused_unread(float_libpath, tmp_path, unread):
    wide = fc.vifelix(40, 16, 1e-5, 3.0, [fc.parallel(2, 1, 264, 16, 64, 1, 8, 8, 8, [0.9], None)])
    path = fc.write_checkpoint(str(tmp_path / "wide"), wide, fc.make_weights(wide, 3))
    with pytest.raises(NotImplementedError, match="264"):
        unread.load(path, device="cpu", page=16)
    with pytest.raises(AssertionError):                # in slots it would be loaded
        unread.load(path, device="cpu")
    fits = fc.vifelix(40, 16, 1e-5, 3.0, [fc.parallel(2, 1, 250, 16, 64, 1, 8, 8, 8, [0.9], None)])
    path = fc.write_checkpoint(str(tmp_path / "fits"), fits, fc.make_weights(fits, 3))
    with pytest.raises(AssertionError):
        unread.load(path, device="cpu", page=16)
    for bad in (dict(page=12), dict(page=-8), dict(page=2048), dict(page=16, pages=0)):
        with pytest.raises(ValueError):
            unread.load(path, device="cpu", **bad)
    latent = fc.write_checkpoint(str(tmp_path / "latent"), fc.ODD, fc.make_weights(fc.ODD, 11))
    with pytest.raises(NotImplementedError):
        unread.load(latent, device="cpu", page=16)


def test_a_step_of_too_many_sequences_is_refused_unchanged(float_libpath):
    """in front of the cache, which would have grown, and of the first layer's write"""
    import torch
    M = importlib.import_module(PKG + ".float_model")
    cfg = fc.vifelix(40, 16, 1e-5, 3.0, [fc.parallel(2, 1, 24, 16, 64, 1, 8, 8, 8, [0.9], None)])
    shapes = {k: v.shape for k, v in fc.make_weights(cfg, 3).items()}
    args = config.parse_config(cfg, shapes)
    args.page, args.max_batch_size = 16, 1100
    model = M.FloatTransformer(args, torch.bfloat16)
    model.cache = None                                 # whoever asks for it fails
    for S in (1, 3):
        with pytest.raises(ValueError, match="1024"):
            model.step(torch.zeros(1025, S, dtype=torch.int64), 0, list(range(1025)))


@pytest.mark.parametrize("more", [["--sample"], ["--samples", "2"], ["--sample", "--top-k", "3", "--samples", "2"]])
def test_the_program_refuses_to_draw_integer_tokens_unread(tmp_path, monkeypatch, more):
    G, R = (importlib.import_module(PKG + "." + n) for n in ("generate", "registry"))
    (tmp_path / "config.json").write_text(json.dumps({"vocab_size": 100, "dim": 64, "n_layers": 1}))
    assert R.architecture_of(config.read_config(str(tmp_path))) == R.INTEGER_MODEL

    def load(*a, **kw):
        raise AssertionError("the model was loaded")
    monkeypatch.setattr(R, "load", load)
    with pytest.raises(SystemExit):
        G.main(["--model", str(tmp_path), "--tokens", "1"] + more)
    with pytest.raises(AssertionError):
        G.main(["--model", str(tmp_path), "--tokens", "1"])
