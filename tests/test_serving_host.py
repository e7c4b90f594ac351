"""The command line's sampling options reach the model, and what no model has is refused."""
import pytest


class Model:
    def __init__(self):
        self.calls = []

    def generate(self, prompts, n, **how):
        self.calls.append((prompts, n, how, getattr(self, "kv_cache", None)))
        return [[1, 2]]

    def status(self):
        pass


class Cached(Model):
    kv_cache = "bf16"


def run(monkeypatch, model, *argv):
    from baranet_bdml_b200 import __main__ as main, registry
    monkeypatch.setattr(registry, "load_model", lambda folder, dtype: model)
    return main.main(["generate", "--model", "x", "--prompt", "5 17 3", *argv])


def test_options_reach_the_model(monkeypatch, capsys):
    model = Cached()
    assert run(monkeypatch, model, "--temperature", "0.7", "--top-k", "40", "--top-p", "0.9", "--min-p", "0.05", "--seed", "3", "--kv-cache", "int8") == 0
    assert run(monkeypatch, model) == 0
    assert model.calls[0] == ([[5, 17, 3]], 50, dict(temperature=0.7, top_k=40, top_p=0.9, min_p=0.05, seed=3), "int8")
    assert model.calls[1][2] == dict(temperature=0.0, top_k=0, top_p=1.0, min_p=0.0, seed=None)
    assert capsys.readouterr().out == "1 2\n1 2\n"


def test_a_cache_of_another_kind_is_refused(monkeypatch, capsys):
    model = Model()
    with pytest.raises(SystemExit):
        run(monkeypatch, model, "--kv-cache", "e4m3")
    assert not model.calls and "--kv-cache" in capsys.readouterr().err
