"""The workspace of a Kv8Cache's attention is sized under the cache's device,
not under the caller's (device and library are stand-ins)."""
import contextlib
import importlib

import torch

KV8 = importlib.import_module("numerics-and-sparse-attn_b200.kv8")


def test_workspace_is_sized_under_the_caches_device(monkeypatch):
    current, asked = ["cuda:0"], []

    @contextlib.contextmanager
    def on_device(device):
        before, current[0] = current[0], str(device)
        yield
        current[0] = before

    class Library:
        def nsa_kv8_workspace_bytes(self, desc, heads, n_tokens):
            asked.append(current[0])
            return 1024

    monkeypatch.setattr(KV8._lib, "on_device", on_device)
    monkeypatch.setattr(KV8, "_scratch", lambda device, nbytes, stream: (str(device), nbytes))
    monkeypatch.setattr(KV8, "_stream", lambda index: 0)
    c = KV8.Kv8Cache.__new__(KV8.Kv8Cache)
    c.device, c.batch, c._index, c._lib, c._desc_ref, c._ws_bytes = torch.device("cuda", 1), 2, 1, Library(), None, {}
    assert c._scratch(8, 1) == ("cuda:1", 1024) and c._scratch(8, 1) == ("cuda:1", 1024)
    assert asked == ["cuda:1"] and current == ["cuda:0"]
