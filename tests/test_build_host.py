"""CPU: what makes the libraries be rebuilt, and what a build refuses."""
import torch

import q3attn.build as build


def test_another_torch_means_another_build(monkeypatch):
    """The bindings are compiled against torch's C++ interface: a library built for another torch is not up to date."""
    here = build.source_digest()
    assert build.source_digest() == here
    monkeypatch.setattr(torch, "__version__", "9.9.9+cu999")
    assert build.source_digest() != here and not build.up_to_date()
    monkeypatch.undo()
    monkeypatch.setattr(torch._C, "_GLIBCXX_USE_CXX11_ABI", not torch._C._GLIBCXX_USE_CXX11_ABI)
    assert build.source_digest() != here
