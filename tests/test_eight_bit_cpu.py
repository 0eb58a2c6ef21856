"""Host-side choices of the eight-bit operators that need no GPU."""

from __future__ import annotations

import sys
import sysconfig

import pytest
import torch
import torch.nn as nn

from double_attention_b200 import DoubleAttentionBlock, build, eight_bit, experiment_config


class _Adapted(nn.Linear):
    def forward(self, x):
        return super().forward(x) + 1


@pytest.mark.parametrize("change", ["none", "hook", "pre-hook", "backward hook", "sequence hook", "subclass", "instance",
                                    "activation", "global hook"])
def test_a_feed_forward_with_hooks_or_forwards_of_its_own_is_called_as_modules(change: str, monkeypatch) -> None:
    """With activations kept in 8 bits the branch reads the layers' weights; what its modules do besides has to run."""
    block = DoubleAttentionBlock(experiment_config("a1"), feedforward_dim=1536)
    calls: list[str] = []
    monkeypatch.setattr(eight_bit, "FEEDFORWARD_CHECKPOINT8", True)
    monkeypatch.setattr(eight_bit, "checkpoint8_supported", lambda x, *layers: True)
    monkeypatch.setattr(eight_bit, "feedforward_checkpoint8", lambda x, first, second: calls.append("kept") or torch.zeros_like(x))
    note, handle = lambda *args: calls.append(change), None
    if change == "hook":
        block.feedforward[2].register_forward_hook(note)
    elif change == "pre-hook":
        block.feedforward[0].register_forward_pre_hook(note)
    elif change == "backward hook":
        block.feedforward[0].register_full_backward_hook(note)
    elif change == "sequence hook":
        block.feedforward.register_forward_hook(note)
    elif change == "subclass":
        block.feedforward[0] = _Adapted(512, 1536)
    elif change == "instance":
        block.feedforward[0].forward = lambda x, layer=block.feedforward[0]: nn.functional.linear(x, 2 * layer.weight, layer.bias)
    elif change == "activation":
        block.feedforward[1] = nn.ReLU()
    elif change == "global hook":
        handle = nn.modules.module.register_module_forward_hook(note)
    x = torch.randn(2, 3, 512)
    try:
        y = block._feedforward_branch(x, None, None)
        if change == "none":
            assert calls == ["kept"]
        else:
            assert "kept" not in calls
            assert torch.equal(y, block.feedforward(x))
            if "hook" in change and "backward" not in change:
                assert change in calls
    finally:
        if handle is not None:
            handle.remove()


def test_a_checkpoint_without_dimensions_is_refused() -> None:
    x = torch.zeros(1, 32, dtype=torch.int8)
    kept = eight_bit.Checkpoint8(x, x[:, :1], (), torch.bfloat16)
    for call in (kept.restore, lambda: eight_bit.weight_grad_checkpoint8(torch.zeros(8, dtype=torch.bfloat16), kept),
                 lambda: eight_bit.gelu_checkpoint8_backward(torch.zeros((), dtype=torch.bfloat16), kept)):
        with pytest.raises(ValueError, match="takes a checkpoint"):
            call()


def _copy_of_the_package(tmp_path, monkeypatch) -> None:
    """The build's paths moved to ``tmp_path``, with a library that is up to date (no nvcc run)."""
    for name in ("libda_b200.so", build.HOST_PATH.name):
        (tmp_path / name).write_bytes(b"")
    monkeypatch.setattr(build, "PACKAGE_DIR", tmp_path)
    monkeypatch.setattr(build, "BUILD_DIR", tmp_path)
    monkeypatch.setattr(build, "LIB_PATH", tmp_path / "libda_b200.so")
    monkeypatch.setattr(build, "HOST_PATH", tmp_path / build.HOST_PATH.name)
    monkeypatch.setattr(build, "_needs_build", lambda *args: False)
    for source in build.CSRC.glob("*.cu"):
        (tmp_path / f"{source.stem}.o").write_bytes(b"")
    (tmp_path / "libda_b200.so").write_bytes(b"library")  # newer than its objects


@pytest.mark.parametrize("missing", ["compiler", "headers"])
def test_the_library_builds_without_the_host_extension(missing: str, tmp_path, monkeypatch) -> None:
    _copy_of_the_package(tmp_path, monkeypatch)
    build.HOST_PATH.unlink()
    if missing == "compiler":
        monkeypatch.setenv("CXX", str(tmp_path / "no-such-compiler"))
    else:
        paths = dict(sysconfig.get_paths(), include=str(tmp_path))
        monkeypatch.setattr(sysconfig, "get_paths", lambda: paths)
    with pytest.warns(RuntimeWarning, match="was not built"):
        assert build.build() == build.LIB_PATH
    assert build.LIB_PATH.read_bytes() == b"library" and not build.HOST_PATH.exists()


def test_calls_do_without_the_host_extension(monkeypatch) -> None:
    monkeypatch.setattr(eight_bit, "_host_module", None)
    monkeypatch.setitem(sys.modules, "double_attention_b200._host_calls", None)  # (importing it raises ImportError)
    monkeypatch.delattr(sys.modules["double_attention_b200"], "_host_calls", raising=False)
    with pytest.warns(RuntimeWarning, match="cannot be used"):
        host = eight_bit._host()
    assert host.linear() is None and host.norm(1, 2) is None and eight_bit._host() is host


def test_the_host_extension_is_rebuilt_for_another_interpreter_pytorch_source_or_command(tmp_path, monkeypatch) -> None:
    _copy_of_the_package(tmp_path, monkeypatch)
    assert build.HOST_PATH.name.endswith(sysconfig.get_config_var("EXT_SUFFIX"))  # as this interpreter looks for it
    runs: list[list[str]] = []

    def compiler(cmd, **kwargs):
        runs.append(cmd)
        build.Path(cmd[cmd.index("-o") + 1]).write_bytes(b"extension")
        return type("Done", (), {"returncode": 0})()

    monkeypatch.setattr(build.subprocess, "run", compiler)
    source = tmp_path / "host_calls.cpp"
    source.write_text("one")
    monkeypatch.setattr(build, "HOST_SRC", source)
    build.HOST_PATH.write_bytes(b"of unknown origin")

    def runs_of_a_build() -> int:
        runs.clear()
        assert build.build_host_calls() == build.HOST_PATH
        return len(runs)

    assert runs_of_a_build() == 1 and build.HOST_PATH.read_bytes() == b"extension"
    assert runs_of_a_build() == 0
    source.write_text("two")
    assert runs_of_a_build() == 1 and runs_of_a_build() == 0
    monkeypatch.setattr(torch, "__version__", "0.0")  # an older one than was there
    assert runs_of_a_build() == 1 and runs_of_a_build() == 0
    monkeypatch.setenv("CXX", "another")
    assert runs_of_a_build() == 1 and runs_of_a_build() == 0
    build.HOST_PATH.unlink()
    assert runs_of_a_build() == 1


def test_an_extension_built_for_another_pytorch_is_not_called(monkeypatch) -> None:
    _host_calls = pytest.importorskip("double_attention_b200._host_calls")  # (where it could be built)
    monkeypatch.setattr(eight_bit, "_host_module", None)
    monkeypatch.setattr(_host_calls, "torch_version", "0.0")
    with pytest.warns(RuntimeWarning, match="built for PyTorch 0.0"):
        assert eight_bit._host() is not _host_calls
