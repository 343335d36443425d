"""The host's side of clipping, without a GPU: arguments, refusals, and where a rank without gradients puts
its state."""
import ctypes
import inspect
import subprocess
import sys
import types

import pytest
import torch

from muon_sr_b200 import _lib, clip_grad_norm_, clipping, get_total_norm
from muon_sr_b200 import kernels as K
from tests.conftest import ROOT


class OnDevice:
    """A parameter of CUDA device `index` as far as the tables look at one."""

    def __init__(self, index, grad=True):
        self.index, self.grad = index, grad or None

    def get_device(self):
        return self.index


@pytest.mark.parametrize("params,want", [
    ([OnDevice(1), OnDevice(1)], 1),
    ([OnDevice(0, grad=False), OnDevice(1)], 1),   # those with a gradient come first
    ([OnDevice(1, grad=False)], 1),
    ([], 3),                                       # nothing says where: the current device
])
def test_rank_without_gradients_uses_the_parameters_device(params, want, monkeypatch):
    made = []
    monkeypatch.setattr(K, "GradTable", lambda grads, device=None: made.append((grads, device)))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    clipping._gradients(params, types.SimpleNamespace(owned=lambda ps: []))
    assert made == [([], want)]


def test_rank_without_gradients_refuses_cpu_parameters():
    """As the ranks that hold the gradients do, so that none waits for another."""
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    with pytest.raises(ValueError, match="no CPU path"):
        clipping._gradients([p], types.SimpleNamespace(owned=lambda ps: []))


def test_arguments_of_the_torch_namesakes():
    """torch.nn.utils takes `foreach`, which chooses between its own loops."""
    p = torch.nn.Parameter(torch.zeros(3))
    for foreach in (None, True, False):
        assert float(get_total_norm([], 2.0, False, foreach)) == 0.0
        assert float(clip_grad_norm_([p], 1.0, 2.0, False, foreach)) == 0.0
        assert float(get_total_norm([], foreach=foreach)) == 0.0
        assert float(clip_grad_norm_([p], 1.0, foreach=foreach)) == 0.0
    for ours, theirs in ((get_total_norm, torch.nn.utils.get_total_norm),
                         (clip_grad_norm_, torch.nn.utils.clip_grad_norm_)):
        names = list(inspect.signature(theirs).parameters)
        assert list(inspect.signature(ours).parameters)[:len(names)] == names


def test_8bit_launch_of_nothing_needs_no_hyperparameters():
    """In a process of its own: the call read through the null pointer."""
    code = ("from muon_sr_b200 import _lib; import ctypes; lib = _lib.load(); x = ctypes.create_string_buffer(64); "
            "assert lib.msr_adamw8bit(None, 0, None, None, None, None) == 0; "
            "assert lib.msr_adamw8bit_scaled(None, 0, None, None, None, ctypes.addressof(x) // 16 * 16 + 16, None) == 0; "
            "assert lib.msr_adamw8bit(None, 1, None, None, None, None) == 1; "
            "hp = _lib.Adam8Hparams(); hp.block_size = 100; "
            "assert lib.msr_adamw8bit(None, 0, None, None, ctypes.byref(hp), None) == 1")
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert done.returncode == 0, (done.returncode, done.stderr)


def test_norms_of_each_entry_need_an_aligned_pointer():
    lib = _lib.load()
    at = ctypes.create_string_buffer(64)
    ptr = (ctypes.addressof(at) + 15) // 16 * 16      # never dereferenced: every call is refused
    need = lib.msr_grad_norm_workspace_bytes(1)
    entry = (ctypes.c_int64 * 3)(ptr, 4, 0)
    for off in (1, 2, 3):
        assert lib.msr_grad_norm(entry, 1, 2, 1.0, 1.0, ptr, ptr + 32 + off, ptr, need, None) == 1
        assert b"each" in lib.msr_last_error()


def test_grad_scale_outside_fp32_is_refused():
    """The factor that the kernels multiply by is fp32: beyond its range it would be 0 or infinity."""
    p = torch.nn.Parameter(torch.zeros(3))
    lib = _lib.load()
    at = ctypes.create_string_buffer(64)
    ptr = (ctypes.addressof(at) + 15) // 16 * 16      # never dereferenced: every call is refused
    for bad in (3.5e38, 1e300, 2.0 ** -127, 1e-46, 1e-320):
        with pytest.raises(ValueError, match="grad_scale"):
            clip_grad_norm_([p], 1.0, grad_scale=bad)
        with pytest.raises(ValueError, match="grad_scale"):
            clipping.clipped_step(types.SimpleNamespace(param_groups=[]), 1.0, bad)
        assert lib.msr_grad_factor(ptr, 2, bad, 1.0, None) == 1
        assert b"scale" in lib.msr_last_error()
    for good in (2.0 ** -126, 3.4e38):
        assert float(clip_grad_norm_([p], 1.0, grad_scale=good)) == 0.0


def test_scaled_apply_needs_its_factor():
    lib = _lib.load()
    at = ctypes.create_string_buffer(64)
    ptr = (ctypes.addressof(at) + 15) // 16 * 16      # never dereferenced: every call is refused or empty
    for bad in (None, ptr + 2):
        assert lib.msr_muon_apply_scaled(None, 0, 0.02, 1.0, bad, None) == 1
        assert lib.msr_muon_apply_rec_scaled(None, 0, ptr, bad, None) == 1
    assert lib.msr_muon_apply_rec_scaled(None, 0, ptr + 4, ptr, None) == 1
    assert lib.msr_muon_apply_scaled(None, 1, 0.02, 1.0, ptr, None) == 1
    assert lib.msr_muon_apply_scaled(None, 0, 0.02, 1.0, ptr, None) == 0
