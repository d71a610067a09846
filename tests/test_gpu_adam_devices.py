"""FusedAdam's launches run on its parameters' device: tensors of another one are refused (a stand-in says where it lies: one GPU
is enough)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Elsewhere:
  """a tensor's face, on another device; nothing reads its memory"""
  dtype, is_cuda, device = torch.float32, True, torch.device("cuda:1")

  def __init__(self, *shape):
    self.shape = torch.Size(shape)

  def numel(self):
    return self.shape.numel()

  def is_contiguous(self):
    return True

  def __getattr__(self, name):
    raise AssertionError(f"{name} of a tensor on another device was asked for")


def test_gradients_and_parameters_of_another_device():
  from orca_amd import ops
  from orca_amd._lib import OrcaError
  opt = ops.FusedAdam({"a": torch.zeros(3, 4, device=DEV), "b": torch.zeros(5, device=DEV)})
  for max_norm in (None, 1.0):
    with pytest.raises(OrcaError, match="gradient of b"):
      opt.step({"a": torch.ones(3, 4, device=DEV), "b": Elsewhere(5)}, max_norm=max_norm)
  assert opt.steps == {"a": 0, "b": 0} and not bool(opt.params["a"].any())
  with pytest.raises(OrcaError, match="parameter b"):
    ops.FusedAdam({"a": torch.zeros(3, 4, device=DEV), "b": Elsewhere(5)})
  opt.step({"a": torch.ones(3, 4, device=DEV)})
  assert bool((opt.params["a"] != 0).all())
