"""Batch-invariant mode in a process that has used the device before: what it may still change there."""
import os

import pytest
import torch

from vllm_b200 import envs
from vllm_b200.utils import batch_invariant as bi


@pytest.fixture
def mode(monkeypatch):
    """The mode asked for; variables and settings of the process are put back."""
    m, flags = torch.backends.cuda.matmul, ("allow_tf32", "allow_bf16_reduced_precision_reduction", "allow_fp16_reduced_precision_reduction")
    before, cudnn = {f: getattr(m, f) for f in flags}, torch.backends.cudnn.allow_tf32
    for k in (*bi._NCCL, "CUBLAS_WORKSPACE_CONFIG"):
        monkeypatch.setenv(k, "")                    # (so that what the call sets is undone)
        monkeypatch.delenv(k)
    monkeypatch.setenv("VLLM_BATCH_INVARIANT", "1")
    envs._cache.clear()
    yield monkeypatch
    for f, v in before.items():
        setattr(m, f, v)
    torch.backends.cudnn.allow_tf32 = cudnn
    envs._cache.clear()


@pytest.mark.parametrize("used", [False, True])
def test_workspaces_keep_their_size_once_the_device_is_in_use(mode, used):
    mode.setattr(torch.cuda, "is_initialized", lambda: used)
    assert bi.apply_env_overrides()
    assert os.environ.get("CUBLAS_WORKSPACE_CONFIG") == (None if used else ":4096:8")
    assert os.environ["NCCL_ALGO"] == "allreduce:tree" and not torch.backends.cuda.matmul.allow_tf32


def test_a_size_that_the_user_chose_stays(mode):
    mode.setenv("CUBLAS_WORKSPACE_CONFIG", ":16:8")
    assert bi.apply_env_overrides() and os.environ["CUBLAS_WORKSPACE_CONFIG"] == ":16:8"
