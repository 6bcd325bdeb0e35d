"""What token_log_probs and distillation_loss refuse of tensors on the GPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(gpu_device):
    from gpt_triton_amd import kernels

    return kernels


def test_scores(K, gpu_device, monkeypatch):
    x = torch.zeros(4, 300, dtype=torch.float16, device=gpu_device)
    t = torch.zeros(4, dtype=torch.int64, device=gpu_device)
    with pytest.raises(TypeError):
        K.token_log_probs(x.bfloat16(), t)
    with pytest.raises(TypeError):
        K.token_log_probs(x, t.int())
    with pytest.raises(AssertionError):
        K.token_log_probs(x, t[:3])
    with pytest.raises(AssertionError):
        K.token_log_probs(x, torch.zeros(4, 2, dtype=torch.int64, device=gpu_device)[:, 0])
    with pytest.raises(RuntimeError):
        K.token_log_probs(x, t.cpu())
    with pytest.raises(AssertionError):
        K.token_log_probs(x, t, top=301)
    with pytest.raises(AssertionError):
        K.token_log_probs(x, t, top=-1)
    with pytest.raises(NotImplementedError):
        K.token_log_probs(x, t, top=129)
    for tau in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            K.token_log_probs(x, t, temperature=tau)
    monkeypatch.setenv("GPTMI_CHECK_IDS", "1")
    K.token_log_probs(x, t - 100)
    with pytest.raises(IndexError):
        K.token_log_probs(x, t + 300)


def test_distillation(K, gpu_device, monkeypatch):
    x = torch.zeros(4, 300, device=gpu_device)
    ids = torch.zeros(4, 3, dtype=torch.int64, device=gpu_device)
    teacher = torch.zeros(4, 3, device=gpu_device)
    w = torch.ones(4, device=gpu_device)
    for args, error in (((x, ids.int(), teacher), TypeError), ((x, ids[:3], teacher), AssertionError),
                        ((x, ids, teacher[:, :2]), AssertionError), ((x, ids, teacher.double()), TypeError),
                        ((x, ids[:, :0], teacher[:, :0]), AssertionError), ((x, ids.cpu(), teacher), RuntimeError),
                        ((x, ids, teacher, 0.0), ValueError), ((x, ids, teacher, 1.0, w.half()), TypeError),
                        ((x, ids, teacher, 1.0, w[:3]), AssertionError),
                        ((x, ids.repeat(1, 43), teacher.repeat(1, 43)), NotImplementedError)):
        for call in (K.distillation_loss, K.distillation_loss_and_grad):
            with pytest.raises(error):
                call(*args)
    monkeypatch.setenv("GPTMI_CHECK_IDS", "1")
    with pytest.raises(IndexError):
        K.distillation_loss(x, ids + 300, teacher)
