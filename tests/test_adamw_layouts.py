"""What the AdamW steps say of tensors that are not dense (no GPU is needed to be refused)."""
import pytest
import torch


def test_sparse_tensors_are_named():
    from fast_sp_gs_amd.adamw import AdamW, adamw_step, grad_norm
    t = torch.zeros(4, 3)
    with pytest.raises(RuntimeError, match='grad must be dense'):
        grad_norm([t.to_sparse()])
    with pytest.raises(RuntimeError, match='param must be dense'):
        adamw_step([t.to_sparse()], [t], [t], [t], [torch.zeros(())])
    embedding = torch.nn.Embedding(5, 3, sparse=True)
    embedding(torch.tensor([1, 2])).sum().backward()
    with pytest.raises(RuntimeError, match='grad must be dense'):
        AdamW(embedding.parameters(), max_norm=1.0).step()
