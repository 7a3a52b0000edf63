"""Masks as 32-bit words."""
import torch


def words_of(on):
    """bool[..., vocab] as 32-bit words, with ones behind the last logit."""
    pad = torch.ones(*on.shape[:-1], -on.shape[-1] % 32, dtype=torch.bool, device=on.device)
    bits = torch.cat([on, pad], -1).view(*on.shape[:-1], -1, 32).int()
    return (bits << torch.arange(32, device=on.device, dtype=torch.int32)).sum(-1, dtype=torch.int32)
