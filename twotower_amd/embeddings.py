"""Embedding registry, mirroring twotower/embeddings.py (BaseEmbedding :10-21,
LookupEmbedding :24-40, REGISTRY :159-164, build :166-181).

`LookupEmbedding` keeps the reference's parameter layout (submodule `.embedding` holding an
nn.Embedding(V, E, padding_idx=0) weight, same init) so state_dicts interchange, and adds
`pool_mean(ids)`: the fused HIP gather + masked mean-pool that the towers call instead of
materialising the (B, L, E) lookup.
"""
from __future__ import annotations

import logging
from abc import ABC

import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.overrides import _get_current_function_mode_stack
from torch.utils._device import DeviceContext

from . import _lib, ops

logger = logging.getLogger("twotower_amd.embeddings")


class BaseEmbedding(nn.Module, ABC):
    """Base class for all embedding layers (twotower/embeddings.py:10-21)."""

    def __init__(self, vocab_size: int, embedding_dim: int, padding_idx: int = 0):
        super().__init__()
        self.vocab_size = vocab_size
        self.embedding_dim = embedding_dim
        self.padding_idx = padding_idx

    def log_params(self):
        logger.info(f"Embedding parameters: {self.vocab_size * self.embedding_dim:,}")


_EMBEDDING_FORWARD = nn.Embedding.forward


def _plain_embedding(m) -> bool:
    """An nn.Embedding whose forward is nothing but the row gather of a type the HIP lookup has."""
    w = m.weight
    return (type(m) is nn.Embedding and m.max_norm is None and not m.scale_grad_by_freq and not m.sparse
            and type(w) in (nn.Parameter, torch.Tensor) and w.dtype in _lib.ELEM_DTYPES and w.is_contiguous()
            and not (m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks)
            and "forward" not in m.__dict__ and nn.Embedding.forward is _EMBEDDING_FORWARD
            and not nn.modules.module._has_any_global_hook())


def _observed() -> bool:
    """Whether a tracer, function transform, forward-mode derivative, dispatch or function mode follows torch's own
    calls: it would not see a kernel's.  (torch.set_default_device is such a mode, and looks at factories alone.)"""
    return (torch.compiler.is_compiling() or torch._C._are_functorch_transforms_active()
            or torch._C._len_torch_dispatch_stack() > 0 or torch.jit.is_tracing()
            or forward_ad._current_level >= 0
            or (torch._C._len_torch_function_stack() > 0
                and any(type(m) is not DeviceContext for m in _get_current_function_mode_stack())))


class LookupEmbedding(BaseEmbedding):
    """Trainable lookup table (twotower/embeddings.py:24-40) with a fused pooled lookup."""

    scale = 1.0  # (of modules that were pickled without one)

    def __init__(self, vocab_size: int, embedding_dim: int, padding_idx: int = 0,
                 scatter_mode: str = "sorted", scale: float = 1.0):
        """scale: factor of the token rows that forward() returns (e.g. embedding_dim ** 0.5); the pooled
        lookup is the reference's and takes none."""
        super().__init__(vocab_size, embedding_dim, padding_idx)
        self.scale = float(scale)
        self.embedding = nn.Embedding(vocab_size, embedding_dim, padding_idx=padding_idx)
        if scatter_mode not in ("sorted", "atomic"):
            raise ValueError(f"scatter_mode must be 'sorted' or 'atomic', got {scatter_mode!r}")
        self.scatter_mode = scatter_mode
        self.log_params()

    @property
    def weight(self) -> torch.Tensor:
        return self.embedding.weight

    def forward(self, input_ids: torch.Tensor) -> torch.Tensor:
        """(B, L) ids -> (B, L, E) rows times ``scale``: the reference's unfused contract, for foreign
        towers.  The towers of this package never call it (they use pool_mean).  On the GPU one HIP
        gather forward and, for the dense table gradient, a sum over sorted tokens (ops.embedding_lookup).  An
        id outside the table, which torch's gather stops at, yields a row of NaN there."""
        if torch.jit.is_scripting():
            return self.embedding(input_ids) * self.scale
        return self._rows(input_ids)

    @torch.jit.unused
    def _rows(self, input_ids: torch.Tensor) -> torch.Tensor:
        inner = self.embedding
        if (isinstance(input_ids, torch.Tensor) and input_ids.is_cuda and inner.weight.is_cuda  # (fx: a Proxy is none)
                and not _observed() and _plain_embedding(inner)):
            return ops.embedding_lookup(inner.weight, input_ids, self.scale, inner.padding_idx, strict=True)
        rows = inner(input_ids)
        return rows if self.scale == 1.0 else rows * self.scale

    def pool_mean(self, input_ids: torch.Tensor) -> torch.Tensor:
        """(B, L) ids -> (B, E): sum_{ids>0} W[ids] / (count + 1e-9) on the HIP bag kernel
        (twotower/encoders.py:62-72 fused with the lookup at embeddings.py:40)."""
        mode = _lib.TT_SCATTER_SORTED if self.scatter_mode == "sorted" else _lib.TT_SCATTER_ATOMIC
        return ops.bag_mean_pool(self.embedding.weight, input_ids, self.padding_idx, mode)


class _Unavailable(BaseEmbedding):
    """word2vec / glove need gensim and a network download (embeddings.py:49,101,107); neither
    exists in this environment, and both are outside the accelerated path."""

    def __init__(self, *args, **kwargs):
        raise ImportError(f"{type(self).__name__}: pretrained vectors need gensim + network access; "
                          "not provided by twotower_amd")


class FrozenWord2Vec(_Unavailable):
    pass


class GloVeEmbedding(_Unavailable):
    pass


REGISTRY = {
    "lookup": LookupEmbedding,
    "word2vec": FrozenWord2Vec,
    "glove": GloVeEmbedding,
}


def build(name: str, vocab_size: int, **kwargs) -> BaseEmbedding:
    """Build an embedding layer by name (twotower/embeddings.py:166-181)."""
    if name not in REGISTRY:
        raise ValueError(f"Unknown embedding: {name}. Available options: {list(REGISTRY.keys())}")
    return REGISTRY[name](vocab_size=vocab_size, **kwargs)
