"""algx: B200-native (sm_100a) kernels for the Algebraic Transformer hot path.

Public API, mirroring the reference's ``algebraic.kernels`` modules:

* ``algx.kernels.flash.flash_attention``    (kernels/flash.py:763)
* ``algx.kernels.fused_head.fused_head``    (kernels/fused_head.py:260)
* ``algx.kernels.qk_norm.qk_rms_norm``      (kernels/qk_norm.py:62)

Serving, which the reference has not:

* ``algx.kernels.paged``   paged key/value cache: append, attention, eviction
* ``algx.kernels.verify``  verification of drafted tokens, sampling
* ``algx.serve``           the model over its cache: prompts, decoding, drafts

The first three are torch ``autograd.Function``s over the C ABI of ``libalgx.so``.
``algx.torch_ops`` registers all of these as ``torch.library``
operators (``torch.ops.algx.*``) for tracers that need opaque nodes.
"""

__version__ = "0.1.0"
