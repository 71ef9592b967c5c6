"""B200 kernels behind the reference's kernel entry points
(hybrid_xmamba/kernels/__init__.py:3-9): ``apply_tfla`` and ``selective_scan``,
plus the extended entries ``selective_scan_fn``, ``mlstm_chunkwise_fwd`` /
``mlstm_chunkwise_bwd``, ``ssd_chunk_scan`` / ``ssd_chunk_scan_fn`` (with its
backward), ``linear_attention`` / ``linear_attention_step`` (linear attention
with a constant decay per head), ``slstm_scan``, ``causal_conv1d``,
``rmsnorm``, ``qk_norm_rope`` (norms of q's and k's heads with the position
rotation) and ``sample_tokens``."""
from .selective_scan.scan_interface import selective_scan, selective_scan_fn
from .tfla.tfla_interface import apply_tfla, mlstm_chunkwise_bwd, mlstm_chunkwise_fwd
from .ssd import ssd_chunk_scan, ssd_chunk_scan_bwd, ssd_chunk_scan_fn
from .linear_attn import linear_attention, linear_attention_bwd, linear_attention_step
from .slstm import slstm_scan
from .conv import causal_conv1d
from .norm import rmsnorm
from .qk_norm_rope import qk_norm_rope, qk_norm_rope_bwd
from .sample import sample_tokens

__all__ = ["apply_tfla", "selective_scan", "selective_scan_fn", "mlstm_chunkwise_fwd", "mlstm_chunkwise_bwd",
           "ssd_chunk_scan", "ssd_chunk_scan_bwd", "ssd_chunk_scan_fn", "linear_attention", "linear_attention_bwd",
           "linear_attention_step", "slstm_scan", "causal_conv1d", "rmsnorm", "qk_norm_rope", "qk_norm_rope_bwd",
           "sample_tokens"]
