"""hisparse_b200 — nano-hisparse's per-step sparse-decode hot path on B200.

Operators with the reference's signatures (drop-in for the modules of the
same names in nano_hisparse):

  selection.quest_selection   Quest scoring + shared top-k + token expansion
  row_index.resolve_rows      resident/hot lookup, LRU replacement, miss plan
  row_kernels.gather_rows     pinned host -> pool miss gather (zero-copy)
  row_kernels.attend_rows     physical-row GQA decode attention
  attention.row_attention     resolve + gather + attend through a cache

and those of a verification step, which checks several drafted tokens of a
request in one forward:

  norm_rope.qk_norm_rope      per-head query/key norms with the rotation
  tree.attend_tree            attention of a tree of drafted tokens over cache rows
  logprobs.token_logprobs     log probabilities, entropy, top alternatives

and those of a cache held in 8 bits (CacheConfig(dtype=torch.float8_e4m3fn)), which
the classes and functions above take by themselves on such a cache:

  quantized.append_quantized  rows quantised as they are written
  quantized.read_quantized    rows read back
  quantized.attend_quantized  decode attention over them

plus RowCache (device state and the resolve stream/event protocol),
DecodeBatch (the same hot path for B requests per launch) and
plugin.install (routes an imported reference package through these kernels).
All compute runs in libhisparse.so (sm_100a CUDA, C ABI in include/hisparse.h,
include/hisparse_verify.h and include/hisparse_quantized.h).
"""

from .attention import row_attention
from .batched import DecodeBatch
from .cache import LayerTables, RowCache, RowLease
from .config import ACTIVE_TAIL_PAGES, CacheConfig, CapacityError, HotConfig
from .draft import PromptLookup
from .logprobs import TokenLogprobs, token_logprobs
from .norm_rope import qk_norm_rope, rope_frequencies
from .quantized import append_quantized, attend_quantized, read_quantized
from .row_index import LogicalTopK, RowPlan, resolve_rows
from .row_kernels import MappedHost, attend_rows, gather_rows
from .selection import Selection, quest_selection
from .tree import attend_tree, tree_mask

__all__ = [
    "ACTIVE_TAIL_PAGES", "CacheConfig", "CapacityError", "DecodeBatch", "HotConfig", "LayerTables",
    "LogicalTopK", "MappedHost", "PromptLookup", "RowCache", "RowLease", "RowPlan", "Selection",
    "TokenLogprobs", "append_quantized", "attend_quantized", "attend_rows", "attend_tree",
    "gather_rows", "qk_norm_rope", "quest_selection", "read_quantized", "resolve_rows",
    "rope_frequencies", "row_attention", "token_logprobs", "tree_mask",
]
