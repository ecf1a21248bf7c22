"""octex for MI355X: approximate k-nearest-neighbor search by E8-lattice cell lists (cuvs::neighbors::octex),
with every search step a hand-written HIP kernel for gfx950.

    import octex_amd as octex
    index = octex.load("index_dir")        # or octex.build(xb, "index_dir")
    D, I = index.search(xq, k=10)          # (distances, neighbors), nearest first

Operators on rows of scores, for models that make the queries or read the neighbors (octex_amd/scores.py):
quantize_rows, int8_scores, log_probs, log_probs_backward, distill, distill_backward, distill_step, policy_loss,
policy_loss_backward, policy_step, balance_loss, balance_loss_backward, balance_step.  Rows of a table by ids, and the table's
gradient (octex_amd/tables.py): embed, embed_backward.

Drop-ins: `from octex_amd import cuvs as cagra` (cuvs.neighbors.cagra calls) and `from octex_amd import faiss`
(Faiss GPU index calls).
"""

from .index import Index, build, build_in_memory, load
from .scores import (BalanceLoss, LogProbs, PolicyLoss, balance_loss, balance_loss_backward, balance_step, distill,
                     distill_backward, distill_step, int8_scores, log_probs, log_probs_backward, policy_loss,
                     policy_loss_backward, policy_step, quantize_rows)
from .tables import embed, embed_backward

__version__ = "0.1.0"
__all__ = ["BalanceLoss", "Index", "LogProbs", "PolicyLoss", "balance_loss", "balance_loss_backward", "balance_step", "build",
           "build_in_memory", "distill", "distill_backward", "distill_step", "embed", "embed_backward", "int8_scores", "load",
           "log_probs", "log_probs_backward", "policy_loss", "policy_loss_backward", "policy_step", "quantize_rows",
           "__version__"]
