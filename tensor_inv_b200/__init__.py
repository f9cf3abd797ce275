"""tensor_inv_b200: B200-native (sm_100a) CRT-emulated float64 matmul for tensor_inv.

Drop-in for the reference package's public API (src/tensor_inv/__init__.py:1-6):
``crt_matmul``, ``lu``, ``cholesky``, ``rsvd``.  The compute path is the C-ABI library
``libtensor_inv_crt.so`` (hand-written CUDA for sm_100a); there is no CPU fallback.

Beside them, without a counterpart in the reference: ``low_rank_matmul`` applies low-rank factors
(such as ``rsvd``'s) next to a shared product, and ``dropout`` is the counter-based dropout it uses.
"""

from tensor_inv_b200.cholesky import cholesky
from tensor_inv_b200.crt_matmul import crt_matmul, crt_matmul_update
from tensor_inv_b200.dropout import dropout, dropout_backward
from tensor_inv_b200.low_rank import low_rank_matmul, low_rank_matmul_backward
from tensor_inv_b200.lu import lu
from tensor_inv_b200.rsvd import rsvd

__all__ = ["cholesky", "crt_matmul", "crt_matmul_update", "dropout", "dropout_backward",
           "low_rank_matmul", "low_rank_matmul_backward", "lu", "rsvd"]
