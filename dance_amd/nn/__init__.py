from .gnn import AdaptiveSAGE
from .typed import GatedResidualNorm, RowNorm, TypedLinear, group_rows

__all__ = ["AdaptiveSAGE", "GatedResidualNorm", "RowNorm", "TypedLinear", "group_rows"]
