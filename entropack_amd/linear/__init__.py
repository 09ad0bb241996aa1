from .adapters import AdaptedLinear, low_rank_update
from .ahead import DecodeAhead
from .grouped import CompressedGroupedLinear, grouped_int8_linear, grouped_linear
from .groups import RowGroups, combine_rows, group_rows
from .linear import CompressedINT8Linear, CompressedLinear, QuantizedLinear

__all__ = ["AdaptedLinear", "CompressedGroupedLinear", "CompressedINT8Linear", "CompressedLinear", "DecodeAhead", "QuantizedLinear", "RowGroups",
           "combine_rows", "group_rows", "grouped_int8_linear", "grouped_linear", "low_rank_update"]
