"""entropack_amd: the lossy decode-and-matmul path of EntroPack, built for AMD Instinct MI355X (gfx950).

Drop-in names: `compress`, `decompress`, `CompressedTensor`, `EntroPackLossyConfig`, `TileANSConfig`, `CompressedLinear`,
`CompressedINT8Linear`; `BatchDecompressor` / `DecodeAhead` decode many layers per pass; `group_rows`,
`grouped_linear`, `combine_rows` and `low_rank_update` (with `CompressedGroupedLinear`, `AdaptedLinear`) let every activation row pick its
weight. Decoding runs on the `hip` backend only.
"""
from .compression import BatchDecompressor, CompressedTensor, CompressionFallbackWarning, compress, decompress, decompress_many
from .linear import (AdaptedLinear, CompressedGroupedLinear, CompressedINT8Linear, CompressedLinear, DecodeAhead, RowGroups, combine_rows, group_rows,
                     grouped_int8_linear, grouped_linear, low_rank_update)
from .registry import DispatchError
from .schemes import CompressionConfig, EntroPackLossyConfig, LatticeRANSConfig, RawConfig, TileANSConfig

__version__ = "0.1.0"

__all__ = [
    "AdaptedLinear", "BatchDecompressor", "CompressedGroupedLinear", "CompressedINT8Linear", "CompressedLinear", "CompressedTensor", "CompressionConfig", "CompressionFallbackWarning", "DecodeAhead", "DispatchError", "EntroPackLossyConfig",
    "LatticeRANSConfig", "RawConfig", "RowGroups", "TileANSConfig", "__version__", "combine_rows", "compress", "decompress", "decompress_many",
    "group_rows", "grouped_int8_linear", "grouped_linear", "low_rank_update",
]
