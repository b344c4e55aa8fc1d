"""Native kernels of the MLA backend (libmla_amd.so via ctypes)."""

from .lib import (
    MLAKernelError,
    PageTables,
    decode_plan,
    device_cu_count,
    gqa_chunk,
    gqa_decode,
    gqa_prompt,
    gqa_workspace,
    gqa_workspace_bytes,
    load_library,
    mla_decode,
    mla_decode_merge,
    mla_prefill,
    page_table_from_tokens,
    page_tables_from_lengths,
    store_rows,
)

__all__ = [
    "MLAKernelError",
    "PageTables",
    "decode_plan",
    "device_cu_count",
    "gqa_chunk",
    "gqa_decode",
    "gqa_prompt",
    "gqa_workspace",
    "gqa_workspace_bytes",
    "load_library",
    "mla_decode",
    "mla_decode_merge",
    "mla_prefill",
    "page_table_from_tokens",
    "page_tables_from_lengths",
    "store_rows",
]
