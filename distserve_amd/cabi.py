"""ctypes binding of the kvmove C ABI (``include/kvmove.h``), one Python function per entry point.

Pointers are plain integers (``tensor.data_ptr()``), streams are ``hipStream_t`` values as
integers (``torch.cuda.current_stream().cuda_stream``).  A nonzero return code raises
``KvmError`` carrying ``kvm_last_error()``.

The module-level functions bind the package's own ``lib/libkvmove.so``.  ``Binding(path)``
binds any other build of the same interface with the same functions as methods (the tests
bind the exploration build, which has its own registry and options, beside the product).
"""
from __future__ import annotations

import ctypes
import os
from typing import List, Sequence

KVM_OK = 0
KVM_EINVAL = -1
KVM_ERANGE = -2
KVM_EDUP = -3
KVM_ENOTREG = -4
KVM_EHIP = -5
KVM_EHANDLE = -6
KVM_EMISMATCH = -7
KVM_HANDLE_WORDS = 18
KVM_ABI_MAJOR = 1
KVM_IPC_MAX_ALLOC_BYTES = 1 << 31

# every symbol include/kvmove.h declares
EXPORTS = (
    "kvm_version", "kvm_last_error", "kvm_get_mem_handle", "kvm_register_mem_handle",
    "kvm_register_source", "kvm_reset", "kvm_opened_handles", "kvm_migrate", "kvm_swap", "kvm_copy_plain",
    "kvm_set_option", "kvm_get_option", "kvm_migrate_plan", "kvm_swap_plan", "kvm_debug_divide",
    "kvm_plan_words", "kvm_plan_step", "kvm_write_kv", "kvm_read_kv", "kvm_attention_workspace",
    "kvm_paged_attention", "kvm_prompt_attention",
)

# element types and pool formats of the cache operators
KVM_F16, KVM_BF16, KVM_F32 = 0, 1, 2
KVM_CACHE_PLAIN, KVM_CACHE_E4M3 = 0, 1
KVM_MAX_HEAD_DIM = 256


class KvmError(RuntimeError):
    def __init__(self, code: int, text: str):
        super().__init__(f"{text} (kvmove error {code})")
        self.code = code


class KvmGeom(ctypes.Structure):
    _fields_ = [
        ("num_layers", ctypes.c_int64), ("num_kv_heads", ctypes.c_int64), ("block_size", ctypes.c_int64),
        ("head_dim", ctypes.c_int64), ("dtype_bytes", ctypes.c_int64),
        ("ctx_pp_size", ctypes.c_int32), ("ctx_tp_size", ctypes.c_int32),
        ("dec_pp_size", ctypes.c_int32), ("dec_tp_size", ctypes.c_int32),
        ("dec_pp_rank", ctypes.c_int32), ("dec_tp_rank", ctypes.c_int32),
        ("ctx_instance", ctypes.c_int64),
    ]


class KvmStep(ctypes.Structure):
    """What a step plan says about itself (filled by ``plan_step``)."""

    _fields_ = [(name, ctypes.c_int64) for name in (
        "words", "num_seqs", "num_tokens", "num_kv_tokens", "num_pages", "num_blocks", "block_size", "num_heads",
        "num_kv_heads", "head_dim", "all_new", "dtype", "format", "row_tiles", "num_row_tiles", "num_row_groups",
        "num_tile_items", "num_joins", "join_rows", "part_rows", "row_part_rows", "item_part_rows", "table_at",
        "slots_at", "pages_at", "row_tiles_at", "row_starts_at", "tile_items_at", "joins_at")] + [("seal", ctypes.c_uint64), ("device", ctypes.c_int64)]


class KvmCache(ctypes.Structure):
    """One layer of a K/V pool pair."""

    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p)] + [(name, ctypes.c_int64) for name in (
        "num_blocks", "num_layers", "layer", "num_kv_heads", "block_size", "head_dim")] + [
        ("dtype", ctypes.c_int32), ("format", ctypes.c_int32), ("extent", ctypes.c_int64)]


class KvmRows(ctypes.Structure):
    """Rows [tokens][heads][head_dim] by base pointer and strides in elements."""

    _fields_ = [("ptr", ctypes.c_void_p), ("token_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64),
                ("extent", ctypes.c_int64)]


def _lib_path() -> str:
    lib_dir = os.environ.get("KVMOVE_LIB_DIR") or os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib")
    return os.path.join(lib_dir, "libkvmove.so")


def _load(path: str) -> ctypes.CDLL:
    if not os.path.exists(path):
        raise RuntimeError(f"{os.path.basename(path)} not found at {path}; build it with "
                           "`python distserve_amd/csrc/build.py`")
    lib = ctypes.CDLL(path)
    i64, i32, vp, ip = ctypes.c_int64, ctypes.c_int32, ctypes.c_void_p, ctypes.POINTER(ctypes.c_int64)
    lib.kvm_version.restype = ctypes.c_int
    lib.kvm_last_error.restype = ctypes.c_char_p
    # the shapes bound below are those of one major version; any other must not be called
    if lib.kvm_version() // 10000 != KVM_ABI_MAJOR:
        raise RuntimeError(f"{path} is kvmove version {lib.kvm_version()}; this binding is written for major "
                           f"version {KVM_ABI_MAJOR}")
    lib.kvm_get_mem_handle.argtypes = [vp, i64, ip]
    lib.kvm_register_mem_handle.argtypes = [ip, ip, i64, i64, ip, ip, i64]
    lib.kvm_register_source.argtypes = [i32, i32, i32, i32, i64, i64, vp, vp, i64, i64]
    lib.kvm_reset.argtypes = []
    lib.kvm_opened_handles.argtypes = []
    lib.kvm_opened_handles.restype = i64
    lib.kvm_migrate.argtypes = [ctypes.POINTER(KvmGeom), ip, ip, i64, vp, vp, i64, vp]
    lib.kvm_swap.argtypes = [ip, ip, i64, ctypes.c_int, vp, vp, vp, vp, i64, i64, i64, vp]
    lib.kvm_copy_plain.argtypes = [vp, vp, i64, vp]
    lib.kvm_set_option.argtypes = [ctypes.c_char_p, i64]
    lib.kvm_get_option.argtypes = [ctypes.c_char_p]
    lib.kvm_get_option.restype = i64
    lib.kvm_migrate_plan.argtypes = [ctypes.POINTER(KvmGeom), i64, vp, vp, i64, ip]
    lib.kvm_swap_plan.argtypes = [ip, ip, i64, i64, ctypes.c_int, i64, i64, ip]
    lib.kvm_debug_divide.argtypes = [ctypes.c_uint32, ctypes.c_uint32]
    lib.kvm_debug_divide.restype = ctypes.c_uint32
    i32p, f32 = ctypes.POINTER(ctypes.c_int32), ctypes.c_float
    step, cache, rows = ctypes.POINTER(KvmStep), ctypes.POINTER(KvmCache), ctypes.POINTER(KvmRows)
    lib.kvm_plan_words.argtypes = [i64] * 5
    lib.kvm_plan_words.restype = i64
    lib.kvm_plan_step.argtypes = [ip, ip, i64, ip, ip, i64, i64, i64, i64, i64, i32, i32, i32p, i64, step]
    lib.kvm_write_kv.argtypes = [step, vp, cache, rows, rows, vp]
    lib.kvm_read_kv.argtypes = [step, vp, cache, rows, rows, vp]
    lib.kvm_attention_workspace.argtypes = [step]
    lib.kvm_attention_workspace.restype = i64
    lib.kvm_paged_attention.argtypes = [step, vp, cache, rows, rows, f32, vp, i64, vp]
    lib.kvm_prompt_attention.argtypes = [step, vp, rows, rows, rows, rows, f32, vp, i64, vp]
    for name in EXPORTS:
        fn = getattr(lib, name)
        if name not in ("kvm_last_error", "kvm_get_option", "kvm_version", "kvm_debug_divide",
                        "kvm_opened_handles", "kvm_plan_words", "kvm_attention_workspace"):
            fn.restype = ctypes.c_int
    return lib


def _arr(values: Sequence[int]):
    if isinstance(values, ctypes.Array):
        return values
    return (ctypes.c_int64 * len(values))(*values)


def index_array(values: Sequence[int]):
    """A block-index list converted once, for callers that reuse it across calls."""
    return _arr(list(values))


def geom(num_layers, num_kv_heads, block_size, head_dim, dtype_bytes, ctx_pp=1, ctx_tp=1,
         dec_pp=1, dec_tp=1, dec_pp_rank=0, dec_tp_rank=0, ctx_instance=0) -> KvmGeom:
    return KvmGeom(num_layers, num_kv_heads, block_size, head_dim, dtype_bytes,
                   ctx_pp, ctx_tp, dec_pp, dec_tp, dec_pp_rank, dec_tp_rank, ctx_instance)


class Binding:
    """One loaded build of the library.  Every build has its own registry of context pools
    and its own options."""

    # names a caller may want beside the functions, so that a Binding can stand in for this module
    KvmError, KvmGeom = KvmError, KvmGeom
    KVM_OK, KVM_EINVAL, KVM_ERANGE, KVM_EDUP, KVM_ENOTREG = KVM_OK, KVM_EINVAL, KVM_ERANGE, KVM_EDUP, KVM_ENOTREG
    KVM_EHIP, KVM_EHANDLE, KVM_EMISMATCH = KVM_EHIP, KVM_EHANDLE, KVM_EMISMATCH
    KVM_HANDLE_WORDS, KVM_IPC_MAX_ALLOC_BYTES, EXPORTS = KVM_HANDLE_WORDS, KVM_IPC_MAX_ALLOC_BYTES, EXPORTS
    geom, index_array = staticmethod(geom), staticmethod(index_array)

    def __init__(self, path: str):
        self.path = path
        self.lib = _load(path)

    def _check(self, rc: int) -> None:
        if rc != KVM_OK:
            raise KvmError(rc, self.lib.kvm_last_error().decode())

    def version(self) -> int:
        return self.lib.kvm_version()

    def get_mem_handle(self, dev_ptr: int, nbytes: int) -> List[int]:
        out = (ctypes.c_int64 * KVM_HANDLE_WORDS)()
        self._check(self.lib.kvm_get_mem_handle(dev_ptr, nbytes, out))
        return list(out)

    def register_mem_handle(self, k_handle, v_handle, num_layers, num_kv_heads, context_pc, decoding_pc,
                            ctx_instance: int = 0) -> None:
        if len(k_handle) != KVM_HANDLE_WORDS or len(v_handle) != KVM_HANDLE_WORDS:
            raise KvmError(KVM_EHANDLE, f"a memory handle has {KVM_HANDLE_WORDS} words")
        if len(context_pc) != 4 or len(decoding_pc) != 4:
            raise KvmError(KVM_EINVAL, "parallel configs are [tp_size, tp_rank, pp_size, pp_rank]")
        self._check(self.lib.kvm_register_mem_handle(_arr(k_handle), _arr(v_handle), num_layers, num_kv_heads,
                                                     _arr(context_pc), _arr(decoding_pc), ctx_instance))

    def register_source(self, ctx_pp_size, ctx_tp_size, pp_rank, tp_rank, num_layers, num_kv_heads,
                        k_ptr: int, v_ptr: int, nbytes_each: int, ctx_instance: int = 0) -> None:
        self._check(self.lib.kvm_register_source(ctx_pp_size, ctx_tp_size, pp_rank, tp_rank, num_layers,
                                                 num_kv_heads, k_ptr, v_ptr, nbytes_each, ctx_instance))

    def reset(self) -> None:
        self._check(self.lib.kvm_reset())

    def opened_handles(self) -> int:
        """Allocations of other processes that registration currently keeps mapped."""
        return self.lib.kvm_opened_handles()

    def migrate(self, g: KvmGeom, ctx_idx: Sequence[int], dec_idx: Sequence[int], dst_k: int, dst_v: int,
                dst_num_blocks: int, stream: int = 0, n: int | None = None) -> None:
        n = len(ctx_idx) if n is None else n
        if n == len(ctx_idx) and len(ctx_idx) != len(dec_idx):
            raise KvmError(KVM_EINVAL, f"{len(ctx_idx)} context blocks but {len(dec_idx)} decoding blocks")
        self._check(self.lib.kvm_migrate(ctypes.byref(g), _arr(ctx_idx), _arr(dec_idx), n, dst_k, dst_v,
                                         dst_num_blocks, stream))

    def swap(self, src_ids: Sequence[int], dst_ids: Sequence[int], is_swap_in: bool, k_gpu: int, v_gpu: int,
             k_host: int, v_host: int, slab_bytes: int, n_gpu_blocks: int, n_host_blocks: int,
             stream: int = 0) -> None:
        if len(src_ids) != len(dst_ids):
            raise KvmError(KVM_EINVAL, f"{len(src_ids)} source blocks but {len(dst_ids)} target blocks")
        self._check(self.lib.kvm_swap(_arr(src_ids), _arr(dst_ids), len(src_ids), 1 if is_swap_in else 0, k_gpu,
                                      v_gpu, k_host, v_host, slab_bytes, n_gpu_blocks, n_host_blocks, stream))

    def copy_plain(self, dst: int, src: int, nbytes: int, stream: int = 0) -> None:
        self._check(self.lib.kvm_copy_plain(dst, src, nbytes, stream))

    def set_option(self, name: str, value: int) -> None:
        self._check(self.lib.kvm_set_option(name.encode(), value))

    def get_option(self, name: str) -> int:
        v = self.lib.kvm_get_option(name.encode())
        if v == KVM_EINVAL and self.lib.kvm_last_error():
            raise KvmError(KVM_EINVAL, self.lib.kvm_last_error().decode())
        return v

    def swap_plan(self, src_ids: Sequence[int], dst_ids: Sequence[int], slab_bytes: int, is_swap_in: bool = False,
                  n_gpu_blocks: int = 0, n_host_blocks: int = 0) -> dict:
        if len(src_ids) != len(dst_ids):
            raise KvmError(KVM_EINVAL, f"{len(src_ids)} source blocks but {len(dst_ids)} target blocks")
        out = (ctypes.c_int64 * 4)()
        self._check(self.lib.kvm_swap_plan(_arr(src_ids), _arr(dst_ids), len(src_ids), slab_bytes,
                                           1 if is_swap_in else 0, n_gpu_blocks, n_host_blocks, out))
        return dict(zip(("mode", "copies_per_pool", "launches", "workgroups_per_pool_kind"), list(out)))

    def migrate_plan(self, g: KvmGeom, n: int, dst_k: int, dst_v: int, dst_num_blocks: int = 0) -> dict:
        out = (ctypes.c_int64 * 10)()
        self._check(self.lib.kvm_migrate_plan(ctypes.byref(g), n, dst_k, dst_v, dst_num_blocks, out))
        keys = ("workgroups_per_block", "threads", "vector_bytes", "segments", "launches",
                "payload_bytes_per_block", "simple_kernel", "max_work_items", "vectors_per_lane",
                "pairs_per_launch")
        return dict(zip(keys, list(out)))

    def debug_divide(self, n: int, d: int) -> int:
        return self.lib.kvm_debug_divide(n, d)

    # ---- cache operators

    def plan_step(self, first_token: Sequence[int], new_tokens: Sequence[int], block_table: Sequence[Sequence[int]],
                  num_blocks: int, block_size: int, num_heads: int, num_kv_heads: int, head_dim: int, dtype: int,
                  format: int = KVM_CACHE_PLAIN):
        """(KvmStep, the plan's words as a ctypes array): the words go to device memory as they are.
        ``num_blocks == 0``: a plan without a cache, ``block_table`` is ignored."""
        n = len(first_token)
        if len(new_tokens) != n or (num_blocks and len(block_table) != n):
            raise KvmError(KVM_EINVAL, f"{n} first tokens, {len(new_tokens)} lengths and {len(block_table)} block tables")
        tables = block_table if num_blocks else []
        flat = [block for table in tables for block in table]
        room = self.lib.kvm_plan_words(n, max(0, sum(new_tokens)), len(flat), num_heads, num_kv_heads)
        words = (ctypes.c_int32 * max(room, 64))()
        step = KvmStep()
        self._check(self.lib.kvm_plan_step(_arr(first_token), _arr(new_tokens), n, _arr(flat), _arr([len(t) for t in tables]),
                                           num_blocks, block_size, num_heads, num_kv_heads, head_dim, dtype, format,
                                           words, len(words), ctypes.byref(step)))
        return step, words

    def write_kv(self, step: KvmStep, words: int, cache: KvmCache, k: KvmRows, v: KvmRows, stream: int = 0) -> None:
        self._check(self.lib.kvm_write_kv(ctypes.byref(step), words, ctypes.byref(cache), ctypes.byref(k),
                                          ctypes.byref(v), stream))

    def read_kv(self, step: KvmStep, words: int, cache: KvmCache, k_out: KvmRows, v_out: KvmRows,
                stream: int = 0) -> None:
        self._check(self.lib.kvm_read_kv(ctypes.byref(step), words, ctypes.byref(cache), ctypes.byref(k_out),
                                         ctypes.byref(v_out), stream))

    def attention_workspace(self, step: KvmStep) -> int:
        need = self.lib.kvm_attention_workspace(ctypes.byref(step))
        if need < 0:
            self._check(need)
        return need

    def paged_attention(self, step: KvmStep, words: int, cache: KvmCache, q: KvmRows, out: KvmRows, scale: float,
                        workspace: int = 0, workspace_bytes: int = 0, stream: int = 0) -> None:
        self._check(self.lib.kvm_paged_attention(ctypes.byref(step), words, ctypes.byref(cache), ctypes.byref(q),
                                                 ctypes.byref(out), scale, workspace, workspace_bytes, stream))

    def prompt_attention(self, step: KvmStep, words: int, q: KvmRows, k: KvmRows, v: KvmRows, out: KvmRows,
                         scale: float, workspace: int = 0, workspace_bytes: int = 0, stream: int = 0) -> None:
        self._check(self.lib.kvm_prompt_attention(ctypes.byref(step), words, ctypes.byref(q), ctypes.byref(k),
                                                  ctypes.byref(v), ctypes.byref(out), scale, workspace,
                                                  workspace_bytes, stream))


default = Binding(_lib_path())
lib = default.lib

version = default.version
get_mem_handle = default.get_mem_handle
register_mem_handle = default.register_mem_handle
register_source = default.register_source
reset = default.reset
opened_handles = default.opened_handles
migrate = default.migrate
swap = default.swap
copy_plain = default.copy_plain
set_option = default.set_option
get_option = default.get_option
swap_plan = default.swap_plan
migrate_plan = default.migrate_plan
debug_divide = default.debug_divide
plan_step = default.plan_step
write_kv = default.write_kv
read_kv = default.read_kv
attention_workspace = default.attention_workspace
paged_attention = default.paged_attention
prompt_attention = default.prompt_attention
