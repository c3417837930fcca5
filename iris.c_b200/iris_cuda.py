"""ctypes binding of libiris_cuda.so (the C ABI declared in include/iris_cuda.h).

Used by the tests, bench.py and __graft_entry__.py.  It loads the in-tree
library built by ``make -C iris.c_b200 cuda`` and fails loudly when it is
missing: there is no CPU or framework fallback behind these calls.
"""
from __future__ import annotations

import ctypes as C
import os
import weakref

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libiris_cuda.so")

OK = 0
ERR_ARG, ERR_OOM, ERR_CUDA, ERR_IO, ERR_TIMEOUT, ERR_NODEV, ERR_INJECTED = -1, -2, -3, -4, -5, -6, -7

_fp = C.POINTER(C.c_float)
_u16p = C.POINTER(C.c_uint16)


class FluxConfig(C.Structure):
    _fields_ = [("hidden", C.c_int), ("heads", C.c_int), ("head_dim", C.c_int), ("mlp", C.c_int),
                ("n_double", C.c_int), ("n_single", C.c_int), ("text_dim", C.c_int),
                ("channels", C.c_int), ("rope_theta", C.c_float)]

    @classmethod
    def from_hf(cls, cfg: dict) -> "FluxConfig":
        h = cfg["num_attention_heads"] * cfg["attention_head_dim"]
        return cls(hidden=h, heads=cfg["num_attention_heads"], head_dim=cfg["attention_head_dim"],
                   mlp=int(h * cfg.get("mlp_ratio", 3.0)), n_double=cfg["num_layers"],
                   n_single=cfg["num_single_layers"], text_dim=cfg["joint_attention_dim"],
                   channels=cfg["in_channels"], rope_theta=float(cfg.get("rope_theta", 2000.0)))


class KernelTime(C.Structure):
    _fields_ = [("name", C.c_char * 32), ("flops", C.c_double), ("bytes", C.c_double), ("ms", C.c_float)]


class ZImageConfig(C.Structure):
    _fields_ = [("dim", C.c_int), ("heads", C.c_int), ("n_layers", C.c_int), ("n_refiner", C.c_int),
                ("cap_feat_dim", C.c_int), ("in_channels", C.c_int), ("patch_size", C.c_int),
                ("ffn_dim", C.c_int), ("adaln_dim", C.c_int), ("t_mid", C.c_int), ("rope_theta", C.c_float),
                ("axes_dims", C.c_int * 3)]

    @classmethod
    def from_dict(cls, c: dict) -> "ZImageConfig":
        return cls(dim=c["dim"], heads=c["dim"] // 128, n_layers=c["n_layers"], n_refiner=c["n_refiner"],
                   cap_feat_dim=c["cap_feat_dim"], in_channels=c["in_channels"], patch_size=c["patch_size"],
                   ffn_dim=c["ffn_dim"], adaln_dim=min(c["dim"], 256), t_mid=c["t_mid"],
                   rope_theta=float(c["rope_theta"]), axes_dims=(C.c_int * 3)(*c["axes_dims"]))


class Qwen3Config(C.Structure):
    """iris_cuda_qwen3_config_t."""
    _fields_ = [("hidden", C.c_int), ("intermediate", C.c_int), ("heads", C.c_int), ("kv_heads", C.c_int),
                ("head_dim", C.c_int), ("vocab", C.c_int), ("layers", C.c_int), ("rope_theta", C.c_float)]

    @classmethod
    def from_hf(cls, c: dict) -> "Qwen3Config":
        return cls(c["hidden_size"], c["intermediate_size"], c["num_attention_heads"], c["num_key_value_heads"],
                   c.get("head_dim", 128), c["vocab_size"], c["num_hidden_layers"], c.get("rope_theta", 1e6))


class Image(C.Structure):
    """iris_cuda_image_t (the reference's iris_image layout, iris.h:73-78)."""
    _fields_ = [("width", C.c_int), ("height", C.c_int), ("channels", C.c_int),
                ("data", C.POINTER(C.c_uint8))]


class Ref(C.Structure):
    _fields_ = [("latent", _fp), ("h", C.c_int), ("w", C.c_int), ("t_offset", C.c_int)]


class RopeScaling(C.Structure):
    """iris_gpu_rope_scaling_t."""
    _fields_ = [("factor", C.c_double), ("original_len", C.c_double), ("low", C.c_double), ("high", C.c_double),
                ("amplitude", C.c_double)]


class Rope(C.Structure):
    """iris_gpu_rope_t: a rotation of the first rot_dim columns of each head."""
    _fields_ = [("layout", C.c_int), ("rot_dim", C.c_int), ("amplitude", C.c_float), ("turns", C.c_uint64 * 128)]

    @classmethod
    def of(cls, rot_dim: int, theta: float, interleaved: bool = False, factor: float = 1.0, original_len: float = 0.0,
           low: float = 1.0, high: float = 32.0, amplitude: float = 1.0) -> "Rope":
        """Frequencies theta^(-2i / rot_dim), scaled for long contexts (iris_gpu_rope_scaling_t)."""
        r = cls()
        sc = RopeScaling(factor, original_len, low, high, amplitude)
        _ok(lib().iris_gpu_rope_init(C.byref(r), int(interleaved), rot_dim, theta, C.byref(sc)))
        return r

    @classmethod
    def of_freqs(cls, freqs, interleaved: bool = False, amplitude: float = 1.0) -> "Rope":
        """Frequencies of the caller's own [rot_dim / 2], radians per position."""
        r = cls()
        f = np.ascontiguousarray(freqs, np.float64)
        _ok(lib().iris_gpu_rope_init_freqs(C.byref(r), int(interleaved), 2 * f.size,
                                           f.ctypes.data_as(C.POINTER(C.c_double)), amplitude))
        return r


class KvCache(C.Structure):
    """iris_gpu_kv_cache_t: a paged key-value cache over the caller's own pools."""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("table", C.c_void_p), ("num_pages", C.c_int),
                ("page_size", C.c_int), ("kv_heads", C.c_int), ("head_dim", C.c_int), ("num_seqs", C.c_int),
                ("max_blocks", C.c_int), ("table_stride", C.c_int64), ("page_stride", C.c_int64),
                ("token_stride", C.c_int64), ("head_stride", C.c_int64)]

    @classmethod
    def of(cls, k, v, table) -> "KvCache":
        """k, v: bf16 device tensors seen as [pages, slots, heads, columns] (any order of
        slots and heads in memory, columns contiguous, both laid out alike); table:
        int32 [sequences, blocks].  The tensors are kept alive."""
        if _dtype(k) != "bfloat16" or _dtype(v) != "bfloat16" or _dtype(table) != "int32":
            raise IrisCudaError("KvCache: pools are bfloat16, the page table int32")
        c = _pages("KvCache", k, v, table)
        c.tensors = (k, v, table)
        return c


def _pages(what: str, k, v, table) -> KvCache:
    """The pools' and the table's description."""
    if len(k.shape) != 4 or tuple(k.shape) != tuple(v.shape) or \
            any(n > 1 and a != b for n, a, b in zip(k.shape, k.stride(), v.stride())):
        raise IrisCudaError(f"{what}: pools [pages, slots, heads, columns] laid out alike")
    if k.stride(3) != 1 or len(table.shape) != 2 or table.stride(1) != 1:
        raise IrisCudaError(f"{what}: columns and table rows are contiguous")
    stride = [s if n > 1 else 0 for n, s in zip(k.shape, k.stride())]  # of an axis of one: never used
    return KvCache(k.data_ptr(), v.data_ptr(), table.data_ptr(), *k.shape, *table.shape, table.stride(0), *stride[:3])


class KvCache8(C.Structure):
    """iris_gpu_kv_cache8_t: the same in 8 bits, with an exponent for each block of tokens and head."""
    _fields_ = [("pages", KvCache), ("k_exp", C.c_void_p), ("v_exp", C.c_void_p), ("block", C.c_int),
                ("exp_page_stride", C.c_int64), ("exp_block_stride", C.c_int64), ("exp_head_stride", C.c_int64)]

    @classmethod
    def of(cls, k, v, k_exp, v_exp, table) -> "KvCache8":
        """k, v: float8_e4m3fn (or uint8) device tensors as KvCache.of takes them; k_exp, v_exp: uint8 [pages, blocks
        of a page, heads], laid out alike; table: int32 [sequences, blocks].  The tensors are kept alive."""
        if any(_dtype(t) not in ("float8_e4m3fn", "uint8") for t in (k, v)) or _dtype(table) != "int32" or \
                _dtype(k_exp) != "uint8" or _dtype(v_exp) != "uint8":
            raise IrisCudaError("KvCache8: pools are float8_e4m3fn, exponents uint8, the page table int32")
        c = cls(_pages("KvCache8", k, v, table))
        pages, slots, heads = k.shape[:3]
        if len(k_exp.shape) != 3 or tuple(k_exp.shape) != tuple(v_exp.shape) or k_exp.shape[0] != pages or \
                k_exp.shape[2] != heads or not k_exp.shape[1] or slots % k_exp.shape[1] or \
                any(n > 1 and a != b for n, a, b in zip(k_exp.shape, k_exp.stride(), v_exp.stride())):
            raise IrisCudaError("KvCache8: exponents [pages, blocks of a page, heads] laid out alike")
        c.k_exp, c.v_exp, c.block = k_exp.data_ptr(), v_exp.data_ptr(), slots // k_exp.shape[1]
        c.exp_page_stride, c.exp_block_stride, c.exp_head_stride = (
            s if n > 1 else 0 for n, s in zip(k_exp.shape, k_exp.stride()))
        c.tensors = (k, v, k_exp, v_exp, table)
        c.head_dim, c.kv_heads = c.pages.head_dim, c.pages.kv_heads
        return c


class Weights4(C.Structure):
    """iris_gpu_weights4_t: weights of 4 bits with a scale for each group of columns."""
    _fields_ = [("q", C.c_void_p), ("scale", C.c_void_p), ("zero", C.c_void_p), ("n", C.c_int), ("k", C.c_int),
                ("group", C.c_int), ("scale_f32", C.c_int), ("q_stride", C.c_int64), ("scale_stride", C.c_int64),
                ("zero_stride", C.c_int64)]

    @classmethod
    def of(cls, q, scale, zero=None) -> "Weights4":
        """q: uint8 [n, k / 2], two columns a byte, the low half first; scale: bfloat16 or float32 [n, groups]; zero:
        uint8 [n, groups], or None: 8.  The tensors are kept alive."""
        if _dtype(q) != "uint8" or _dtype(scale) not in ("bfloat16", "float32") or (zero is not None and _dtype(zero) != "uint8"):
            raise IrisCudaError("Weights4: weights are uint8, scales bfloat16 or float32, zeros uint8")
        if len(q.shape) != 2 or len(scale.shape) != 2 or scale.shape[0] != q.shape[0] or not scale.shape[1] or \
                2 * q.shape[1] % scale.shape[1] or (zero is not None and tuple(zero.shape) != tuple(scale.shape)):
            raise IrisCudaError("Weights4: weights [n, k / 2], scales and zeros [n, groups]")
        if any(t is not None and t.shape[1] > 1 and t.stride(1) != 1 for t in (q, scale, zero)):
            raise IrisCudaError("Weights4: rows are contiguous")
        n, k = q.shape[0], 2 * q.shape[1]
        c = cls(q.data_ptr(), scale.data_ptr(), None if zero is None else zero.data_ptr(), n, k, k // scale.shape[1],
                _dtype(scale) == "float32", *(0 if t is None or n == 1 else t.stride(0) for t in (q, scale, zero)))
        c.tensors = (q, scale, zero)
        return c


PROGRESS_CB = C.CFUNCTYPE(None, C.c_int, C.c_int)

# name -> (restype, argtypes) for every exported entry point of include/iris_cuda.h
SIGNATURES = {
    "iris_cuda_init": (C.c_int, [C.c_int]),
    "iris_cuda_available": (C.c_int, []),
    "iris_cuda_cleanup": (None, []),
    "iris_cuda_last_error": (C.c_char_p, []),
    "iris_cuda_device_status": (C.c_int, [C.c_int]),
    "iris_cuda_synchronize": (C.c_int, []),
    "iris_cuda_stream": (C.c_void_p, []),
    "iris_cuda_kernel_launches": (C.c_uint64, []),
    "iris_cuda_selftest_wait_timeout": (C.c_int, []),
    "iris_cuda_flux_load": (C.c_void_p, [C.c_char_p]),
    "iris_cuda_flux_random": (C.c_void_p, [C.POINTER(FluxConfig), C.c_uint64, C.c_float, C.c_int]),
    "iris_cuda_flux_load_tp": (C.c_void_p, [C.c_char_p, C.c_int, C.c_int]),
    "iris_cuda_flux_random_tp": (C.c_void_p, [C.POINTER(FluxConfig), C.c_uint64, C.c_float, C.c_int,
                                              C.c_int, C.c_int]),
    "iris_cuda_flux_free": (None, [C.c_void_p]),
    "iris_cuda_flux_get_config": (C.c_int, [C.c_void_p, C.POINTER(FluxConfig)]),
    "iris_cuda_flux_read_weight": (C.c_int, [C.c_void_p, C.c_char_p, _u16p, C.c_size_t]),
    "iris_cuda_flux_weight_bytes": (C.c_size_t, [C.c_void_p]),
    "iris_cuda_flux_load_lora": (C.c_int, [C.c_void_p, C.c_char_p, C.c_float]),
    "iris_cuda_flux_unload_lora": (C.c_int, [C.c_void_p]),
    "iris_cuda_flux_lora_adapters": (C.c_int, [C.c_void_p]),
    "iris_cuda_flux_lora_stats": (C.c_int, [C.c_void_p, C.POINTER(C.c_double), C.POINTER(C.c_double)]),
    "iris_cuda_lora_probe": (C.c_int, [C.c_char_p, C.c_int, C.c_int, C.c_int, C.c_int, C.POINTER(C.c_int)]),
    "iris_cuda_flux_load_ip_adapter": (C.c_int, [C.c_void_p, C.c_char_p, C.c_char_p, C.c_float]),
    "iris_cuda_flux_load_ip_adapter_mem": (C.c_int, [C.c_void_p, C.c_char_p, _fp, C.c_int, C.c_float]),
    "iris_cuda_flux_unload_ip_adapter": (C.c_int, [C.c_void_p]),
    "iris_cuda_flux_set_ip_schedule": (C.c_int, [C.c_void_p, C.c_char_p]),
    "iris_cuda_flux_set_ip_step": (C.c_int, [C.c_void_p, C.c_int, C.c_int]),
    "iris_cuda_flux_ip_embeds": (C.c_int, [C.c_void_p, _fp, C.c_int]),
    "iris_cuda_flux_set_sref_csd": (C.c_int, [C.c_void_p, C.c_char_p, _fp, C.c_int, C.c_float]),
    "iris_cuda_flux_set_csd_delta": (C.c_int, [C.c_void_p, _fp]),
    "iris_cuda_flux_set_csd_skip": (C.c_int, [C.c_void_p, C.c_int]),
    "iris_cuda_flux_set_sref_bands": (C.c_int, [C.c_void_p, C.c_float, C.c_float]),
    "iris_cuda_transformer_forward": (C.c_void_p, [C.c_void_p, _fp, C.c_int, C.c_int, _fp, C.c_int,
                                                   C.c_float]),
    "iris_cuda_transformer_forward_with_multi_refs": (C.c_void_p, [C.c_void_p, _fp, C.c_int, C.c_int,
                                                                   C.POINTER(Ref), C.c_int, _fp,
                                                                   C.c_int, C.c_float]),
    "iris_cuda_flux_forward_dev": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int, C.c_int,
                                             C.POINTER(Ref), C.c_int, C.c_void_p, C.c_int,
                                             C.c_float, C.c_void_p]),
    "iris_cuda_flux_run_block": (C.c_int, [C.c_void_p, C.c_int, C.c_int, _fp, C.c_int, C.c_int,
                                           C.c_int, C.c_float]),
    "iris_cuda_flux_profile": (C.c_int, [C.c_void_p, C.c_float, C.POINTER(KernelTime), C.c_int]),
    "iris_cuda_official_schedule": (C.c_void_p, [C.c_int, C.c_int]),
    "iris_cuda_linear_schedule": (C.c_void_p, [C.c_int]),
    "iris_cuda_zimage_schedule": (C.c_void_p, [C.c_int, C.c_int]),
    "iris_cuda_init_noise": (C.c_void_p, [C.c_int, C.c_int, C.c_int, C.c_int, C.c_int64]),
    "iris_cuda_sample_euler": (C.c_void_p, [C.c_void_p, _fp, C.c_int, C.c_int, C.c_int, C.c_int,
                                            _fp, C.c_int, _fp, C.c_int, PROGRESS_CB]),
    "iris_cuda_sample_euler_cfg": (C.c_void_p, [C.c_void_p, _fp, C.c_int, C.c_int, C.c_int, C.c_int,
                                                _fp, C.c_int, _fp, C.c_int, C.c_float, _fp, C.c_int,
                                                PROGRESS_CB]),
    "iris_cuda_sample_euler_with_multi_refs": (C.c_void_p, [C.c_void_p, _fp, C.c_int, C.c_int,
                                                            C.c_int, C.c_int, C.POINTER(Ref), C.c_int,
                                                            _fp, C.c_int, _fp, C.c_int, PROGRESS_CB]),
    "iris_cuda_sample_euler_dev": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_void_p,
                                             C.c_int, C.c_void_p, C.c_int, C.c_float, _fp, C.c_int]),
    "iris_cuda_comm_unique_id": (C.c_int, [C.c_void_p, C.c_size_t]),
    "iris_cuda_comm_init": (C.c_int, [C.c_void_p, C.c_int, C.c_int]),
    "iris_cuda_comm_destroy": (None, []),
    "iris_cuda_comm_world": (C.c_int, []),
    "iris_cuda_comm_rank": (C.c_int, []),
    "iris_cuda_sample_euler_cfg_pair": (C.c_void_p, [C.c_void_p, _fp, C.c_int, C.c_int, C.c_int, C.c_int,
                                                     _fp, C.c_int, _fp, C.c_int, C.c_float, _fp, C.c_int,
                                                     PROGRESS_CB]),
    "iris_cuda_sample_euler_cfg_pair_dev": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int, C.c_int,
                                                      C.c_void_p, C.c_void_p, C.c_int, C.c_float, _fp,
                                                      C.c_int]),
    "iris_cuda_zimage_load": (C.c_void_p, [C.c_char_p]),
    "iris_cuda_zimage_random": (C.c_void_p, [C.POINTER(ZImageConfig), C.c_uint64, C.c_float, C.c_int]),
    "iris_cuda_zimage_free": (None, [C.c_void_p]),
    "iris_cuda_zimage_get_config": (C.c_int, [C.c_void_p, C.POINTER(ZImageConfig)]),
    "iris_cuda_zimage_weight_bytes": (C.c_size_t, [C.c_void_p]),
    "iris_cuda_zi_transformer_forward": (C.c_void_p, [C.c_void_p, _fp, C.c_int, C.c_int, C.c_float, _fp,
                                                      C.c_int]),
    "iris_cuda_sample_euler_zimage": (C.c_void_p, [C.c_void_p, _fp, C.c_int, C.c_int, C.c_int, C.c_int,
                                                   C.c_int, _fp, C.c_int, _fp, C.c_int, PROGRESS_CB]),
    "iris_cuda_sample_euler_zimage_dev": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_void_p,
                                                    C.c_int, _fp, C.c_int]),
    "iris_cuda_vae_load": (C.c_void_p, [C.c_char_p, C.c_int, C.c_float, C.c_float]),
    "iris_cuda_vae_free": (None, [C.c_void_p]),
    "iris_cuda_vae_weight_bytes": (C.c_size_t, [C.c_void_p]),
    "iris_cuda_vae_decode": (C.c_void_p, [C.c_void_p, _fp, C.c_int, C.c_int, C.c_int]),
    "iris_cuda_image_free": (None, [C.c_void_p]),
    "iris_cuda_vae_decode_f32": (C.c_int, [C.c_void_p, _fp, C.c_int, C.c_int, _fp]),
    "iris_cuda_vae_decode_dev": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_void_p,
                                           C.c_void_p]),
    "iris_cuda_vae_graph_kernels": (C.c_uint64, [C.c_void_p]),
    "iris_cuda_vae_random": (C.c_void_p, [C.c_int, C.c_float, C.c_float, C.c_uint64]),
    "iris_cuda_qwen3_load": (C.c_void_p, [C.c_char_p]),
    "iris_cuda_qwen3_random": (C.c_void_p, [C.POINTER(Qwen3Config), C.c_uint64]),
    "iris_cuda_qwen3_free": (None, [C.c_void_p]),
    "iris_cuda_qwen3_get_config": (C.c_int, [C.c_void_p, C.POINTER(Qwen3Config)]),
    "iris_cuda_qwen3_weight_bytes": (C.c_size_t, [C.c_void_p]),
    "iris_cuda_qwen3_set_extraction_mode": (C.c_int, [C.c_void_p, C.c_int]),
    "iris_cuda_qwen3_text_dim": (C.c_int, [C.c_void_p]),
    "iris_cuda_qwen3_forward": (C.c_void_p, [C.c_void_p, C.POINTER(C.c_int), C.POINTER(C.c_int), C.c_int]),
    "iris_cuda_qwen3_forward_dev": (C.c_int, [C.c_void_p, C.POINTER(C.c_int), C.POINTER(C.c_int), C.c_int,
                                              C.c_void_p]),
    "iris_cuda_qwen3_load_lm": (C.c_void_p, [C.c_char_p]),
    "iris_cuda_qwen3_random_lm": (C.c_void_p, [C.POINTER(Qwen3Config), C.c_uint64]),
    "iris_cuda_qwen3_lm_create": (C.c_void_p, [C.c_void_p, C.c_int, C.c_int, C.c_int]),
    "iris_cuda_qwen3_lm_free": (None, [C.c_void_p]),
    "iris_cuda_qwen3_lm_cache_bytes": (C.c_size_t, [C.c_void_p]),
    "iris_cuda_qwen3_lm_step": (C.c_int, [C.c_void_p] + [C.POINTER(C.c_int)] * 4 + [C.c_int, C.c_int, _fp, _fp,
                                                                                  C.POINTER(C.c_int), _fp]),
    "iris_cuda_qwen3_lm_sample": (C.c_int, [C.c_void_p] + [C.POINTER(C.c_int)] * 3 + [C.c_int, _fp, C.POINTER(C.c_int), _fp, _fp,
                                            C.POINTER(C.c_double), C.POINTER(C.c_int), _fp]),
    "iris_cuda_qwen3_lm_length": (C.c_int, [C.c_void_p, C.c_int]),
    "iris_cuda_qwen3_graph_kernels": (C.c_uint64, [C.c_void_p]),
    "iris_cuda_qwen3_profile": (C.c_int, [C.c_void_p, C.POINTER(KernelTime), C.c_int]),
    "iris_cuda_vae_profile": (C.c_int, [C.c_void_p, C.POINTER(KernelTime), C.c_int]),
    # iris_gpu_* surface (iris_metal.h names)
    "iris_gpu_tensor_create": (C.c_void_p, [_fp, C.c_size_t]),
    "iris_gpu_tensor_alloc": (C.c_void_p, [C.c_size_t]),
    "iris_gpu_tensor_alloc_persistent": (C.c_void_p, [C.c_size_t]),
    "iris_gpu_tensor_set_persistent": (None, [C.c_void_p, C.c_int]),
    "iris_gpu_tensor_read": (None, [C.c_void_p, _fp]),
    "iris_gpu_tensor_write": (None, [C.c_void_p, _fp]),
    "iris_gpu_tensor_free": (None, [C.c_void_p]),
    "iris_gpu_tensor_size": (C.c_size_t, [C.c_void_p]),
    "iris_gpu_tensor_is_f16": (C.c_int, [C.c_void_p]),
    "iris_gpu_tensor_alloc_f16": (C.c_void_p, [C.c_size_t]),
    "iris_gpu_tensor_create_bf16": (C.c_void_p, [_fp, C.c_size_t]),
    "iris_gpu_tensor_f32_to_bf16": (C.c_void_p, [C.c_void_p]),
    "iris_gpu_tensor_bf16_to_f32": (C.c_void_p, [C.c_void_p]),
    "iris_gpu_convert_f32_to_bf16_into": (C.c_int, [C.c_void_p, C.c_void_p]),
    "iris_gpu_convert_bf16_to_f32_into": (C.c_int, [C.c_void_p, C.c_void_p]),
    "iris_gpu_sync": (None, []),
    "iris_gpu_batch_begin": (None, []),
    "iris_gpu_batch_end": (None, []),
    "iris_gpu_linear_bf16_native": (C.c_void_p, [C.c_void_p, _u16p, C.c_int, C.c_int, C.c_int]),
    "iris_gpu_linear_bf16_native_into": (C.c_int, [C.c_void_p, C.c_void_p, _u16p, C.c_int, C.c_int,
                                                   C.c_int]),
    "iris_gpu_adaln_norm_bf16": (None, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int,
                                        C.c_int, C.c_float]),
    "iris_gpu_adaln_norm_bf16_noalloc": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
                                                   C.c_int, C.c_int, C.c_float, C.c_void_p]),
    "iris_gpu_qk_rms_norm_bf16": (None, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int,
                                         C.c_int, C.c_int, C.c_float]),
    "iris_gpu_rope_unified_bf16": (None, [C.c_void_p, C.c_void_p, _fp, _fp, _fp, _fp, _fp, _fp,
                                          C.c_int, C.c_int, C.c_int, C.c_int, C.c_int]),
    "iris_gpu_rope_2d_bf16": (None, [C.c_void_p, _fp, _fp, C.c_int, C.c_int, C.c_int, C.c_int]),
    "iris_gpu_attention_fused_bf16": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
                                                C.c_int, C.c_int, C.c_int, C.c_int, C.c_float]),
    "iris_gpu_silu_mul_bf16": (None, [C.c_void_p, C.c_void_p, C.c_int]),
    "iris_gpu_gated_add_bf16": (None, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int]),
    "iris_gpu_concat_seq_bf16": (None, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int,
                                        C.c_int]),
    "iris_gpu_slice_seq_bf16": (None, [C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int]),
    "iris_gpu_split_qkv_mlp_bf16": (None, [C.c_void_p] * 6 + [C.c_int] * 3),
    "iris_gpu_concat_attn_mlp_bf16": (None, [C.c_void_p] * 3 + [C.c_int] * 3),
    "iris_metal_available": (C.c_int, []),
    "iris_metal_shaders_available": (C.c_int, []),
    "iris_bf16_pipeline_available": (C.c_int, []),
    "iris_gpu_add_bf16": (None, [C.c_void_p] * 3 + [C.c_int]),
    "iris_gpu_copy_bf16": (None, [C.c_void_p, C.c_void_p, C.c_size_t]),
    "iris_gpu_head_rms_norm_bf16": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_float]),
    "iris_gpu_linear_bf16_bf16out": (C.c_void_p, [C.c_void_p, _u16p, C.c_int, C.c_int, C.c_int]),
    "iris_gpu_attention_mps_bf16": (C.c_int, [C.c_void_p] * 4 + [C.c_int] * 4 + [C.c_float]),
    "iris_gpu_attention_bf16_native": (C.c_int, [C.c_void_p] * 4 + [C.c_int] * 4 + [C.c_float]),
    "iris_gpu_tensor_data": (_fp, [C.c_void_p]),
    "iris_gpu_linear": (C.c_void_p, [C.c_void_p, _fp, _fp, C.c_int, C.c_int, C.c_int]),
    "iris_gpu_linear_bf16": (C.c_void_p, [C.c_void_p, _u16p, C.c_int, C.c_int, C.c_int]),
    "iris_gpu_linear_bf16_into": (C.c_int, [C.c_void_p, C.c_void_p, _u16p, C.c_int, C.c_int, C.c_int]),
    "iris_gpu_adaln_norm": (None, [C.c_void_p, C.c_void_p, _fp, _fp, C.c_int, C.c_int, C.c_float]),
    "iris_gpu_rms_norm_f32": (None, [C.c_void_p, C.c_void_p, _fp, C.c_int, C.c_int, C.c_float]),
    "iris_gpu_qk_rms_norm": (None, [C.c_void_p, C.c_void_p, _fp, _fp, C.c_int, C.c_int, C.c_int, C.c_float]),
    "iris_gpu_rope_single_f32": (None, [C.c_void_p, _fp, _fp, C.c_int, C.c_int, C.c_int]),
    "iris_gpu_rope_single_pair_f32": (None, [C.c_void_p, C.c_void_p, _fp, _fp, C.c_int, C.c_int, C.c_int]),
    "iris_gpu_rope_unified": (None, [C.c_void_p, C.c_void_p, _fp, _fp, _fp, _fp] + [C.c_int] * 5),
    "iris_gpu_silu_mul": (None, [C.c_void_p, C.c_void_p, C.c_int]),
    "iris_gpu_gated_add": (None, [C.c_void_p, _fp, C.c_void_p, C.c_int, C.c_int]),
    "iris_gpu_split_qkv_mlp": (None, [C.c_void_p] * 6 + [C.c_int] * 3),
    "iris_gpu_concat_attn_mlp": (None, [C.c_void_p] * 3 + [C.c_int] * 3),
    "iris_gpu_attention_fused": (C.c_int, [C.c_void_p] * 4 + [C.c_int] * 4 + [C.c_float]),
    "iris_gpu_attention_bf16": (C.c_int, [C.c_void_p] * 4 + [C.c_int] * 4 + [C.c_float]),
    "iris_gpu_add_f32": (None, [C.c_void_p] * 3 + [C.c_int]),
    "iris_gpu_copy_f32": (None, [C.c_void_p, C.c_void_p, C.c_size_t]),
    "iris_gpu_copy_region_f32": (None, [C.c_void_p, C.c_size_t, C.c_void_p, C.c_size_t, C.c_size_t]),
    "iris_metal_attention_fused": (C.c_int, [_fp] * 4 + [C.c_int] * 4 + [C.c_float]),
    "iris_metal_attention": (None, [_fp] * 5 + [C.c_int] * 4 + [C.c_float]),
    "iris_metal_set_attention_bias": (None, [C.c_int, C.c_float]),
    "iris_gpu_chain_begin": (None, []),
    "iris_gpu_chain_end": (None, []),
    "iris_gpu_in_chain": (C.c_int, []),
    "iris_metal_begin_batch": (None, []),
    "iris_metal_end_batch": (None, []),
    "iris_metal_in_batch": (C.c_int, []),
    "iris_metal_sync": (None, []),
    "iris_metal_wait_idle": (None, []),
    "iris_metal_init": (C.c_int, []),
    "iris_metal_cleanup": (None, []),
    "iris_metal_reset": (None, []),
    "iris_metal_reset_transient": (None, []),
    "iris_metal_rope_cache_begin": (None, []),
    "iris_metal_clear_weight_cache_only": (None, []),
    "iris_metal_clear_bf16_cache_only": (None, []),
    "iris_metal_clear_f16_cache_only": (None, []),
    "iris_metal_clear_activation_pool_only": (None, []),
    "iris_metal_memory_used": (C.c_size_t, []),
    "iris_metal_warmup_bf16": (None, [_u16p, C.c_size_t]),
    "iris_metal_warmup_bf16_buffer": (None, [_u16p, C.c_size_t]),
    "iris_metal_warmup_bf16_buffers_parallel": (None, [C.POINTER(_u16p), C.POINTER(C.c_size_t), C.c_int]),
    "iris_gpu_op_failures": (C.c_ulong, []),
    # language-model operators
    "iris_gpu_rope_init": (C.c_int, [C.POINTER(Rope), C.c_int, C.c_int, C.c_double, C.POINTER(RopeScaling)]),
    "iris_gpu_rope_init_freqs": (C.c_int, [C.POINTER(Rope), C.c_int, C.c_int, C.POINTER(C.c_double), C.c_double]),
    "iris_gpu_rope_append": (C.c_int, [C.POINTER(KvCache), C.POINTER(Rope), C.c_void_p, C.c_int64, C.c_void_p,
                                       C.c_void_p, C.c_void_p, C.c_int64, C.c_int64, C.c_int64, C.c_int, C.c_void_p,
                                       C.c_void_p, C.c_float, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_void_p]),
    "iris_gpu_attention_paged_workspace": (C.c_size_t, [C.POINTER(KvCache), C.c_int]),
    "iris_gpu_attention_paged": (C.c_int, [C.POINTER(KvCache), C.c_void_p, C.c_void_p, C.c_int64, C.c_int64,
                                           C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_float, C.c_void_p,
                                           C.c_size_t, C.c_void_p]),
    "iris_gpu_token_logprobs_workspace": (C.c_size_t, [C.c_int, C.c_int]),
    "iris_gpu_token_logprobs": (C.c_int, [C.c_void_p, C.c_int, C.c_int64, C.c_int, C.c_int, C.c_void_p, C.c_void_p,
                                          C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t,
                                          C.c_void_p]),
    "iris_gpu_rope_append8": (C.c_int, [C.POINTER(KvCache8), C.POINTER(Rope), C.c_void_p, C.c_int64, C.c_void_p,
                                        C.c_void_p, C.c_void_p, C.c_int64, C.c_int64, C.c_int64, C.c_int, C.c_void_p,
                                        C.c_void_p, C.c_float, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_void_p]),
    "iris_gpu_attention_paged8_workspace": (C.c_size_t, [C.POINTER(KvCache8), C.c_int]),
    "iris_gpu_attention_paged8": (C.c_int, [C.POINTER(KvCache8), C.c_void_p, C.c_void_p, C.c_int64, C.c_int64,
                                            C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_float, C.c_void_p,
                                            C.c_size_t, C.c_void_p]),
    "iris_gpu_sample_tokens": (C.c_int, [C.c_void_p, C.c_int, C.c_int64, C.c_int, C.c_int] + [C.c_void_p] * 9),
    "iris_gpu_quantize4": (C.c_int, [C.POINTER(Weights4), C.c_void_p, C.c_int, C.c_int64, C.c_void_p]),
    "iris_gpu_linear4": (C.c_int, [C.POINTER(Weights4), C.c_void_p, C.c_int64, C.c_int, C.c_void_p, C.c_int64,
                                   C.c_void_p, C.c_int64, C.c_int, C.c_void_p]),
}

_libc = C.CDLL(None)
_libc.free.argtypes = [C.c_void_p]
_libc.free.restype = None


class IrisCudaError(RuntimeError):
    pass


def load(path: str = LIB_PATH) -> C.CDLL:
    if not os.path.exists(path):
        raise IrisCudaError(f"{path} not built: run `make -C iris.c_b200 cuda` (no fallback path exists)")
    lib = C.CDLL(path)
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    return lib


_LIB = None


def lib() -> C.CDLL:
    global _LIB
    if _LIB is None:
        _LIB = load()
    return _LIB


def last_error() -> str:
    return (lib().iris_cuda_last_error() or b"").decode()


def _f(a: np.ndarray):
    assert a.dtype == np.float32 and a.flags["C_CONTIGUOUS"]
    return a.ctypes.data_as(_fp)


def _take_floats(ptr, n, shape=None) -> np.ndarray:
    if not ptr:
        raise IrisCudaError(last_error() or "call failed")
    # the library's malloc'd buffer becomes the array's memory (no copy); it is
    # freed when the last view of it goes away
    buf = (C.c_float * n).from_address(ptr)
    weakref.finalize(buf, _libc.free, ptr)
    arr = np.frombuffer(buf, np.float32)
    return arr.reshape(shape) if shape is not None else arr


class Flux:
    """Resident Flux.2 Klein transformer (libiris_cuda)."""

    def __init__(self, handle):
        if not handle:
            raise IrisCudaError(last_error() or "model creation failed")
        self.h = handle
        cfg = FluxConfig()
        lib().iris_cuda_flux_get_config(self.h, C.byref(cfg))
        self.cfg = cfg

    @classmethod
    def load(cls, model_dir: str, tp_rank: int = 0, tp_size: int = 1) -> "Flux":
        if tp_size == 1:
            return cls(lib().iris_cuda_flux_load(model_dir.encode()))
        return cls(lib().iris_cuda_flux_load_tp(model_dir.encode(), tp_rank, tp_size))

    @classmethod
    def random(cls, cfg: FluxConfig, seed: int, std: float = 0.02, norm_unit: bool = False,
               tp_rank: int = 0, tp_size: int = 1) -> "Flux":
        if tp_size == 1:
            return cls(lib().iris_cuda_flux_random(C.byref(cfg), seed, std, int(norm_unit)))
        return cls(lib().iris_cuda_flux_random_tp(C.byref(cfg), seed, std, int(norm_unit), tp_rank, tp_size))

    def close(self):
        if self.h:
            lib().iris_cuda_flux_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def weight_bytes(self) -> int:
        return lib().iris_cuda_flux_weight_bytes(self.h)

    def read_weight(self, name: str, shape) -> np.ndarray:
        out = np.zeros(int(np.prod(shape)), np.uint16)
        rc = lib().iris_cuda_flux_read_weight(self.h, name.encode(), out.ctypes.data_as(_u16p), out.size)
        if rc:
            raise IrisCudaError(last_error())
        return out.reshape(shape)

    def load_lora(self, path: str, scale: float = 1.0) -> int:
        """iris_load_lora: fold a LoRA file (XLabs / Kohya / Diffusers / BFL) into
        the weights at strength `scale`; returns the number of adapters applied."""
        if lib().iris_cuda_flux_load_lora(self.h, path.encode(), float(scale)):
            raise IrisCudaError(last_error())
        return lib().iris_cuda_flux_lora_adapters(self.h)

    def unload_lora(self) -> None:
        if lib().iris_cuda_flux_unload_lora(self.h):
            raise IrisCudaError(last_error())

    @property
    def lora_adapters(self) -> int:
        return lib().iris_cuda_flux_lora_adapters(self.h)

    def lora_stats(self) -> tuple[float, float]:
        """(device ms, bytes moved) of the last LoRA fold."""
        ms, nb = C.c_double(), C.c_double()
        lib().iris_cuda_flux_lora_stats(self.h, C.byref(ms), C.byref(nb))
        return ms.value, nb.value

    def load_ip_adapter(self, bundle_dir: str, features, scale_mult: float = 1.0) -> None:
        """iris_load_ip_adapter: features = a path to raw f32 rows, or an array."""
        if isinstance(features, str):
            rc = lib().iris_cuda_flux_load_ip_adapter(self.h, bundle_dir.encode(), features.encode(), scale_mult)
        else:
            f = np.ascontiguousarray(features, np.float32)
            n = f.shape[0] if f.ndim > 1 else 1
            rc = lib().iris_cuda_flux_load_ip_adapter_mem(self.h, bundle_dir.encode(), _f(f), n, scale_mult)
        if rc:
            raise IrisCudaError(last_error())

    def unload_ip_adapter(self) -> None:
        if lib().iris_cuda_flux_unload_ip_adapter(self.h):
            raise IrisCudaError(last_error())

    def set_ip_schedule(self, spec: str) -> None:
        if lib().iris_cuda_flux_set_ip_schedule(self.h, spec.encode()):
            raise IrisCudaError(last_error())

    def set_ip_step(self, step: int, num_steps: int) -> None:
        if lib().iris_cuda_flux_set_ip_step(self.h, step, num_steps):
            raise IrisCudaError(last_error())

    def ip_embeds(self, tokens: int) -> np.ndarray:
        out = np.zeros(tokens * self.cfg.hidden, np.float32)
        n = lib().iris_cuda_flux_ip_embeds(self.h, _f(out), out.size)
        if n < 0:
            raise IrisCudaError(last_error())
        return out[:n].reshape(-1, self.cfg.hidden)

    def set_sref_csd(self, csdmod_path, csd, scale: float) -> None:
        """iris_set_sref_csd: the CSD modulation delta on the timestep embedding (None: off)."""
        if csdmod_path is None:
            rc = lib().iris_cuda_flux_set_sref_csd(self.h, None, None, 0, 0.0)
        else:
            c = np.ascontiguousarray(csd, np.float32).ravel()
            rc = lib().iris_cuda_flux_set_sref_csd(self.h, csdmod_path.encode(), _f(c), c.size, scale)
        if rc:
            raise IrisCudaError(last_error())

    def set_sref_bands(self, shf: float, slf: float) -> None:
        if lib().iris_cuda_flux_set_sref_bands(self.h, shf, slf):
            raise IrisCudaError(last_error())

    def run_block(self, kind: int, idx: int, hidden: np.ndarray, txt_seq: int, img_h: int, img_w: int,
                  t: float) -> np.ndarray:
        hid = np.ascontiguousarray(hidden, np.float32).copy()
        rc = lib().iris_cuda_flux_run_block(self.h, kind, idx, _f(hid), txt_seq, img_h, img_w, t)
        if rc:
            raise IrisCudaError(last_error())
        return hid

    def forward(self, latent: np.ndarray, txt: np.ndarray, t: float, refs=()) -> np.ndarray:
        lat = np.ascontiguousarray(latent, np.float32)
        tx = np.ascontiguousarray(txt, np.float32)
        c, h, w = lat.shape
        if refs:
            keep = [np.ascontiguousarray(r, np.float32) for r in refs]
            arr = (Ref * len(keep))(*[Ref(_f(r), r.shape[1], r.shape[2], 10 * (i + 1))
                                      for i, r in enumerate(keep)])
            p = lib().iris_cuda_transformer_forward_with_multi_refs(self.h, _f(lat), h, w, arr, len(keep),
                                                                    _f(tx), tx.shape[0], t)
        else:
            p = lib().iris_cuda_transformer_forward(self.h, _f(lat), h, w, _f(tx), tx.shape[0], t)
        return _take_floats(p, c * h * w, (c, h, w))

    def profile(self, t: float, max_entries: int = 512):
        """Per-kernel CUDA-event times of one forward over the last input shape."""
        buf = (KernelTime * max_entries)()
        n = lib().iris_cuda_flux_profile(self.h, t, buf, max_entries)
        if n < 0:
            raise IrisCudaError(last_error())
        return [dict(name=buf[i].name.decode(), flops=buf[i].flops, bytes=buf[i].bytes, ms=buf[i].ms)
                for i in range(n)]

    def sample_euler(self, z, txt, schedule, refs=(), txt_uncond=None, guidance=1.0, cfg_pair=False):
        """Euler sampler; cfg_pair=True splits the CFG branches over the
        process's 2-rank communicator (comm_init)."""
        zz = np.ascontiguousarray(z, np.float32)
        tx = np.ascontiguousarray(txt, np.float32)
        sc = np.ascontiguousarray(schedule, np.float32)
        c, h, w = zz.shape
        cb = PROGRESS_CB(0)
        if cfg_pair:
            tu = np.ascontiguousarray(txt_uncond, np.float32)
            p = lib().iris_cuda_sample_euler_cfg_pair(self.h, _f(zz), 1, c, h, w, _f(tx), tx.shape[0], _f(tu),
                                                      tu.shape[0], guidance, _f(sc), len(sc) - 1, cb)
        elif txt_uncond is not None:
            tu = np.ascontiguousarray(txt_uncond, np.float32)
            p = lib().iris_cuda_sample_euler_cfg(self.h, _f(zz), 1, c, h, w, _f(tx), tx.shape[0], _f(tu),
                                                 tu.shape[0], guidance, _f(sc), len(sc) - 1, cb)
        elif refs:
            keep = [np.ascontiguousarray(r, np.float32) for r in refs]
            arr = (Ref * len(keep))(*[Ref(_f(r), r.shape[1], r.shape[2], 10 * (i + 1))
                                      for i, r in enumerate(keep)])
            p = lib().iris_cuda_sample_euler_with_multi_refs(self.h, _f(zz), 1, c, h, w, arr, len(keep),
                                                             _f(tx), tx.shape[0], _f(sc), len(sc) - 1, cb)
        else:
            p = lib().iris_cuda_sample_euler(self.h, _f(zz), 1, c, h, w, _f(tx), tx.shape[0], _f(sc),
                                             len(sc) - 1, cb)
        return _take_floats(p, c * h * w, (c, h, w))


def comm_unique_id() -> bytes:
    """A new NCCL unique id (IRIS_CUDA_COMM_ID_BYTES bytes) for comm_init."""
    buf = C.create_string_buffer(128)
    if lib().iris_cuda_comm_unique_id(buf, 128):
        raise IrisCudaError(last_error())
    return buf.raw


def comm_init(uid: bytes, world: int, rank: int) -> None:
    buf = C.create_string_buffer(bytes(uid), 128)
    if lib().iris_cuda_comm_init(buf, world, rank):
        raise IrisCudaError(last_error())


def comm_destroy() -> None:
    lib().iris_cuda_comm_destroy()


def comm_groups(world: int, group_size: int):
    """Rank groups of `group_size` consecutive ranks ((0,1), (2,3), ... for CFG
    pairs); every rank is in exactly one."""
    if group_size < 1 or world % group_size:
        raise ValueError(f"world {world} is not a multiple of group size {group_size}")
    return [tuple(range(g, g + group_size)) for g in range(0, world, group_size)]


def comm_init_group(exchange, rank: int, world: int, group_size: int) -> tuple:
    """Create this rank's NCCL communicator over its group of `group_size`
    consecutive ranks.  `exchange(obj)` must return the list of every rank's
    obj (e.g. torch.distributed.all_gather_object); the first rank of each
    group creates the id.  Returns (group, rank in group)."""
    groups = comm_groups(world, group_size)
    group = next(g for g in groups if rank in g)
    mine = comm_unique_id() if rank == group[0] else None
    ids = exchange(mine)
    comm_init(ids[group[0]], len(group), group.index(rank))
    return group, group.index(rank)


LORA_FORMATS = {1: "xlabs", 2: "kohya", 3: "diffusers", 4: "bfl"}


def lora_probe(path: str, n_double: int, n_single: int, hidden: int, mlp: int) -> dict:
    """Host-only: adapters of a LoRA file matching a model of this shape."""
    k = (C.c_int * 5)()
    n = lib().iris_cuda_lora_probe(path.encode(), n_double, n_single, hidden, mlp, k)
    if n < 0:
        raise IrisCudaError(last_error())
    return {"format": LORA_FORMATS[k[0]], "adapters": n, "qkv": k[1], "proj": k[2], "linear1": k[3],
            "linear2": k[4]}


def official_schedule(steps: int, seq: int) -> np.ndarray:
    return _take_floats(lib().iris_cuda_official_schedule(steps, seq), steps + 1)


def zimage_schedule(steps: int, seq: int) -> np.ndarray:
    return _take_floats(lib().iris_cuda_zimage_schedule(steps, seq), steps + 1)


def init_noise(c: int, h: int, w: int, seed: int) -> np.ndarray:
    return _take_floats(lib().iris_cuda_init_noise(1, c, h, w, seed), c * h * w, (c, h, w))


class ZImage:
    """Resident Z-Image S3-DiT transformer (libiris_cuda)."""

    def __init__(self, handle):
        if not handle:
            raise IrisCudaError(last_error() or "model creation failed")
        self.h = handle
        cfg = ZImageConfig()
        lib().iris_cuda_zimage_get_config(self.h, C.byref(cfg))
        self.cfg = cfg

    @classmethod
    def load(cls, model_dir: str) -> "ZImage":
        return cls(lib().iris_cuda_zimage_load(model_dir.encode()))

    @classmethod
    def random(cls, cfg: ZImageConfig, seed: int, std: float = 0.02, norm_unit: bool = False) -> "ZImage":
        return cls(lib().iris_cuda_zimage_random(C.byref(cfg), seed, std, int(norm_unit)))

    def close(self):
        if self.h:
            lib().iris_cuda_zimage_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def forward(self, latent: np.ndarray, cap: np.ndarray, t: float) -> np.ndarray:
        lat = np.ascontiguousarray(latent, np.float32)
        cp = np.ascontiguousarray(cap, np.float32)
        c, h, w = lat.shape
        p = lib().iris_cuda_zi_transformer_forward(self.h, _f(lat), h, w, t, _f(cp), cp.shape[0])
        return _take_floats(p, c * h * w, (c, h, w))

    def sample_euler(self, z: np.ndarray, cap: np.ndarray, schedule) -> np.ndarray:
        zz = np.ascontiguousarray(z, np.float32)
        cp = np.ascontiguousarray(cap, np.float32)
        sc = np.ascontiguousarray(schedule, np.float32)
        c, h, w = zz.shape
        p = lib().iris_cuda_sample_euler_zimage(self.h, _f(zz), 1, c, h, w, self.cfg.patch_size, _f(cp),
                                                cp.shape[0], _f(sc), len(sc) - 1, PROGRESS_CB(0))
        return _take_floats(p, c * h * w, (c, h, w))


class Vae:
    """Resident autoencoder decoder (libiris_cuda): latent -> RGB image."""

    def __init__(self, handle, z: int):
        if not handle:
            raise IrisCudaError(last_error() or "VAE load failed")
        self.h = handle
        self.z = z

    @classmethod
    def load(cls, vae_dir: str, z: int = 0, scaling: float = 0.0, shift: float = 0.0) -> "Vae":
        """z <= 0: latent channels, scaling and shift from vae_dir/config.json."""
        h = lib().iris_cuda_vae_load(vae_dir.encode(), z, scaling, shift)
        zz = z
        if zz <= 0:
            import json
            import os
            cfg = os.path.join(vae_dir, "config.json")
            zz = json.load(open(cfg)).get("latent_channels", 32) if os.path.exists(cfg) else 32
        return cls(h, zz)

    @classmethod
    def random(cls, z: int = 32, seed: int = 1, scaling: float = 0.0, shift: float = 0.0) -> "Vae":
        return cls(lib().iris_cuda_vae_random(z, scaling, shift, seed), z)

    def profile(self, max_entries: int = 512):
        """Per-kernel CUDA-event times of one decode at the last latent size."""
        arr = (KernelTime * max_entries)()
        n = lib().iris_cuda_vae_profile(self.h, arr, max_entries)
        if n < 0:
            raise IrisCudaError(last_error())
        return [dict(name=arr[i].name.decode(), ms=arr[i].ms, flops=arr[i].flops, bytes=arr[i].bytes)
                for i in range(n)]

    def close(self):
        if self.h:
            lib().iris_cuda_vae_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def weight_bytes(self) -> int:
        return lib().iris_cuda_vae_weight_bytes(self.h)

    def decode(self, latent: np.ndarray) -> np.ndarray:
        """[4z, h, w] latent -> uint8 [16h, 16w, 3] (iris_vae_decode)."""
        lat = np.ascontiguousarray(latent, np.float32)
        _, h, w = lat.shape
        p = lib().iris_cuda_vae_decode(self.h, _f(lat), 1, h, w)
        if not p:
            raise IrisCudaError(last_error())
        img = C.cast(p, C.POINTER(Image)).contents
        out = np.ctypeslib.as_array(img.data, shape=(img.height, img.width, img.channels)).copy()
        lib().iris_cuda_image_free(p)
        return out

    def decode_f32(self, latent: np.ndarray) -> np.ndarray:
        """[4z, h, w] latent -> f32 RGB planes [3, 16h, 16w] before the uint8 conversion."""
        lat = np.ascontiguousarray(latent, np.float32)
        _, h, w = lat.shape
        out = np.zeros((3, 16 * h, 16 * w), np.float32)
        if lib().iris_cuda_vae_decode_f32(self.h, _f(lat), h, w, _f(out)):
            raise IrisCudaError(last_error())
        return out

    def graph_kernels(self) -> int:
        return lib().iris_cuda_vae_graph_kernels(self.h)


class Qwen3:
    """Resident Qwen3 text encoder (libiris_cuda): token ids -> text embeddings."""

    def __init__(self, handle):
        if not handle:
            raise IrisCudaError(last_error() or "text encoder creation failed")
        self.h = handle

    @classmethod
    def load(cls, model_dir: str) -> "Qwen3":
        return cls(lib().iris_cuda_qwen3_load(model_dir.encode()))

    @classmethod
    def random(cls, cfg: Qwen3Config, seed: int) -> "Qwen3":
        return cls(lib().iris_cuda_qwen3_random(C.byref(cfg), seed))

    @classmethod
    def load_lm(cls, model_dir: str) -> "Qwen3":
        """With every layer, the final norm and the head: usable by Qwen3Lm."""
        return cls(lib().iris_cuda_qwen3_load_lm(model_dir.encode()))

    @classmethod
    def random_lm(cls, cfg: Qwen3Config, seed: int) -> "Qwen3":
        return cls(lib().iris_cuda_qwen3_random_lm(C.byref(cfg), seed))

    def close(self):
        if self.h:
            lib().iris_cuda_qwen3_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def set_extraction_mode(self, mode: int) -> None:
        if lib().iris_cuda_qwen3_set_extraction_mode(self.h, mode):
            raise IrisCudaError(last_error())

    def text_dim(self) -> int:
        return lib().iris_cuda_qwen3_text_dim(self.h)

    def profile(self, max_entries: int = 1024):
        """Per-kernel CUDA-event times of one forward at the last sequence length."""
        arr = (KernelTime * max_entries)()
        n = lib().iris_cuda_qwen3_profile(self.h, arr, max_entries)
        if n < 0:
            raise IrisCudaError(last_error())
        return [dict(name=arr[i].name.decode(), ms=arr[i].ms, flops=arr[i].flops) for i in range(n)]

    def forward(self, ids, mask=None) -> np.ndarray:
        """ids / mask [S] -> f32 [S, text_dim] (qwen3_forward)."""
        ip = C.POINTER(C.c_int)
        ids = np.ascontiguousarray(ids, np.int32)
        m = None if mask is None else np.ascontiguousarray(mask, np.int32)
        p = lib().iris_cuda_qwen3_forward(self.h, ids.ctypes.data_as(ip),
                                          None if m is None else m.ctypes.data_as(ip), len(ids))
        return _take_floats(p, len(ids) * self.text_dim(), (len(ids), self.text_dim()))


class Qwen3Lm:
    """The text model as a language model (libiris_cuda): a session with a paged
    key-value cache.  The model comes from Qwen3.load_lm / random_lm."""

    def __init__(self, model: Qwen3, num_seqs: int = 1, max_len: int = 2048, max_tokens: int = 512):
        self.h = lib().iris_cuda_qwen3_lm_create(model.h, num_seqs, max_len, max_tokens)
        if not self.h:
            raise IrisCudaError(last_error() or "language model session failed")
        self.model = model  # kept alive

    def close(self):
        if self.h:
            lib().iris_cuda_qwen3_lm_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def cache_bytes(self) -> int:
        return lib().iris_cuda_qwen3_lm_cache_bytes(self.h)

    def length(self, seq: int) -> int:
        n = lib().iris_cuda_qwen3_lm_length(self.h, seq)
        if n < 0:
            raise IrisCudaError(last_error())
        return n

    def step(self, ids, seq, pos, targets=None, top_k: int = 0) -> dict:
        """Feed tokens; per token: logprob (with targets), entropy, top_ids, top_logprobs."""
        ip = C.POINTER(C.c_int)
        arrs = [None if a is None else np.ascontiguousarray(a, np.int32) for a in (ids, seq, pos, targets)]
        n = len(arrs[0])
        if any(a is not None and a.shape != (n,) for a in arrs):
            raise IrisCudaError("step: ids, seq, pos and targets are lists of one length")
        out = dict(logprob=np.zeros(n, np.float32), entropy=np.zeros(n, np.float32),
                   top_ids=np.zeros((n, top_k), np.int32), top_logprobs=np.zeros((n, top_k), np.float32))
        rc = lib().iris_cuda_qwen3_lm_step(
            self.h, *[None if a is None else a.ctypes.data_as(ip) for a in arrs], n, top_k, _f(out["logprob"]),
            _f(out["entropy"]), out["top_ids"].ctypes.data_as(ip), _f(out["top_logprobs"]))
        if rc:
            raise IrisCudaError(last_error())
        return out


    def sample(self, ids, seq, pos, uniform, temperature=None, top_k=None, top_p=None, min_p=None) -> dict:
        """Feed tokens and draw the next one behind each (iris_gpu_sample_tokens): next, logprobs.  The settings are
        one number for all tokens, a list of them, or None."""
        ip, n = C.POINTER(C.c_int), len(ids)
        ints = [np.ascontiguousarray(a, np.int32) for a in (ids, seq, pos)]
        u = np.ascontiguousarray(uniform, np.float64)
        of = lambda a, ty: None if a is None else np.array(np.broadcast_to(np.asarray(a, ty), (n,)))  # noqa: E731
        try:
            t, k, p, m = of(temperature, np.float32), of(top_k, np.int32), of(top_p, np.float32), of(min_p, np.float32)
        except ValueError:
            raise IrisCudaError("sample: the settings are one number or as many as tokens") from None
        if any(a.shape != (n,) for a in (*ints, u)):
            raise IrisCudaError("sample: ids, seq, pos and uniform are lists of one length")
        out = dict(next=np.zeros(n, np.int32), logprobs=np.zeros(n, np.float32))
        opt = lambda a, ty: None if a is None else a.ctypes.data_as(C.POINTER(ty))  # noqa: E731
        if lib().iris_cuda_qwen3_lm_sample(self.h, *[a.ctypes.data_as(ip) for a in ints], n, opt(t, C.c_float), opt(k, C.c_int),
                                           opt(p, C.c_float), opt(m, C.c_float), opt(u, C.c_double),
                                           out["next"].ctypes.data_as(ip), _f(out["logprobs"])):
            raise IrisCudaError(last_error())
        return out


# ---------------------------------------------------------------- language-model operators
# Device tensors are anything with data_ptr(), shape, stride() and dtype (torch's
# are); every call queues its work on `stream` (a cudaStream_t as an integer, 0:
# the default stream) and raises IrisCudaError when it is refused.

def _ok(rc: int) -> None:
    if rc:
        raise IrisCudaError(last_error())


_DTYPES: dict = {}  # dtype object -> its name (a step of one token is a few microseconds: no string work per call)


def _dtype(t) -> str:
    d = t.dtype
    name = _DTYPES.get(d)
    if name is None:
        name = _DTYPES[d] = str(d).rpartition(".")[2]
    return name


def _need(what: str, t, dtype: str, shape: tuple):
    """Address of t after a check of its type, shape and contiguous last axis (None: 0)."""
    if t is None:
        return None
    if _dtype(t) != dtype or t.shape != shape or (shape[-1] > 1 and t.stride()[-1] != 1):
        raise IrisCudaError(f"{what}: needs {dtype} {shape}, contiguous in the last axis; "
                            f"got {_dtype(t)} {tuple(t.shape)}")
    return t.data_ptr()


def _heads_rows(what: str, t, dtype: str, rows: int, heads: int, head_dim: int):
    """(address, row stride) of [rows, heads, head_dim] or [rows, heads * head_dim]."""
    shape, stride = t.shape, t.stride()
    if _dtype(t) != dtype or stride[-1] != 1 or not (
            shape == (rows, heads * head_dim) if len(shape) == 2 else
            shape == (rows, heads, head_dim) and (heads == 1 or stride[1] == head_dim)):
        raise IrisCudaError(f"{what}: needs {dtype} [{rows}, {heads}, {head_dim}] with contiguous rows; "
                            f"got {_dtype(t)} {tuple(shape)}")
    return t.data_ptr(), stride[0] if rows > 1 else heads * head_dim


def rope_append(cache: KvCache, rope: Rope | None, q_out, q, k, v, seq, pos, *, heads: int, q_norm=None, k_norm=None,
                eps: float = 1e-6, stream: int = 0) -> None:
    """iris_gpu_rope_append: rotate the new tokens' Q and K, write K and V to the cache."""
    _append(lib().iris_gpu_rope_append, cache, rope, q_out, q, k, v, seq, pos, heads, q_norm, k_norm, eps, stream)


def rope_append8(cache: KvCache8, rope: Rope | None, q_out, q, k, v, seq, pos, *, heads: int, q_norm=None, k_norm=None,
                 eps: float = 1e-6, stream: int = 0) -> None:
    """iris_gpu_rope_append8: the same into an 8-bit cache."""
    _append(lib().iris_gpu_rope_append8, cache, rope, q_out, q, k, v, seq, pos, heads, q_norm, k_norm, eps, stream)


def _append(call, cache, rope, q_out, q, k, v, seq, pos, heads, q_norm, k_norm, eps, stream) -> None:
    n, d, nkv = seq.shape[0], cache.head_dim, cache.kv_heads
    ty = _dtype(k)
    if ty not in ("float32", "bfloat16"):
        raise IrisCudaError(f"rope_append: k is {ty}")
    kp, ldk = _heads_rows("k", k, ty, n, nkv, d)
    vp, ldv = _heads_rows("v", v, ty, n, nkv, d)
    qp = op = None
    ldq = ldo = 0
    if heads:
        qp, ldq = _heads_rows("q", q, ty, n, heads, d)
        op, ldo = _heads_rows("q_out", q_out, "bfloat16", n, heads, d)
    _ok(call(cache, rope, op, ldo, qp, kp, vp, ldq, ldk, ldv, ty == "float32", _need("q_norm", q_norm, "float32", (d,)),
             _need("k_norm", k_norm, "float32", (d,)), eps, _need("seq", seq, "int32", (n,)),
             _need("pos", pos, "int32", (n,)), n, heads, stream))


def attention_paged_workspace(cache: KvCache, heads: int) -> int:
    n = lib().iris_gpu_attention_paged_workspace(cache, heads)
    if not n:
        raise IrisCudaError(last_error())
    return n


def attention_paged(cache: KvCache, out, q, seq, pos, *, scale: float, workspace, stream: int = 0) -> None:
    """iris_gpu_attention_paged: q, out [rows, heads, head_dim]; seq None: row t is sequence t."""
    _attend(lib().iris_gpu_attention_paged, cache, out, q, seq, pos, scale, workspace, stream)


def attention_paged8_workspace(cache: KvCache8, heads: int) -> int:
    n = lib().iris_gpu_attention_paged8_workspace(cache, heads)
    if not n:
        raise IrisCudaError(last_error())
    return n


def attention_paged8(cache: KvCache8, out, q, seq, pos, *, scale: float, workspace, stream: int = 0) -> None:
    """iris_gpu_attention_paged8: the same over an 8-bit cache."""
    _attend(lib().iris_gpu_attention_paged8, cache, out, q, seq, pos, scale, workspace, stream)


def _attend(call, cache, out, q, seq, pos, scale, workspace, stream) -> None:
    n, d = pos.shape[0], cache.head_dim
    heads = q.shape[1] if len(q.shape) == 3 else q.shape[1] // d
    qp, ldq = _heads_rows("q", q, "bfloat16", n, heads, d)
    op, ldo = _heads_rows("out", out, "bfloat16", n, heads, d)
    _ok(call(cache, op, qp, ldo, ldq, _need("seq", seq, "int32", (n,)), _need("pos", pos, "int32", (n,)), n, heads, scale,
             workspace.data_ptr(), workspace.numel() * workspace.element_size(), stream))


def token_logprobs_workspace(rows: int, vocab: int) -> int:
    n = lib().iris_gpu_token_logprobs_workspace(rows, vocab)
    if not n:
        raise IrisCudaError(last_error())
    return n


def token_logprobs(logits, targets, logprob, entropy, top_ids, top_logprobs, *, workspace, stream: int = 0) -> None:
    """iris_gpu_token_logprobs: logits [rows, vocab]; the outputs may be None."""
    rows, vocab = logits.shape
    ty = _dtype(logits)
    if ty not in ("float32", "bfloat16") or logits.stride(1) != 1:
        raise IrisCudaError(f"token_logprobs: logits {ty}, stride {logits.stride(1)} between a row's values")
    k = top_ids.shape[1] if top_ids is not None else top_logprobs.shape[1] if top_logprobs is not None else 0
    if k and rows > 1 and any(t is not None and t.stride(0) != k for t in (top_ids, top_logprobs)):
        raise IrisCudaError("token_logprobs: the alternatives' rows lie one after the other")
    _ok(lib().iris_gpu_token_logprobs(logits.data_ptr(), ty == "float32", logits.stride(0) if rows > 1 else vocab, rows,
                                      vocab, _need("targets", targets, "int32", (rows,)),
                                      _need("logprob", logprob, "float32", (rows,)),
                                      _need("entropy", entropy, "float32", (rows,)), k,
                                      _need("top_ids", top_ids, "int32", (rows, k)),
                                      _need("top_logprobs", top_logprobs, "float32", (rows, k)),
                                      workspace.data_ptr(), workspace.numel() * workspace.element_size(), stream))


def sample_tokens(logits, uniform, ids, *, temperature=None, top_k=None, top_p=None, min_p=None, logprobs=None, kept=None,
                  stream: int = 0) -> None:
    """iris_gpu_sample_tokens: the next token of each row of logits [rows, vocab] into ids, drawn with uniform (float64);
    the settings are tensors [rows] or None."""
    rows, vocab = logits.shape
    ty = _dtype(logits)
    if ty not in ("float32", "bfloat16") or logits.stride(1) != 1:
        raise IrisCudaError(f"sample_tokens: logits {ty}, stride {logits.stride(1)} between a row's values")
    of = (rows,)
    _ok(lib().iris_gpu_sample_tokens(logits.data_ptr(), ty == "float32", logits.stride(0) if rows > 1 else vocab, rows,
                                     vocab, _need("temperature", temperature, "float32", of),
                                     _need("top_k", top_k, "int32", of), _need("top_p", top_p, "float32", of),
                                     _need("min_p", min_p, "float32", of), _need("uniform", uniform, "float64", of),
                                     _need("ids", ids, "int32", of), _need("logprobs", logprobs, "float32", of),
                                     _need("kept", kept, "int32", of), stream))


def quantize4(w: Weights4, weights, stream: int = 0) -> None:
    """iris_gpu_quantize4: round weights [n, k] (bfloat16 or float32) into w's tensors."""
    ty = _dtype(weights)
    if ty not in ("float32", "bfloat16") or tuple(weights.shape) != (w.n, w.k) or weights.stride(1) != 1:
        raise IrisCudaError(f"quantize4: needs float32 or bfloat16 [{w.n}, {w.k}] with contiguous rows; got {ty} "
                            f"{tuple(weights.shape)}")
    _ok(lib().iris_gpu_quantize4(w, weights.data_ptr(), ty == "float32", weights.stride(0), stream))


def linear4(out, x, w: Weights4, *, add=None, stream: int = 0) -> None:
    """iris_gpu_linear4: out [rows, n] = x [rows, k] times the weights (+ add [rows, n])."""
    rows = x.shape[0]
    ty = _dtype(out)
    if ty not in ("float32", "bfloat16"):
        raise IrisCudaError(f"linear4: out is {ty}")
    _ok(lib().iris_gpu_linear4(w, _need("x", x, "bfloat16", (rows, w.k)), x.stride(0), rows,
                               _need("out", out, ty, (rows, w.n)), out.stride(0), _need("add", add, ty, (rows, w.n)),
                               0 if add is None else add.stride(0), ty == "float32", stream))
