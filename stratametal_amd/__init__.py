"""stratametal_amd - MI355X (gfx950) quantized mixture-of-experts block.

Python host binding of the C ABI in include/smoe.h (libsmoe.so, built by stratametal_amd/build.py).  The
arithmetic lives in the HIP kernels; this module only passes device pointers (torch tensors supply the
memory and the stream) and turns refused calls into exceptions, as the reference's wrappers throw
MetalError (metal/include/strata/metal/device.hpp:28-31).  There is no CPU fallback: without the built
library every entry point raises.
"""
from __future__ import annotations

import ctypes as C
import functools
import os
from dataclasses import dataclass
from typing import Dict, Optional

_HERE = os.path.dirname(os.path.abspath(__file__))
# SMOE_LIB names another build of the same library (the host-sanitized lib/libsmoe_asan.so, for tests/test_sanitize.py)
LIB_PATH = os.environ.get("SMOE_LIB") or os.path.join(_HERE, "lib", "libsmoe.so")
_LIB = None

Q2_0 = 42
IQ2_S = 22
PATH_AUTO, PATH_GEMV, PATH_MFMA = 0, 1, 2
ROUTER_BF16, ROUTER_F32 = 0, 1  # smoe_geom.router_dtype
MFMA_TOKENS = 128  # SMOE_PATH_AUTO runs the prefill (MFMA) contract from this many tokens on
MFMA_CHUNK = 128   # columns per MFMA work item

_STATUS = {0: "ok", -1: "invalid argument", -2: "buffer too small", -3: "unsupported ggml type",
           -4: "HIP runtime error", -5: "misaligned pointer", -6: "NULL pointer"}


class SmoeError(RuntimeError):
    """A call the library refused (status != SMOE_OK); `.status` is the smoe_status code."""

    def __init__(self, status: int, msg: str):
        super().__init__(f"{_STATUS.get(status, status)}: {msg}")
        self.status = status


class _Geom(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("n_embd", "n_ff", "n_ff_shared", "n_expert", "top_k", "w_type", "sh_type",
                                         "router_dtype", "sh_gate_type", "sh_up_type", "sh_down_type")]


class _Weights(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("gate_exps", "up_exps", "down_exps", "router", "gate_sh", "up_sh",
                                          "down_sh", "gate_inp_sh", "logit_bias")]


class _Trace(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("logits", "ids", "weights", "counts", "offsets", "perm", "slot", "sgate",
                                          "stage_events", "xq", "hq", "parts", "shared", "overflow", "egate", "eup",
                                          "sgu", "shq")]


class _Ends(C.Structure):
    _fields_ = [("pre", C.c_void_p), ("post", C.c_void_p), ("eps", C.c_float), ("res_scale", C.c_float),
                ("y_scale", C.c_float), ("gate_act", C.c_int32)]


class _Linear(C.Structure):
    _fields_ = [("n_in", C.c_int32), ("n_out", C.c_int32), ("w_type", C.c_int32), ("act", C.c_int32), ("w", C.c_void_p),
                ("w2", C.c_void_p), ("bias", C.c_void_p), ("bias2", C.c_void_p)]


class _Linear4(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("n_in", "n_out", "x_type", "act", "group", "s_type")] + \
               [(n, C.c_void_p) for n in ("w", "w2", "scales", "scales2", "zeros", "zeros2", "bias", "bias2")]


class _Rope(C.Structure):
    _fields_ = [("head_dim", C.c_int32), ("rot_dim", C.c_int32), ("layout", C.c_int32), ("scale", C.c_float),
                ("turns", C.c_void_p)]


class _Kv(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p)] + \
               [(n, C.c_int32) for n in ("type", "n_pages", "page_size", "n_kv_heads", "head_dim")]


class _Hc(C.Structure):
    _fields_ = [("hc", C.c_int32), ("hc_lr", C.c_int32), ("eps", C.c_float), ("norm", C.c_void_p),
                ("down", C.c_void_p), ("up", C.c_void_p), ("inject", C.c_void_p)]


STAGES = ("router", "route", "gate_up", "down", "combine")
STATUS_X_FP16, STATUS_H_FP16, STATUS_WAIT = 1, 2, 4  # bits of a call's status mask (smoe.h SMOE_STATUS_*)


def set_wait_limit(polls: int) -> int:
    """The bound of the fused decode launch's waits (smoe_set_wait_limit): polls > 0 sets it, 0 restores the default,
    a negative value makes every wait give up at once (tests of the give-up path).  Returns the previous bound."""
    return int(lib().smoe_set_wait_limit(int(polls)))
STAGE_EVENTS = len(STAGES) + 1


def lib():
    """The loaded libsmoe.so.  Raises ImportError when it has not been built (no fallback exists)."""
    global _LIB
    if _LIB is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(f"{LIB_PATH} is missing: build it with `python -m stratametal_amd.build`")
        L = C.CDLL(LIB_PATH)
        vp, i32, i64, u64, f32 = C.c_void_p, C.c_int32, C.c_int64, C.c_uint64, C.c_float
        sigs = {
            "smoe_workspace_bytes": (C.c_size_t, [vp, i32]),
            "smoe_forward": (i32, [vp, vp, vp, i32, vp, i32, vp, C.c_size_t, vp, vp]),
            "smoe_forward_path": (i32, [vp, vp, vp, i32, vp, i32, vp, C.c_size_t, vp, i32, vp]),
            "smoe_forward_residual": (i32, [vp, vp, vp, vp, f32, vp, i32, vp, i32, vp, C.c_size_t, vp, vp]),
            "smoe_forward_static": (i32, [vp, vp, vp, i32, vp, i32, vp, vp]),
            "smoe_forward_status": (i32, [vp, vp, vp]),
            "smoe_set_wait_limit": (i32, [i32]),
            "smoe_hc_read_workspace_bytes": (C.c_size_t, [vp, i32, i32]),
            "smoe_hc_read": (i32, [vp, i32, vp, i32, vp, vp, vp, C.c_size_t, vp]),
            "smoe_hc_write": (i32, [vp, i32, vp, vp, vp, i32, vp, vp]),
            "smoe_ffn_workspace_bytes": (C.c_size_t, [vp, vp, i32]),
            "smoe_ffn_run": (i32, [vp, vp, vp, vp, i32, vp, i32, vp, C.c_size_t, vp, vp]),
            "smoe_block_ends": (i32, [vp, i32, i32, vp, i32, i64, vp, i32, i64, vp, i64, i64, vp, i64, vp, i32, i64, vp]),
            "smoe_linear_workspace_bytes": (C.c_size_t, [vp, i32]),
            "smoe_linear_run": (i32, [vp, vp, i64, i32, vp, i64, vp, i32, i64, vp, C.c_size_t, vp]),
            "smoe_linear4_workspace_bytes": (C.c_size_t, [vp, i32]),
            "smoe_linear4_run": (i32, [vp, vp, i64, i32, vp, i64, vp, i32, i64, vp, C.c_size_t, vp]),
            "smoe_rope_table": (i32, [i32, C.c_double, i32, C.c_double, C.c_double, C.c_double, C.c_double, vp, vp]),
            "smoe_rope_run": (i32, [vp, vp, i32, i32, vp, i32, i64, vp, i32, i64, vp]),
            "smoe_kv_append": (i32, [vp, vp, vp, vp, i32, i32, vp, i64, i32, vp, i64, vp, i64, vp, i64, vp]),
            "smoe_attend_workspace_bytes": (C.c_size_t, [vp, i32, i32, i32, i64, i32]),
            "smoe_attend": (i32, [vp, vp, i64, i32, i32, vp, vp, i32, vp, i64, i32, i64, f32, i32, i32, vp, i64, vp, vp,
                                  C.c_size_t, vp]),
            "smoe_router_balance_workspace_bytes": (C.c_size_t, [i32, i32]),
            "smoe_router_balance": (i32, [vp, i64, vp, vp, i32, i32, i32, f32, f32, vp, vp, vp, vp, i64, vp, vp, C.c_size_t,
                                          vp]),
            "smoe_router_topk": (i32, [vp, i32, i32, i32, vp, vp, vp]),
            "smoe_router_margin": (i32, [vp, i32, i32, i32, vp, vp, vp]),
            "smoe_f32_to_bf16": (i32, [vp, i64, vp, vp]),
            "smoe_bf16_gemv": (i32, [vp, vp, vp, i32, i32, i32, vp]),
            "smoe_quantize_q8_1": (i32, [vp, i64, vp, vp]),
            "smoe_mmvq": (i32, [i32, vp, i64, vp, i32, i32, i32, vp, vp]),
            "smoe_swiglu_q8": (i32, [vp, vp, i64, vp, vp]),
            "smoe_combine": (i32, [vp, vp, vp, vp, i32, i32, vp]),
            "smoe_dispatch": (i32, [vp, i32, i32, i32, vp, vp, vp, vp, vp]),
            "smoe_expert_bytes": (C.c_size_t, [i32, i32, i64, i64]),
            "smoe_residual_rmsnorm": (i32, [vp, vp, i32, i32, f32, vp, vp]),
            "smoe_expert_scratch_bytes": (C.c_size_t, [i64, i64, i64]),
            "smoe_expert": (i32, [vp, C.c_size_t, vp, i32, i32, i64, i64, i64, vp, vp, C.c_size_t, vp]),
            "smoe_synth_blocks": (i32, [i32, u64, u64, i64, f32, vp, vp]),
            "smoe_synth_bf16": (i32, [u64, u64, i64, f32, vp, vp]),
            "smoe_synth_normal": (i32, [u64, u64, i64, f32, vp, vp]),
            "smoe_status_str": (C.c_char_p, [i32]),
            "smoe_last_error": (C.c_char_p, []),
            "smoe_abi_version": (i32, []),
            "smoe_model_open": (i32, [C.c_char_p, C.POINTER(vp)]),
            "smoe_model_close": (None, [vp]),
            "smoe_model_n_shards": (i32, [vp]),
            "smoe_model_n_tensors": (i64, [vp]),
            "smoe_model_tensor": (i32, [vp, C.c_char_p, vp]),
            "smoe_model_tensor_at": (i32, [vp, i64, C.c_char_p, C.c_size_t, vp]),
            "smoe_model_meta_u64": (i32, [vp, C.c_char_p, C.POINTER(u64)]),
            "smoe_model_meta_str": (i32, [vp, C.c_char_p, C.c_char_p, C.c_size_t]),
            "smoe_layer_plan_for": (i32, [vp, i32, i32, i32, vp]),
            "smoe_layer_upload": (i32, [vp, vp, vp, C.c_size_t, vp, vp, vp]),
            "smoe_expert_blob_bytes": (C.c_size_t, [vp]),
            "smoe_expert_pack": (i32, [vp, vp, i32, vp, vp]),
            "smoe_expert_group": (i32, [vp, i32, i32, i32, vp, vp, vp, vp, vp, vp, vp, vp, vp]),
            "smoe_expert_grouped_workspace_bytes": (C.c_size_t, [vp, i32, i32, i32]),
            "smoe_expert_grouped": (i32, [vp, vp, vp, vp, vp, vp, i32, i32, vp, i32, vp, i32, vp, C.c_size_t, vp]),
            "smoe_verify_workspace_bytes": (C.c_size_t, [vp, i32]),
            "smoe_verify_begin": (i32, [vp, vp, vp, vp, i32, vp, vp, vp, vp, vp, vp, C.c_size_t, vp]),
            "smoe_verify_end": (i32, [vp, i32, vp, vp, i32, vp, vp, C.c_size_t, vp]),
        }
        for name, (res, args) in sigs.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _LIB = L
    return _LIB


def _check(status: int):
    if status != 0:
        raise SmoeError(status, lib().smoe_last_error().decode())


def _ptr(t) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _need(t, name: str, dtype, shape=None, numel=None):
    """Refuse, before any launch, a tensor the kernels would misread or run past: it must be on a GPU, contiguous,
    of `dtype`, and (when given) of `shape` or at least `numel` elements."""
    import torch
    if not isinstance(t, torch.Tensor):
        raise SmoeError(-1, f"{name} is not a tensor")
    if t.dtype != dtype:
        raise SmoeError(-1, f"{name} is {t.dtype}, needs {dtype}")
    if not t.is_contiguous():
        raise SmoeError(-5, f"{name} is not contiguous")
    if shape is not None and t.shape != tuple(shape):
        raise SmoeError(-2, f"{name} has shape {tuple(t.shape)}, needs {tuple(shape)}")
    if numel is not None and t.numel() < numel:
        raise SmoeError(-2, f"{name} has {t.numel()} elements, needs {numel}")
    if not t.is_cuda:
        raise SmoeError(-1, f"{name} is on {t.device}, not a GPU")
    return t


def _int32(v, name: str):
    """Refuse a number that the C call's 32 bits do not hold: ctypes would pass its low bits."""
    if not -1 << 31 <= v < 1 << 31:
        raise SmoeError(-1, f"{name} is {v}, which 32 bits do not hold")
    return v


def _stream(stream=None) -> int:
    import torch
    s = torch.cuda.current_stream() if stream is None else stream
    return s.cuda_stream


def _parts(buf, *sizes):
    """Consecutive views of `buf`, one per size."""
    out, at = [], 0
    for n in sizes:
        out.append(buf[at:at + n])
        at += n
    return out


# the other native GGUF types (smoe.h): type -> (values per block, bytes per block)
Q8_0, Q4_0, Q5_0, IQ4_NL, IQ4_XS, Q3_K, Q4_K, Q5_K, Q6_K = 8, 2, 6, 20, 23, 11, 12, 13, 14
NATIVE_BLOCKS = {Q8_0: (32, 34), Q4_0: (32, 18), Q5_0: (32, 22), IQ4_NL: (32, 18), IQ4_XS: (256, 136),
                 Q3_K: (256, 110), Q4_K: (256, 144), Q5_K: (256, 176), Q6_K: (256, 210)}


def row_bytes(wtype: int, n: int) -> int:
    if wtype == Q2_0:
        return n // 64 * 18
    if wtype == IQ2_S:
        return n // 256 * 82
    if wtype in NATIVE_BLOCKS:
        qk, nb = NATIVE_BLOCKS[wtype]
        return n // qk * nb
    raise ValueError(wtype)


@dataclass
class Geom:
    """Layer geometry (smoe_geom).  Defaults are the benchmark configurations' layer."""
    n_embd: int = 2048
    n_ff: int = 512
    n_ff_shared: int = 512
    n_expert: int = 512
    top_k: int = 10
    w_type: int = Q2_0
    sh_type: int = Q2_0
    router_dtype: int = 0
    # the shared expert's gate, up and down projections in their own native types (0: sh_type)
    sh_gate_type: int = 0
    sh_up_type: int = 0
    sh_down_type: int = 0

    def c(self) -> _Geom:
        return _Geom(self.n_embd, self.n_ff, self.n_ff_shared, self.n_expert, self.top_k, self.w_type, self.sh_type,
                     self.router_dtype, self.sh_gate_type, self.sh_up_type, self.sh_down_type)

    def shared_types(self):
        """(gate, up, down) types of the shared expert."""
        return tuple(t if t else self.sh_type for t in (self.sh_gate_type, self.sh_up_type, self.sh_down_type))

    def expert_bytes(self) -> int:
        return 2 * self.n_ff * row_bytes(self.w_type, self.n_embd) + self.n_embd * row_bytes(self.w_type, self.n_ff)

    def shared_bytes(self) -> int:
        if self.sh_type < 0:
            return 0
        tg, tu, td = self.shared_types()
        return (self.n_ff_shared * (row_bytes(tg, self.n_embd) + row_bytes(tu, self.n_embd))
                + self.n_embd * row_bytes(td, self.n_ff_shared))


def workspace_bytes(g: Geom, max_tokens: int) -> int:
    n = lib().smoe_workspace_bytes(C.byref(g.c()), max_tokens)
    if n == 0:
        raise SmoeError(-1, lib().smoe_last_error().decode() or "bad geometry")
    return n


# ------------------------------------------------------------------------------------------------ layers

WEIGHT_NAMES = ("gate_exps", "up_exps", "down_exps", "router", "gate_sh", "up_sh", "down_sh", "gate_inp_sh",
                "logit_bias")


def synth_layer(g: Geom, seed: int, device="cuda", sigma: float = 0.02, logit_bias=None, stream=None) -> Dict:
    """A synthetic layer generated on the device (streams: 1 gate, 2 up, 3 down, 4 router, 5/6/7 shared
    gate/up/down, 8 shared gate_inp), bit-identical to the test oracle's host generators."""
    import torch
    L = lib()
    st = _stream(stream)
    H, F, Fs, E = g.n_embd, g.n_ff, g.n_ff_shared, g.n_expert

    def blocks(t, stream_id, n_values):
        buf = torch.empty(n_values // (64 if t == Q2_0 else 256) * (18 if t == Q2_0 else 82), dtype=torch.uint8,
                          device=device)
        _check(L.smoe_synth_blocks(t, seed, stream_id, n_values, sigma, buf.data_ptr(), st))
        return buf

    def bf16(stream_id, n):
        buf = torch.empty(n, dtype=torch.int16, device=device)
        _check(L.smoe_synth_bf16(seed, stream_id, n, sigma, buf.data_ptr(), st))
        return buf

    # the router is generated in f32 and kept in f32 (router_dtype 1) or stored as bf16 (the repo's contract)
    router = synth_normal(seed, 4, E * H, sigma, device=device, stream=stream) if g.router_dtype == ROUTER_F32 \
        else bf16(4, E * H)
    w = dict(gate_exps=blocks(g.w_type, 1, E * F * H), up_exps=blocks(g.w_type, 2, E * F * H),
             down_exps=blocks(g.w_type, 3, E * H * F), router=router)
    if g.sh_type >= 0:
        if any(t not in (Q2_0, IQ2_S) for t in g.shared_types()):
            raise ValueError("synth_layer generates Q2_0 and IQ2_S blocks only; upload other native types' blocks")
        tg, tu, td = g.shared_types()
        w.update(gate_sh=blocks(tg, 5, Fs * H), up_sh=blocks(tu, 6, Fs * H),
                 down_sh=blocks(td, 7, H * Fs), gate_inp_sh=bf16(8, H))
    if logit_bias is not None:
        w["logit_bias"] = logit_bias
    return w


def synth_normal(seed: int, stream_id: int, n: int, sigma: float = 1.0, device="cuda", stream=None):
    import torch
    out = torch.empty(n, dtype=torch.float32, device=device)
    _check(lib().smoe_synth_normal(seed, stream_id, n, sigma, out.data_ptr(), _stream(stream)))
    return out


def zipf_targets(n_expert: int, s: float, n_tokens: int, top_k: int):
    """Expected pairs per popularity rank r = 1 .. n_expert under Zipf(s): C * r^-s, capped at n_tokens (a token
    picks an expert at most once), with C such that the counts sum to n_tokens * top_k."""
    import numpy as np
    r = np.arange(1, n_expert + 1, dtype=np.float64)
    lo, hi = 0.0, float(n_tokens) * top_k * n_expert
    for _ in range(200):
        c = 0.5 * (lo + hi)
        if np.minimum(n_tokens, c * r ** -s).sum() < n_tokens * top_k:
            lo = c
        else:
            hi = c
    return np.minimum(n_tokens, 0.5 * (lo + hi) * r ** -s)


@functools.lru_cache(maxsize=8)
def _zipf_bias_cached(n_expert, s, seed, n_tokens, top_k, sigma, sims, iters):
    import numpy as np
    rng = np.random.default_rng(seed)
    rank_of = rng.permutation(n_expert)  # expert e has popularity rank rank_of[e]
    want = zipf_targets(n_expert, s, n_tokens, top_k) * (sims / n_tokens)
    tgt = np.clip(np.rint(want).astype(np.int64), 0, sims - 1)
    eps = rng.standard_normal((sims, n_expert)) * sigma
    b = np.log(want / want.mean()) * sigma
    cols = np.arange(n_expert)
    for _ in range(iters):
        z = eps + b
        head = -np.partition(-z, top_k, axis=1)[:, :top_k + 1]
        head.sort(axis=1)
        vk, vk1 = head[:, 1], head[:, 0]  # each token's k-th and (k+1)-th largest score
        # with the other experts' scores fixed, token t picks e iff b_e > (its k-th largest without e) - eps_te
        d = np.sort(np.where(z >= vk[:, None], vk1[:, None], vk[:, None]) - eps, axis=0)
        lo = np.where(tgt > 0, d[np.maximum(tgt - 1, 0), cols], d[0] - sigma)
        hi = np.where(tgt < sims, d[np.minimum(tgt, sims - 1), cols], d[-1] + sigma)
        b = b + 0.5 * (0.5 * (lo + hi) - b)
    return b[rank_of].astype(np.float32)


def zipf_bias(n_expert: int = 512, s: float = 1.2, seed: int = 1, n_tokens: int = 512, top_k: int = 10,
              n_embd: int = 2048, w_sigma: float = 0.02, sims: int = 4096, iters: int = 24):
    """Router logit bias of the prefill benchmark's routing: expert popularity follows
    Zipf(s) over a seeded rank permutation of the experts, i.e. the expected pairs of the rank-r expert are
    zipf_targets(...)[r-1] (hot experts take every token, many take none).  For x ~ N(0, 1) and router rows
    ~ N(0, w_sigma^2) a token's logits are close to independent N(0, sigma^2), sigma = w_sigma * sqrt(n_embd); the
    bias is fitted to that model by simulating `sims` tokens with fixed noise and solving, expert by expert, for
    the bias at which exactly its target share of the simulated tokens ranks it in their top k (damped
    fixed-point iterations).  Host-side and deterministic; an f32 numpy array of n_expert."""
    sigma = w_sigma * float(n_embd) ** 0.5
    return _zipf_bias_cached(n_expert, float(s), seed, n_tokens, top_k, sigma, sims, iters).copy()


def _weights_c(w: Dict) -> _Weights:
    return _Weights(*[_ptr(w.get(n)) for n in WEIGHT_NAMES])


class MoELayer:
    """One layer's MoE call: the FfnExec shape (metal/include/strata/metal/layer_exec.hpp:113-140) over
    smoe_forward.  Owns a workspace sized for `max_tokens`; weights stay the caller's tensors."""

    def __init__(self, g: Geom, weights: Dict, max_tokens: int, device="cuda"):
        import torch
        self.g = g
        self.w = weights
        self._gc = g.c()
        self._wc = _weights_c(weights)
        self.max_tokens = max_tokens
        self.ws_bytes = workspace_bytes(g, max_tokens)
        self.ws = torch.empty(self.ws_bytes, dtype=torch.uint8, device=device)

    def forward(self, x, y=None, add_shared: bool = True, trace: bool = False, path: int = PATH_AUTO, stream=None,
                stages: bool = False):
        """y = MoE(x).  With `trace`, also returns the routing and the dispatch (logits, ids, weights, counts,
        offsets, perm, slot, sgate); with `stages` as well, the expert stages (xq, hq: q8_1 blocks of x and of each
        pair's h on the decode path; egate, eup: each pair's gate and up dots; sgu, shq: the shared expert's gate and
        up dots ([2][T][n_ff_shared]) and the q8_1 blocks of its h; parts, shared: each pair's expert output and the
        shared expert's, by dispatch position) and the prefill path's fp16 `overflow` mask -- the decode path then
        runs its unfused kernels."""
        import torch
        if x.dim() != 2:
            raise SmoeError(-1, f"x must be (tokens, {self.g.n_embd}), got {tuple(x.shape)}")
        T = x.shape[0]
        _need(x, "x", torch.float32, shape=(T, self.g.n_embd))
        if T > self.max_tokens:
            raise SmoeError(-2, f"{T} tokens exceed the workspace's {self.max_tokens}")
        if y is None:
            y = torch.empty_like(x)
        _need(y, "y", torch.float32, numel=T * self.g.n_embd)
        tr = None
        out = {}
        if trace:
            E, K, dev = self.g.n_expert, self.g.top_k, x.device
            out = dict(logits=torch.empty((T, E), dtype=torch.float32, device=dev),
                       ids=torch.empty((T, K), dtype=torch.int32, device=dev),
                       weights=torch.empty((T, K), dtype=torch.float32, device=dev),
                       counts=torch.empty(E, dtype=torch.int32, device=dev),
                       offsets=torch.empty(E + 1, dtype=torch.int32, device=dev),
                       perm=torch.empty(T * K, dtype=torch.int32, device=dev),
                       slot=torch.empty(T * K, dtype=torch.int32, device=dev),
                       sgate=torch.empty(T, dtype=torch.float32, device=dev))
            names = ["logits", "ids", "weights", "counts", "offsets", "perm", "slot", "sgate"]
            if stages:
                H, F, Fs = self.g.n_embd, self.g.n_ff, max(self.g.n_ff_shared, 32)
                out.update(xq=torch.empty((T, H // 32 * 36), dtype=torch.uint8, device=dev),
                           hq=torch.empty((T * K, F // 32 * 36), dtype=torch.uint8, device=dev),
                           parts=torch.empty((T * K, H), dtype=torch.float32, device=dev),
                           shared=torch.empty((T, H), dtype=torch.float32, device=dev),
                           overflow=torch.full((1,), -1, dtype=torch.int32, device=dev),
                           egate=torch.empty((T * K, F), dtype=torch.float32, device=dev),
                           eup=torch.empty((T * K, F), dtype=torch.float32, device=dev),
                           sgu=torch.empty((2, T, Fs), dtype=torch.float32, device=dev),
                           shq=torch.empty((T, Fs // 32 * 36), dtype=torch.uint8, device=dev))
            tr = _Trace(*[out[n].data_ptr() for n in names], None,
                        *[out[n].data_ptr() if stages else None
                          for n in ("xq", "hq", "parts", "shared", "overflow", "egate", "eup", "sgu", "shq")])
        _check(lib().smoe_forward_path(C.byref(self._gc), C.byref(self._wc), x.data_ptr(), T, y.data_ptr(),
                                       int(add_shared), self.ws.data_ptr(), self.ws_bytes,
                                       None if tr is None else C.byref(tr), path, _stream(stream)))
        return (y, out) if trace else y

    def status(self, stream=None):
        """The status mask of the last call on this layer's workspace (smoe_forward_status), as a device int32
        tensor: 0, or STATUS_X_FP16 | STATUS_H_FP16 (the prefill path's fp16 operand limits) | STATUS_WAIT (a
        fused decode launch's wait gave up; its rows are NaN)."""
        import torch
        out = torch.full((1,), -1, dtype=torch.int32, device=self.ws.device)
        _check(lib().smoe_forward_status(self.ws.data_ptr(), out.data_ptr(), _stream(stream)))
        return out

    def forward_residual(self, x_prev, r_prev, x, y=None, eps: float = 1e-6, add_shared: bool = True, stream=None):
        """The stack junction fused into this layer's call: x = RMSNorm(x_prev + r_prev) (written to `x`), then
        y = MoE(x) (smoe_forward_residual).  `x` must not overlap x_prev, r_prev or y; y may be r_prev."""
        import torch
        if x.dim() != 2:
            raise SmoeError(-1, f"x must be (tokens, {self.g.n_embd}), got {tuple(x.shape)}")
        T = x.shape[0]
        shape = (T, self.g.n_embd)
        for t, name in ((x_prev, "x_prev"), (r_prev, "r_prev"), (x, "x")):
            _need(t, name, torch.float32, shape=shape)
        if T > self.max_tokens:
            raise SmoeError(-2, f"{T} tokens exceed the workspace's {self.max_tokens}")
        if y is None:
            y = torch.empty_like(x)
        _need(y, "y", torch.float32, numel=T * self.g.n_embd)
        _check(lib().smoe_forward_residual(C.byref(self._gc), C.byref(self._wc), x_prev.data_ptr(), r_prev.data_ptr(),
                                           eps, x.data_ptr(), T, y.data_ptr(), int(add_shared), self.ws.data_ptr(),
                                           self.ws_bytes, None, _stream(stream)))
        return y

    __call__ = forward


# ------------------------------------------------------------------------------------------------ layer ends

class HyperConnection:
    """The gated-residual ends of the layer call (smoe_hc_read / smoe_hc_write), the gr_read / gr_write pair of
    FfnExec::run (metal/include/strata/metal/gr.hpp:44-48).  `norm` is [hc * n_embd] f32 (the stored 1 + w);
    `down` [hc_lr][hc * n_embd], `up` [hc * n_embd][hc_lr] and `inject` [hc][hc * n_embd] are bf16 bits (int16)."""

    def __init__(self, n_embd: int, hc: int, hc_lr: int, norm, down, up, inject, eps: float = 1e-6):
        import torch
        hd = hc * n_embd
        _need(norm, "norm", torch.float32, numel=hd)
        for t, name, k in ((down, "down", hc_lr * hd), (up, "up", hd * hc_lr), (inject, "inject", hc * hd)):
            _need(t, name, torch.int16, numel=k)
        self.n_embd, self.hc, self.hc_lr, self.eps = n_embd, hc, hc_lr, eps
        self.tensors = (norm, down, up, inject)
        self._c = _Hc(hc, hc_lr, eps, norm.data_ptr(), down.data_ptr(), up.data_ptr(), inject.data_ptr())
        self._ws = None

    def _stream_tensor(self, R, name="R"):
        import torch
        if R.dim() != 3 or tuple(R.shape[1:]) != (self.hc, self.n_embd):
            raise SmoeError(-1, f"{name} must be (tokens, {self.hc}, {self.n_embd}), got {tuple(R.shape)}")
        return _need(R, name, torch.float32)

    def read(self, R, mixed=None, inject=None, stream=None):
        """mixed [T][n_embd], inject [T][hc] of the streams R [T][hc][n_embd]."""
        import torch
        R = self._stream_tensor(R)
        T = R.shape[0]
        if mixed is None:
            mixed = torch.empty((T, self.n_embd), dtype=torch.float32, device=R.device)
        if inject is None:
            inject = torch.empty((T, self.hc), dtype=torch.float32, device=R.device)
        _need(mixed, "mixed", torch.float32, numel=T * self.n_embd)
        _need(inject, "inject", torch.float32, numel=T * self.hc)
        n = lib().smoe_hc_read_workspace_bytes(C.byref(self._c), self.n_embd, max(T, 1))
        if n == 0:
            raise SmoeError(-1, lib().smoe_last_error().decode() or "bad hyper-connection shape")
        if self._ws is None or self._ws.numel() < n:
            self._ws = torch.empty(n, dtype=torch.uint8, device=R.device)
        _check(lib().smoe_hc_read(C.byref(self._c), self.n_embd, R.data_ptr(), T, mixed.data_ptr(), inject.data_ptr(),
                                  self._ws.data_ptr(), self._ws.numel(), _stream(stream)))
        return mixed, inject

    def write(self, R, y, inject, out=None, stream=None):
        """out = R + y * 2 sigmoid(inject / hc) on every stream; `out` may be R."""
        import torch
        R = self._stream_tensor(R)
        T = R.shape[0]
        _need(y, "y", torch.float32, numel=T * self.n_embd)
        _need(inject, "inject", torch.float32, numel=T * self.hc)
        if out is None:
            out = torch.empty_like(R)
        _need(out, "out", torch.float32, numel=R.numel())
        _check(lib().smoe_hc_write(C.byref(self._c), self.n_embd, R.data_ptr(), y.data_ptr(), inject.data_ptr(), T,
                                   out.data_ptr(), _stream(stream)))
        return out


class FfnLayer:
    """FfnExec::run(residual, out, add_shared, trace) (metal/include/strata/metal/layer_exec.hpp:135-137): gr_read of
    the residual streams, the MoE block, gr_write back onto the streams, in one smoe_ffn_run call.  Owns a workspace
    sized for `max_tokens`."""

    def __init__(self, g: Geom, weights: Dict, hc: HyperConnection, max_tokens: int, device="cuda"):
        import torch
        if hc.n_embd != g.n_embd:
            raise SmoeError(-1, f"hyper connection width {hc.n_embd} != n_embd {g.n_embd}")
        self.g, self.w, self.hc = g, weights, hc
        self._gc, self._wc = g.c(), _weights_c(weights)
        self.max_tokens = max_tokens
        self.ws_bytes = lib().smoe_ffn_workspace_bytes(C.byref(self._gc), C.byref(hc._c), max_tokens)
        if self.ws_bytes == 0:
            raise SmoeError(-1, lib().smoe_last_error().decode() or "bad geometry")
        self.ws = torch.empty(self.ws_bytes, dtype=torch.uint8, device=device)

    def run(self, residual, out=None, add_shared: bool = True, stream=None):
        import torch
        R = self.hc._stream_tensor(residual, "residual")
        T = R.shape[0]
        if T > self.max_tokens:
            raise SmoeError(-2, f"{T} tokens exceed the workspace's {self.max_tokens}")
        if out is None:
            out = torch.empty_like(R)
        _need(out, "out", torch.float32, numel=R.numel())
        _check(lib().smoe_ffn_run(C.byref(self._gc), C.byref(self._wc), C.byref(self.hc._c), R.data_ptr(), T,
                                  out.data_ptr(), int(add_shared), self.ws.data_ptr(), self.ws_bytes, None,
                                  _stream(stream)))
        return out

    __call__ = run


# ------------------------------------------------------------------------------------------------ dense layers

F32, F16, BF16 = 0, 1, 30  # SMOE_F32, SMOE_F16, SMOE_BF16
GATE_NONE, GATE_SIGMOID = 0, 1
ACT_NONE, ACT_SILU, ACT_GELU, ACT_RELU, ACT_RELU2, ACT_SIGMOID = range(6)


_ELEM: Dict = {}


def _elem_type(dtype) -> int:
    """The SMOE_F32 / F16 / BF16 number of a torch dtype (int16: bf16 bits, as elsewhere in this module), or -1."""
    if not _ELEM:
        import torch
        _ELEM.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16, torch.int16: BF16})
    return _ELEM.get(dtype, -1)


def _rows(t, name: str, n: int, tokens: int = -1, device: int = -1):
    """(type, row stride) of a (tokens, n) tensor on GPU `device` whose rows are contiguous, at any stride."""
    import torch
    if not isinstance(t, torch.Tensor):
        raise SmoeError(-1, f"{name} is not a tensor")
    code = _elem_type(t.dtype)
    if code < 0:
        raise SmoeError(-3, f"{name} is {t.dtype}, needs float32, float16 or bfloat16 (or int16: bf16 bits)")
    shape = t.shape
    if len(shape) != 2 or shape[1] != n or (tokens >= 0 and shape[0] != tokens):
        raise SmoeError(-2, f"{name} has shape {tuple(shape)}, needs ({'tokens' if tokens < 0 else tokens}, {n})")
    ld, step = t.stride()
    if step != 1 and n > 1:
        raise SmoeError(-5, f"{name}'s rows are not contiguous")
    _on_device(t, name, device)
    return code, ld


def _new(rows: int, n: int, dtype, device):
    """torch.empty((rows, n)), a third of its time on the host saved."""
    import torch
    return torch.empty_strided((rows, n), (n, 1), dtype=dtype, device=device)


def _on_device(t, name: str, device: int = -1):
    """Refuse a tensor that is on no GPU, or not on the call's."""
    at = t.get_device()
    if at < 0:
        raise SmoeError(-1, f"{name} is on {t.device}, not a GPU")
    if device >= 0 and at != device:
        raise SmoeError(-1, f"{name} is on {t.device}, the call's other tensors on cuda:{device}")


def _current(device: int, stream) -> Optional[int]:
    """The current stream's handle, when a call on `device` runs on it; None: under _on, which makes them current."""
    import torch
    if stream is None and torch._C._cuda_getDevice() == device:
        return torch._C._cuda_getCurrentRawStream(device)
    return None


def _on(device: int, stream):
    """The call's device, and its stream if one is given, current: its outputs and workspace are allocated for them."""
    import torch
    if stream is None:
        return torch.cuda.device(device)
    if stream.device_index != device:
        raise SmoeError(-1, f"the stream is on cuda:{stream.device_index}, the call's tensors on cuda:{device}")
    return torch.cuda.stream(stream)


def _vector(t, name: str, n: int):
    import torch
    return t if t is None else _need(t, name, torch.float32, shape=(n,))


class BlockEnds:
    """The ends of a block on one residual stream (smoe_block_ends), where HyperConnection has them on several: the norm
    after the block (weight `post`, None: no such norm), its gate, the residual scales, and the norm before the next block
    (weight `pre`, None: 1).  Between two blocks `post` is the one's and `pre` the next one's.  The weights are f32 [n_embd]
    tensors.  A call's rows are (tokens, n_embd) tensors of float32, float16 or bfloat16 with any row stride; the gate is
    float32 and broadcasts to them (one per channel, per token, or both)."""

    def __init__(self, n_embd: int, pre=None, post=None, res_scale: float = 1.0, y_scale: float = 1.0, eps: float = 1e-6,
                 gate_act: int = GATE_NONE):
        self.n_embd, self.pre, self.post = n_embd, _vector(pre, "pre", n_embd), _vector(post, "post", n_embd)
        weights = [t for t in (pre, post) if t is not None]
        self._device = weights[0].get_device() if weights else -1
        for t in weights:
            _on_device(t, "post", self._device)
        self._c = _Ends(_ptr(pre), _ptr(post), eps, res_scale, y_scale, gate_act)
        self._ref, self._call = C.byref(self._c), lib().smoe_block_ends

    def _run(self, R, y, gate, out, x, x_dtype, form, stream):
        import torch
        n = self.n_embd
        rt, r_ld = _rows(R, "R", n)
        T, dev = R.shape[0], R.get_device()
        st = _current(dev, stream)
        if st is None:
            with _on(dev, stream):
                return self._run(R, y, gate, out, x, x_dtype, form, None)
        if self._device >= 0 and self._device != dev:
            raise SmoeError(-1, f"the norms' weights are on cuda:{self._device}, the call's tensors on cuda:{dev}")
        yt = y_ld = o_ld = xt = x_ld = g_ld = g_step = 0
        yp = gp = op = xp = None
        if y is not None:
            yt, y_ld = _rows(y, "y", n, T, dev)
            yp = y.data_ptr()
            if out is None:
                out, o_ld = _new(T, n, R.dtype, R.device), n
            else:
                ot, o_ld = _rows(out, "out", n, T, dev)
                if ot != rt:
                    raise SmoeError(-1, f"out is {out.dtype}, needs {R.dtype}")
            op = out.data_ptr()
            if gate is not None:
                g_ld, g_step = self._gate(gate, T, dev)
                gp = gate.data_ptr()
        if form:
            if x is None:
                dtype = x_dtype or R.dtype
                xt = _elem_type(dtype)
                if xt < 0:
                    raise SmoeError(-3, f"x_dtype is {dtype}, needs float32, float16 or bfloat16 (or int16: bf16 bits)")
                x, x_ld = _new(T, n, dtype, R.device), n
            else:
                xt, x_ld = _rows(x, "x", n, T, dev)
            xp = x.data_ptr()
        _check(self._call(self._ref, n, T, R.data_ptr(), rt, r_ld, yp, yt, y_ld, gp, g_ld, g_step, op, o_ld, xp, xt, x_ld,
                          st))
        return out, x

    def _gate(self, gate, T: int, dev: int):
        """(token stride, channel stride) of a gate broadcast to (T, n_embd)."""
        import torch
        if gate.dtype != torch.float32:
            raise SmoeError(-1, f"gate is {gate.dtype}, needs torch.float32")
        _on_device(gate, "gate", dev)
        if gate.dim() == 1 and gate.shape[0] == self.n_embd:
            return 0, gate.stride(0)
        try:
            return gate.expand(T, self.n_embd).stride()
        except RuntimeError:
            raise SmoeError(-2, f"gate has shape {tuple(gate.shape)}, does not broadcast to ({T}, {self.n_embd})") from None

    def read(self, R, x=None, x_dtype=None, stream=None):
        """x = R rs(R) pre, a block's input from the stream (x_dtype None: R's)."""
        return self._run(R, None, None, None, x, x_dtype, True, stream)[1]

    def write(self, R, y, gate=None, out=None, stream=None):
        """out = res_scale R + y_scale g z, the block's output back onto the stream; `out` may be R."""
        return self._run(R, _given(y, "y"), gate, out, None, None, False, stream)[0]

    def join(self, R, y, gate=None, out=None, x=None, x_dtype=None, stream=None):
        """write, then read of the new stream (in f32, before its rounding), in one pass: (out, x)."""
        return self._run(R, _given(y, "y"), gate, out, x, x_dtype, True, stream)


def _given(t, name: str):
    if t is None:
        raise SmoeError(-6, f"{name} is None")
    return t


class Linear:
    """The dense product with its epilogue (smoe_linear_run): y = act(x w' + bias) [* (x w2' + bias2)] [+ residual].
    `w` and `w2` are (n_out, n_in) tensors (or flat ones of those rows) of bfloat16 (or int16: bf16 bits) or float16, the
    biases f32 [n_out].  The weights stay the caller's tensors."""

    def __init__(self, n_in: int, n_out: int, w, bias=None, w2=None, bias2=None, act: int = ACT_NONE):
        for t, name in ((w, "w"), (w2, "w2")):
            if t is not None:
                _need(t, name, w.dtype, shape=(n_in * n_out,) if getattr(t, "ndim", 2) == 1 else (n_out, n_in))
                _on_device(t, name, w.get_device())
        self.n_in, self.n_out, self.dtype = n_in, n_out, w.dtype
        self.tensors = (w, w2, _vector(bias, "bias", n_out), _vector(bias2, "bias2", n_out))
        for t, name in ((bias, "bias"), (bias2, "bias2")):
            if t is not None:
                _on_device(t, name, w.get_device())
        self._type = _elem_type(w.dtype)
        self._c = _Linear(n_in, n_out, self._type, act, w.data_ptr(), _ptr(w2), _ptr(bias), _ptr(bias2))
        self._ref, self._call = C.byref(self._c), lib().smoe_linear_run
        self._sizes: Dict = {}
        if lib().smoe_linear_workspace_bytes(self._ref, 0) == 0:
            raise SmoeError(-1, lib().smoe_last_error().decode())

    def workspace_bytes(self, n_tokens: int) -> int:
        return int(lib().smoe_linear_workspace_bytes(self._ref, n_tokens))

    def _bytes(self, T: int) -> int:
        """workspace_bytes, kept per batch size."""
        n = self._sizes.get(T)
        if n is None:
            n = self._sizes[T] = self.workspace_bytes(T)
        return n

    def run(self, x, residual=None, y=None, y_dtype=None, stream=None):
        """y (tokens, n_out) of `y_dtype` (None: residual's, else x's); `y` may be residual."""
        import torch
        w, N = self.tensors[0], self.n_out
        dev = w.get_device()
        xt, x_ld = _rows(x, "x", self.n_in, -1, dev)
        if xt != self._type:
            raise SmoeError(-1, f"x is {x.dtype}, the weights {self.dtype}")
        st = _current(dev, stream)
        if st is None:
            with _on(dev, stream):
                return self.run(x, residual, y, y_dtype)
        T = x.shape[0]
        rp, rt, r_ld = None, -1, 0
        if residual is not None:
            rt, r_ld = _rows(residual, "residual", N, T, dev)
            rp = residual.data_ptr()
        if y is None:
            dtype = y_dtype or (x if residual is None else residual).dtype
            yt = _elem_type(dtype)
            if yt < 0:
                raise SmoeError(-3, f"y_dtype is {dtype}, needs float32, float16 or bfloat16 (or int16: bf16 bits)")
            y, y_ld = _new(T, N, dtype, x.device), N
        else:
            yt, y_ld = _rows(y, "y", N, T, dev)
        if rt >= 0 and rt != yt:
            raise SmoeError(-1, f"residual is {residual.dtype}, y {y.dtype}")
        # a workspace of the call's own: calls on several streams, captured or not, share none
        n = self._bytes(T)
        ws = torch.empty_strided((n,), (1,), dtype=torch.uint8, device=x.device) if n > 256 else None
        _check(self._call(self._ref, x.data_ptr(), x_ld, T, rp, r_ld, y.data_ptr(), yt, y_ld, _ptr(ws), n, st))
        return y

    __call__ = run


class Linear4:
    """The product with 4-bit weights and group scales (smoe_linear4_run), with Linear's epilogue: y = act(x W' + bias)
    [* (x W2' + bias2)] [+ residual], W[o][i] = scales[i // group][o] (code[o][i] - zeros[i // group][o]).  `w` and `w2` are
    (n_out, n_in / 2) uint8 tensors of two codes to a byte, the even i's low; scales and scales2 (ceil(n_in / group), n_out) of
    float32, float16 or bfloat16; zeros and zeros2 uint8 of that shape (None: 8); the biases f32 [n_out].  The weights stay the
    caller's tensors; x is bfloat16 or float16."""

    def __init__(self, n_in: int, n_out: int, w, scales, zeros=None, group: int = 128, bias=None, w2=None, scales2=None,
                 zeros2=None, bias2=None, act: int = ACT_NONE):
        import torch
        if n_in < 32 or n_in % 32 or group < 32 or group % 32:
            raise SmoeError(-1, "n_in and group must be multiples of 32")
        for v, name in ((n_in, "n_in"), (n_out, "n_out"), (group, "group"), (act, "act")):
            _int32(v, name)
        groups = (-(-n_in // group), n_out)
        given = [(w, "w", torch.uint8, (n_out, n_in // 2)), (scales, "scales", None, groups), (zeros, "zeros", torch.uint8, groups),
                 (bias, "bias", torch.float32, (n_out,)), (w2, "w2", torch.uint8, (n_out, n_in // 2)),
                 (scales2, "scales2", None, groups), (zeros2, "zeros2", torch.uint8, groups), (bias2, "bias2", torch.float32, (n_out,))]
        _given(w, "w"), _given(scales, "scales")
        if (w2 is None) != (scales2 is None):
            raise SmoeError(-6, "w2 and scales2 go together")
        for t, name, dtype, shape in given:
            if t is not None:
                _need(t, name, dtype or scales.dtype, shape=shape)
                _on_device(t, name, w.get_device())
        self.n_in, self.n_out, self.group = n_in, n_out, group
        self.tensors = tuple(t for t, *_ in given)
        self._act, self._cs, self._call = act, {}, lib().smoe_linear4_run
        self._device = w.get_device()
        self._s_type = _elem_type(scales.dtype)
        if self._s_type < 0:
            raise SmoeError(-3, f"scales is {scales.dtype}, needs float32, float16 or bfloat16 (or int16: bf16 bits)")
        self._layer(BF16)

    def _layer(self, x_type: int):
        """(the C layer for x of that type, its reference, its workspace bytes per batch size)"""
        c = self._cs.get(x_type)
        if c is None:
            w, scales, zeros, bias, w2, scales2, zeros2, bias2 = (_ptr(t) for t in self.tensors)
            layer = _Linear4(self.n_in, self.n_out, x_type, self._act, self.group, self._s_type, w, w2, scales, scales2, zeros, zeros2,
                             bias, bias2)
            if lib().smoe_linear4_workspace_bytes(C.byref(layer), 0) == 0:
                raise SmoeError(-1, lib().smoe_last_error().decode())
            c = self._cs[x_type] = (layer, C.byref(layer), {})
        return c

    def workspace_bytes(self, n_tokens: int, dtype=None) -> int:
        layer = self._layer(BF16 if dtype is None else _elem_type(dtype))[1]
        return int(lib().smoe_linear4_workspace_bytes(layer, _int32(n_tokens, "n_tokens")))

    def run(self, x, residual=None, y=None, y_dtype=None, stream=None):
        """y (tokens, n_out) of `y_dtype` (None: residual's, else x's); `y` may be residual."""
        import torch
        N, dev = self.n_out, self._device
        xt, x_ld = _rows(x, "x", self.n_in, -1, dev)
        if xt == F32:
            raise SmoeError(-3, f"x is {x.dtype}, needs float16 or bfloat16 (or int16: bf16 bits)")
        st = _current(dev, stream)
        if st is None:
            with _on(dev, stream):
                return self.run(x, residual, y, y_dtype)
        T = x.shape[0]
        if T >> 31:
            _int32(T, "the number of tokens")
        rp, rt, r_ld = None, -1, 0
        if residual is not None:
            rt, r_ld = _rows(residual, "residual", N, T, dev)
            rp = residual.data_ptr()
        if y is None:
            dtype = y_dtype or (x if residual is None else residual).dtype
            yt = _elem_type(dtype)
            if yt < 0:
                raise SmoeError(-3, f"y_dtype is {dtype}, needs float32, float16 or bfloat16 (or int16: bf16 bits)")
            y, y_ld = _new(T, N, dtype, x.device), N
        else:
            yt, y_ld = _rows(y, "y", N, T, dev)
        if rt >= 0 and rt != yt:
            raise SmoeError(-1, f"residual is {residual.dtype}, y {y.dtype}")
        _, ref, sizes = self._layer(xt)
        n = sizes.get(T)
        if n is None:
            n = sizes[T] = int(lib().smoe_linear4_workspace_bytes(ref, T))
        ws = torch.empty_strided((n,), (1,), dtype=torch.uint8, device=x.device) if n > 256 else None
        _check(self._call(ref, x.data_ptr(), x_ld, T, rp, r_ld, y.data_ptr(), yt, y_ld, _ptr(ws), n, st))
        return y

    __call__ = run


# ------------------------------------------------------------------------------------------------ attention

ROPE_HALF, ROPE_PAIRS = 0, 1
_ROPE_SCALINGS = {"linear": 1, "ntk": 2, "parts": 3}


def rope_table(rot_dim: int, base: float = 10000.0, scaling=None):
    """(revolutions per position, a list of rot_dim / 2, and the scale on turned values) of smoe_rope_table.  `scaling`: None, or
    (kind, factor, ...) for contexts `factor` times as long as the trained ones: "linear" and "ntk" (the base grows) read the
    factor, "parts" also the trained length and the slow and fast ends in turns over it."""
    kind, factor, trained, slow, fast = (tuple(scaling) + (0.0, 0.0, 0.0))[:5] if scaling else ("", 1.0, 0.0, 0.0, 0.0)
    if scaling and kind not in _ROPE_SCALINGS:
        raise SmoeError(-1, f"scaling is {kind!r}, needs one of {sorted(_ROPE_SCALINGS)}")
    if rot_dim < 2 or rot_dim > 1024 or rot_dim % 2:
        raise SmoeError(-1, "rot_dim must be even, 2 to 1024")
    turns, scale = (C.c_double * (rot_dim // 2))(), C.c_float()
    _check(lib().smoe_rope_table(rot_dim, base, _ROPE_SCALINGS.get(kind, 0), factor, trained, slow, fast, turns, C.byref(scale)))
    return list(turns), scale.value


def _heads(t, name: str, heads: int, dim: int, tokens: int = -1, device: int = -1):
    """(type, token stride) of a (tokens, heads, dim) tensor whose tokens' values are contiguous, at any stride."""
    import torch
    if not isinstance(t, torch.Tensor):
        raise SmoeError(-1, f"{name} is not a tensor")
    code = _elem_type(t.dtype)
    if code < 0:
        raise SmoeError(-3, f"{name} is {t.dtype}, needs float32, float16 or bfloat16 (or int16: bf16 bits)")
    shape = t.shape
    if len(shape) != 3 or shape[2] != dim or (heads >= 0 and shape[1] != heads) or (tokens >= 0 and shape[0] != tokens):
        raise SmoeError(-2, f"{name} has shape {tuple(shape)}, needs ({'tokens' if tokens < 0 else tokens}, "
                            f"{'heads' if heads < 0 else heads}, {dim})")
    if shape[0] >> 31 or shape[1] >> 31:
        _int32(max(shape[0], shape[1]), f"a size of {name}")
    ld, step, one = t.stride()
    if one != 1 or (step != dim and shape[1] > 1):
        raise SmoeError(-5, f"a token's values of {name} are not contiguous")
    if device < 0 or t.get_device() != device:
        _on_device(t, name, device)
    return code, ld


def _flat(t, name: str, dtype, n: int, device: int) -> int:
    """The address of an (n,) tensor of `dtype` on GPU `device`: _need and _on_device, most calls with less on the host."""
    try:
        if t.dtype is dtype and t.get_device() == device >= 0 and t.dim() == 1 and t.shape[0] == n and t.is_contiguous():
            return t.data_ptr()
    except AttributeError:
        pass
    _need(t, name, dtype, shape=(n,))
    _on_device(t, name, device)
    return t.data_ptr()


def _new_heads(tokens: int, heads: int, dim: int, dtype, device):
    import torch
    return torch.empty_strided((tokens, heads, dim), (heads * dim, dim, 1), dtype=dtype, device=device)


class Rotary:
    """Rotary positions (smoe_rope_run): the first `rot_dim` (None: all) values of heads of `head_dim` turned in pairs that lie
    half of them apart (ROPE_HALF) or side by side (ROPE_PAIRS), the frequencies from `base` and `scaling` (rope_table), or
    `turns`, the revolutions per position of each pair, with `scale` on turned values.  Positions are int32 tensors; at -p a call
    is the transpose of the one at p."""

    def __init__(self, head_dim: int, rot_dim: Optional[int] = None, base: float = 10000.0, layout: int = ROPE_HALF, scaling=None,
                 turns=None, scale: Optional[float] = None, device="cuda"):
        import torch
        rot_dim = head_dim if rot_dim is None else rot_dim
        for v, name in ((head_dim, "head_dim"), (rot_dim, "rot_dim"), (layout, "layout")):
            _int32(v, name)
        if turns is None:
            turns, own_scale = rope_table(rot_dim, base, scaling)
        else:
            own_scale = 1.0
        self.turns = torch.as_tensor(turns, dtype=torch.float64).to(device).contiguous()
        if self.turns.shape != (rot_dim // 2,):
            raise SmoeError(-2, f"turns has shape {tuple(self.turns.shape)}, needs ({rot_dim // 2},)")
        _on_device(self.turns, "turns")
        self.head_dim, self.rot_dim, self.scale = head_dim, rot_dim, own_scale if scale is None else scale
        self._c = _Rope(head_dim, rot_dim, layout, self.scale, self.turns.data_ptr())
        self._ref, self._device, self._call = C.byref(self._c), self.turns.get_device(), lib().smoe_rope_run
        # (a call without tokens: the sizes alone are checked)
        _check(lib().smoe_rope_run(self._ref, None, 0, 1, None, F32, 0, None, F32, 0, None))

    def run(self, x, positions, y=None, y_dtype=None, stream=None):
        """y (tokens, heads, head_dim) of `y_dtype` (None: x's); `y` may be x."""
        import torch
        xt, x_ld = _heads(x, "x", -1, self.head_dim, -1, self._device)
        T, H, _ = x.shape
        st = _current(self._device, stream)
        if st is None:
            with _on(self._device, stream):
                return self.run(x, positions, y, y_dtype)
        pp = _flat(positions, "positions", torch.int32, T, self._device)
        if y is None:
            dtype = y_dtype or x.dtype
            yt, y_ld = _elem_type(dtype), H * self.head_dim
            if yt < 0:
                raise SmoeError(-3, f"y_dtype is {dtype}, needs float32, float16 or bfloat16 (or int16: bf16 bits)")
            y = _new_heads(T, H, self.head_dim, dtype, x.device)
        else:
            yt, y_ld = _heads(y, "y", H, self.head_dim, T, self._device)
        _check(self._call(self._ref, pp, T, H, x.data_ptr(), xt, x_ld, y.data_ptr(), yt, y_ld, st))
        return y

    __call__ = run


class PagedCache:
    """A cache of keys and values in pages: `k` and `v` are (pages, key heads, tokens of a page, head_dim) tensors of bfloat16 (or
    int16: bf16 bits) or float16.  They stay the caller's tensors."""

    def __init__(self, k, v):
        _given(k, "k"), _given(v, "v")
        if getattr(k, "ndim", 0) != 4:
            raise SmoeError(-2, "k must be (pages, key heads, tokens of a page, head_dim)")
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = (_int32(n, "a size of the cache") for n in k.shape)
        for t, name in ((k, "k"), (v, "v")):
            _need(t, name, k.dtype, shape=k.shape)
            _on_device(t, name, k.get_device())
        self.k, self.v = k, v
        self._type, self._device = _elem_type(k.dtype), k.get_device()
        self._c = _Kv(k.data_ptr(), v.data_ptr(), self._type, *(int(k.shape[i]) for i in (0, 2, 1, 3)))
        self._ref = C.byref(self._c)
        self._sizes: Dict = {}
        self._append, self._attend = lib().smoe_kv_append, lib().smoe_attend
        # (a call without tokens: the sizes alone are checked)
        _check(self._append(self._ref, None, None, None, 0, F32, None, 0, 0, None, 0, None, 0, None, 0, None))

    @classmethod
    def empty(cls, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, dtype=None, device="cuda"):
        """A new cache (its pages' values are any until they are written)."""
        import torch
        k, v = (torch.empty((n_pages, n_kv_heads, page_size, head_dim), dtype=dtype or torch.bfloat16, device=device) for _ in "kv")
        return cls(k, v)

    def append(self, k, v, slots, rotary: Optional[Rotary] = None, positions=None, q=None, q_out=None, stream=None):
        """Writes (tokens, key heads, head_dim) tensors k and v to `slots` (int64: page * page_size + place, one outside the cache
        as -1: not stored), k turned to `positions` when `rotary` is given, and returns q (tokens, heads, head_dim) turned, of the
        cache's type (None without q); `q_out` may be q.  A call's slots are distinct (smoe_kv_append)."""
        import torch
        dev, D, kv = self._device, self.head_dim, self.n_kv_heads
        xt, k_ld = _heads(k, "k", kv, D, -1, dev)
        T = k.shape[0]
        vt, v_ld = _heads(v, "v", kv, D, T, dev)
        st = _current(dev, stream)
        if st is None:
            with _on(dev, stream):
                return self.append(k, v, slots, rotary, positions, q, q_out)
        sp = _flat(slots, "slots", torch.int64, T, dev)
        rp = pp = qp = op = None
        q_ld = o_ld = H = 0
        if rotary is not None:
            rp, pp = rotary._ref, _flat(_given(positions, "positions"), "positions", torch.int32, T, dev)
            if rotary._device != dev:
                raise SmoeError(-1, f"the rotary positions' table is on cuda:{rotary._device}, the cache on cuda:{dev}")
        qt = xt
        if q is not None:
            if rotary is None:
                raise SmoeError(-6, "q without rotary positions")
            qt, q_ld = _heads(q, "q", -1, D, T, dev)
            H = q.shape[1]
            if q_out is None:
                q_out, o_ld = _new_heads(T, H, D, self.k.dtype, q.device), H * D
            else:
                ot, o_ld = _heads(q_out, "q_out", H, D, T, dev)
                if ot != self._type:
                    raise SmoeError(-1, f"q_out is {q_out.dtype}, the cache {self.k.dtype}")
            qp, op = q.data_ptr(), q_out.data_ptr()
        elif q_out is not None:
            raise SmoeError(-6, "q_out without q")
        if vt != xt or qt != xt:
            raise SmoeError(-1, f"q, k and v are of one type, k is {k.dtype}")
        _check(self._append(self._ref, rp, pp, sp, T, xt, qp, q_ld, H, op, o_ld, k.data_ptr(), k_ld, v.data_ptr(), v_ld, st))
        return q_out

    def workspace_bytes(self, n_heads: int, n_tokens: int, n_seqs: int, max_len: int, window: int = 0) -> int:
        for v, name in ((n_heads, "n_heads"), (n_tokens, "n_tokens"), (n_seqs, "n_seqs"), (max_len, "max_len"), (window, "window")):
            _int32(v, name)
        return int(lib().smoe_attend_workspace_bytes(self._ref, n_heads, n_tokens, n_seqs, max_len, window))

    def attend(self, q, q_start, kv_len, pages, scale: Optional[float] = None, causal: bool = True, window: int = 0,
               lse: bool = False, max_len: Optional[int] = None, out=None, stream=None):
        """out (tokens, heads, head_dim): attention of q's rows q_start[b] .. q_start[b + 1] - 1 over the first kv_len[b] keys of
        the pages pages[b] (smoe_attend), `scale` None: head_dim ** -0.5; with `lse` (out, lse (tokens, heads) f32).  q_start
        (sequences + 1,), kv_len (sequences,) and pages (sequences, most pages) are int32 tensors; keys past max_len (None: what
        the pages hold) are not there: the tighter it is, the fewer empty work-groups.  Rows of no sequence are left as they are (new outputs: any
        values)."""
        import torch
        dev, D = self._device, self.head_dim
        qt, q_ld = _heads(q, "q", -1, D, -1, dev)
        if qt != self._type:
            raise SmoeError(-1, f"q is {q.dtype}, the cache {self.k.dtype}")
        st = _current(dev, stream)
        if st is None:
            with _on(dev, stream):
                return self.attend(q, q_start, kv_len, pages, scale, causal, window, lse, max_len, out)
        T, H, _ = q.shape
        B = kv_len.shape[0] if getattr(kv_len, "ndim", 0) == 1 else -1
        lp, sp = _flat(kv_len, "kv_len", torch.int32, B, dev), _flat(q_start, "q_start", torch.int32, B + 1, dev)
        if not isinstance(pages, torch.Tensor) or pages.dtype != torch.int32:
            raise SmoeError(-1, "pages must be an int32 tensor")
        width = pages.shape[1] if pages.dim() == 2 and pages.shape[0] == B else -1
        if width < 0:
            raise SmoeError(-2, f"pages has shape {tuple(pages.shape)}, needs ({B}, most pages)")
        p_ld, p_step = pages.stride()
        if p_step != 1 and width > 1:
            raise SmoeError(-5, "pages' rows are not contiguous")
        if pages.get_device() != dev:
            _on_device(pages, "pages", dev)
        if width >> 31:
            _int32(width, "the pages' width")
        held = min(width * self.page_size, 1 << 30)
        max_len = held if max_len is None else max_len
        if out is None:
            out, o_ld = _new_heads(T, H, D, q.dtype, q.device), H * D
        else:
            ot, o_ld = _heads(out, "out", H, D, T, dev)
            if ot != qt:
                raise SmoeError(-1, f"out is {out.dtype}, q {q.dtype}")
        z = torch.empty_strided((T, H), (H, 1), dtype=torch.float32, device=q.device) if lse else None
        key = (H, T, B, max_len, window)
        n = self._sizes.get(key)
        if n is None:
            n = self.workspace_bytes(*key)
            if n == 0:
                raise SmoeError(-1, lib().smoe_last_error().decode())
            if len(self._sizes) >= 4096:
                self._sizes.clear()
            self._sizes[key] = n
        # a workspace of the call's own: calls on several streams, captured or not, share none
        ws = torch.empty_strided((n,), (1,), dtype=torch.uint8, device=q.device) if n > 256 else None
        _check(self._attend(self._ref, q.data_ptr(), q_ld, T, H, sp, lp, B, pages.data_ptr(), p_ld, width, max_len,
                            D ** -0.5 if scale is None else scale, int(bool(causal)), window, out.data_ptr(), o_ld, _ptr(z), _ptr(ws), n, st))
        return (out, z) if lse else out


# ------------------------------------------------------------------------------------------------ stages

def router_balance(logits, ids, mask=None, balance_coef: float = 1.0, z_coef: float = 0.0, grad: bool = False, stream=None):
    """The router's load over a batch (smoe_router_balance): a dict of loss [4] = (balance_coef balance + z_coef z, balance,
    z, tokens counted), counts [E] (int32) and mean_p [E]; with `grad` also dlogits [T][E] and dbias [E], the gradients of
    loss[0] to the logits and to a bias added to them.  logits (T, E) f32 with any row stride, ids (T, k) int32 as
    router_topk selects them, mask (T,) bool or uint8: the tokens that count."""
    import torch
    if logits.dim() != 2:
        raise SmoeError(-1, "logits must be (tokens, experts)")
    T, E = logits.shape
    if logits.dtype != torch.float32:
        raise SmoeError(-1, f"logits is {logits.dtype}, needs torch.float32")
    _, ld = _rows(logits, "logits", E)
    dev = logits.get_device()
    st = _current(dev, stream)
    if st is None:
        with _on(dev, stream):
            return router_balance(logits, ids, mask, balance_coef, z_coef, grad)
    _need(ids, "ids", torch.int32)
    _on_device(ids, "ids", dev)
    if ids.dim() != 2 or ids.shape[0] != T:
        raise SmoeError(-2, f"ids has shape {tuple(ids.shape)}, needs ({T}, k)")
    if mask is not None:
        _need(mask, "mask", torch.uint8 if mask.dtype == torch.uint8 else torch.bool, shape=(T,))
        _on_device(mask, "mask", dev)
    at, new, f32 = logits.device, torch.empty_strided, torch.float32
    loss, counts = new((4,), (1,), dtype=f32, device=at), new((E,), (1,), dtype=torch.int32, device=at)
    mean_p = new((E,), (1,), dtype=f32, device=at)
    out = dict(loss=loss, counts=counts, mean_p=mean_p)
    dp = bp = None
    if grad:
        out["dlogits"], out["dbias"] = _new(T, E, f32, at), new((E,), (1,), dtype=f32, device=at)
        dp, bp = out["dlogits"].data_ptr(), out["dbias"].data_ptr()
    if T == 0:
        for t in out.values():
            t.zero_()
    n = lib().smoe_router_balance_workspace_bytes(T, E)
    if n == 0 and T > 0:
        raise SmoeError(-1, lib().smoe_last_error().decode())
    ws = new((n,), (1,), dtype=torch.uint8, device=at)
    _check(lib().smoe_router_balance(logits.data_ptr(), ld, ids.data_ptr(), _ptr(mask), T, E, ids.shape[1], balance_coef,
                                     z_coef, loss.data_ptr(), counts.data_ptr(), mean_p.data_ptr(), dp, E, bp, ws.data_ptr(), n, st))
    return out


def router_topk(logits, k: int, stream=None):
    import torch
    if logits.dim() != 2:
        raise SmoeError(-1, "logits must be (tokens, experts)")
    T, E = logits.shape
    _need(logits, "logits", torch.float32)
    ids = torch.empty((T, k), dtype=torch.int32, device=logits.device)
    w = torch.empty((T, k), dtype=torch.float32, device=logits.device)
    _check(lib().smoe_router_topk(logits.data_ptr(), T, E, k, ids.data_ptr(), w.data_ptr(), _stream(stream)))
    return ids, w


def router_margin(logits, k: int, stream=None):
    """The router-margin diagnostic (smoe_router_margin): stats (T, 4) = (p_k - p_k1, logit gap, p_k, p_k1) and
    ids (T, 2) = (id_k, id_k1) of the k-th and (k+1)-th experts by softmax probability."""
    import torch
    if logits.dim() != 2:
        raise SmoeError(-1, "logits must be (tokens, n_expert)")
    _need(logits, "logits", torch.float32)
    T, E = logits.shape
    stats = torch.empty((T, 4), dtype=torch.float32, device=logits.device)
    ids = torch.empty((T, 2), dtype=torch.int32, device=logits.device)
    _check(lib().smoe_router_margin(logits.data_ptr(), T, E, k, stats.data_ptr(), ids.data_ptr(), _stream(stream)))
    return stats, ids


def f32_to_bf16(x, stream=None):
    import torch
    _need(x, "x", torch.float32)
    y = torch.empty(x.shape, dtype=torch.int16, device=x.device)
    _check(lib().smoe_f32_to_bf16(x.data_ptr(), x.numel(), y.data_ptr(), _stream(stream)))
    return y


def bf16_gemv(x_bf16, w_bf16, n_in: int, n_out: int, stream=None):
    import torch
    _need(x_bf16, "x_bf16", torch.int16)
    _need(w_bf16, "w_bf16", torch.int16, numel=n_in * n_out)
    if n_in <= 0 or x_bf16.numel() % n_in:
        raise SmoeError(-1, f"x_bf16 holds {x_bf16.numel()} values, not whole rows of {n_in}")
    n_tok = x_bf16.numel() // n_in
    y = torch.empty((n_tok, n_out), dtype=torch.float32, device=x_bf16.device)
    _check(lib().smoe_bf16_gemv(x_bf16.data_ptr(), w_bf16.data_ptr(), y.data_ptr(), n_in, n_out, n_tok,
                                _stream(stream)))
    return y


def quantize_q8_1(x, stream=None):
    import torch
    _need(x, "x", torch.float32)
    y = torch.empty(x.numel() // 32 * 36, dtype=torch.uint8, device=x.device)
    _check(lib().smoe_quantize_q8_1(x.data_ptr(), x.numel(), y.data_ptr(), _stream(stream)))
    return y


def mmvq(wtype: int, w, x_q8, n_in: int, n_out: int, n_col: int = 1, byte_off: int = 0, stream=None):
    import torch
    _need(w, "w", torch.uint8, numel=byte_off + n_out * row_bytes(wtype, n_in))
    _need(x_q8, "x_q8", torch.uint8, numel=n_col * (n_in // 32) * 36)
    y = torch.empty((n_col, n_out), dtype=torch.float32, device=w.device)
    _check(lib().smoe_mmvq(wtype, w.data_ptr(), byte_off, x_q8.data_ptr(), n_in, n_out, n_col, y.data_ptr(),
                           _stream(stream)))
    return y


def expert(blob, x_q8, gu_type: int, d_type: int, n_embd: int, n_ff: int, n_tok: int, stream=None):
    """One expert's FFN on a [gate | up | down] blob (smoe_expert; the reference's iq_expert)."""
    import torch
    _need(blob, "blob", torch.uint8)
    _need(x_q8, "x_q8", torch.uint8, numel=n_tok * (n_embd // 32) * 36)
    L = lib()
    scratch = torch.empty(L.smoe_expert_scratch_bytes(n_embd, n_ff, n_tok) + 256, dtype=torch.uint8,
                          device=blob.device)
    base = (scratch.data_ptr() + 255) & ~255
    y = torch.empty((n_tok, n_embd), dtype=torch.float32, device=blob.device)
    _check(L.smoe_expert(blob.data_ptr(), blob.numel(), x_q8.data_ptr(), gu_type, d_type, n_embd, n_ff, n_tok,
                         y.data_ptr(), base, scratch.numel() - (base - scratch.data_ptr()), _stream(stream)))
    return y


def residual_rmsnorm(x, r=None, eps: float = 1e-6, out=None, stream=None):
    """RMSNorm(x + r) row by row with unit weight (smoe_residual_rmsnorm); `out` may be `x`."""
    import torch
    _need(x, "x", torch.float32)
    n = x.shape[-1]
    if r is not None:
        _need(r, "r", torch.float32, shape=x.shape)
    out = torch.empty_like(x) if out is None else out
    _need(out, "out", torch.float32, shape=x.shape)
    _check(lib().smoe_residual_rmsnorm(x.data_ptr(), _ptr(r), x.numel() // n, n, eps, out.data_ptr(), _stream(stream)))
    return out


def swiglu_q8(gate, up, stream=None):
    import torch
    _need(gate, "gate", torch.float32)
    _need(up, "up", torch.float32, shape=gate.shape)
    y = torch.empty(gate.numel() // 32 * 36, dtype=torch.uint8, device=gate.device)
    _check(lib().smoe_swiglu_q8(gate.data_ptr(), up.data_ptr(), gate.numel(), y.data_ptr(), _stream(stream)))
    return y


def combine(parts, weights, shared=None, stream=None):
    import torch
    if parts.dim() != 2:
        raise SmoeError(-1, "parts must be (k, n_embd)")
    _need(parts, "parts", torch.float32)
    k, n = parts.shape
    _need(weights, "weights", torch.float32, numel=k)
    if shared is not None:
        _need(shared, "shared", torch.float32, numel=n)
    y = torch.empty(n, dtype=torch.float32, device=parts.device)
    _check(lib().smoe_combine(parts.data_ptr(), weights.data_ptr(), _ptr(shared), y.data_ptr(), n, k,
                              _stream(stream)))
    return y


def dispatch(ids, n_expert: int, stream=None):
    import torch
    if ids.dim() != 2:
        raise SmoeError(-1, "ids must be (tokens, k)")
    _need(ids, "ids", torch.int32)
    T, k = ids.shape
    dev = ids.device
    counts = torch.empty(n_expert, dtype=torch.int32, device=dev)
    offsets = torch.empty(n_expert + 1, dtype=torch.int32, device=dev)
    perm = torch.empty(T * k, dtype=torch.int32, device=dev)
    slot = torch.empty(T * k, dtype=torch.int32, device=dev)
    _check(lib().smoe_dispatch(ids.data_ptr(), T, k, n_expert, counts.data_ptr(), offsets.data_ptr(),
                               perm.data_ptr(), slot.data_ptr(), _stream(stream)))
    return counts, offsets, perm, slot


# ------------------------------------------------------------------------------------------------ GGUF models

class _TensorInfo(C.Structure):
    _fields_ = [("type", C.c_int32), ("n_dims", C.c_int32), ("shard", C.c_int32), ("reserved", C.c_int32),
                ("ne", C.c_uint64 * 4), ("bytes", C.c_uint64), ("file_offset", C.c_uint64), ("host", C.c_void_p)]


class _LayerPlan(C.Structure):
    _fields_ = [("geom", _Geom), ("hc", _Hc), ("device_bytes", C.c_size_t), ("off", C.c_size_t * 12),
                ("layer", C.c_int32), ("with_shared", C.c_int32)]


@dataclass
class TensorInfo:
    name: str
    type: int
    shape: tuple           # GGUF order: shape[0] is a row
    shard: int
    bytes: int
    file_offset: int


class Model:
    """A GGUF v3 model on the host (smoe_model_*: every shard of a split model, mapped read-only), its tensors by
    name, its metadata, and one layer's MoE tensors loaded into device memory (smoe_layer_plan_for /
    smoe_layer_upload, the tensor side of the reference's FfnExec::load)."""

    def __init__(self, path: str):
        self._h = C.c_void_p()
        _check(lib().smoe_model_open(path.encode(), C.byref(self._h)))

    def close(self):
        if self._h:
            lib().smoe_model_close(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def n_shards(self) -> int:
        return int(lib().smoe_model_n_shards(self._h))

    def _info(self, name: str, ti: _TensorInfo) -> TensorInfo:
        return TensorInfo(name, ti.type, tuple(int(ti.ne[d]) for d in range(ti.n_dims)), ti.shard, int(ti.bytes),
                          int(ti.file_offset))

    def tensors(self):
        out = []
        for i in range(int(lib().smoe_model_n_tensors(self._h))):
            buf = C.create_string_buffer(4096)
            ti = _TensorInfo()
            _check(lib().smoe_model_tensor_at(self._h, i, buf, 4096, C.byref(ti)))
            out.append(self._info(buf.value.decode(), ti))
        return out

    def tensor(self, name: str) -> TensorInfo:
        ti = _TensorInfo()
        _check(lib().smoe_model_tensor(self._h, name.encode(), C.byref(ti)))
        return self._info(name, ti)

    def tensor_bytes(self, name: str) -> bytes:
        """The payload as the mapping holds it (a copy)."""
        ti = _TensorInfo()
        _check(lib().smoe_model_tensor(self._h, name.encode(), C.byref(ti)))
        return C.string_at(ti.host, ti.bytes)

    def meta_u64(self, key: str) -> int:
        v = C.c_uint64()
        _check(lib().smoe_model_meta_u64(self._h, key.encode(), C.byref(v)))
        return int(v.value)

    def meta_str(self, key: str) -> str:
        buf = C.create_string_buffer(1 << 16)
        _check(lib().smoe_model_meta_str(self._h, key.encode(), buf, 1 << 16))
        return buf.value.decode()

    def plan(self, layer: int, top_k: int = 0, with_shared: bool = True) -> _LayerPlan:
        p = _LayerPlan()
        _check(lib().smoe_layer_plan_for(self._h, layer, top_k, int(with_shared), C.byref(p)))
        return p

    def load_layer(self, layer: int, top_k: int = 0, with_shared: bool = True, with_hc: bool = False,
                   device="cuda", stream=None):
        """(Geom, weights dict of device tensors, HyperConnection or None) of one layer; the weights are views of
        one device buffer the returned dict also keeps (key "_buffer")."""
        import torch
        p = self.plan(layer, top_k, with_shared)
        buf = torch.empty(p.device_bytes + 256, dtype=torch.uint8, device=device)
        base = (buf.data_ptr() + 255) & ~255
        w, hc = _Weights(), _Hc()
        _check(lib().smoe_layer_upload(self._h, C.byref(p), base, p.device_bytes, C.byref(w),
                                       C.byref(hc) if with_hc else None, _stream(stream)))
        gc = p.geom
        g = Geom(gc.n_embd, gc.n_ff, gc.n_ff_shared, gc.n_expert, gc.top_k, gc.w_type, gc.sh_type, gc.router_dtype,
                 gc.sh_gate_type, gc.sh_up_type, gc.sh_down_type)

        def view(ptr, nbytes):
            o = ptr - buf.data_ptr()
            return buf[o:o + nbytes]

        H, F, E, Fs = g.n_embd, g.n_ff, g.n_expert, g.n_ff_shared
        sizes = dict(gate_exps=E * F * row_bytes(g.w_type, H), up_exps=E * F * row_bytes(g.w_type, H),
                     down_exps=E * H * row_bytes(g.w_type, F),
                     router=E * H * (4 if g.router_dtype == ROUTER_F32 else 2))
        weights = {n: view(getattr(w, n), sizes[n]) for n in sizes}
        if with_shared:
            weights.update(gate_sh=view(w.gate_sh, Fs * row_bytes(g.sh_gate_type, H)),
                           up_sh=view(w.up_sh, Fs * row_bytes(g.sh_up_type, H)),
                           down_sh=view(w.down_sh, H * row_bytes(g.sh_down_type, Fs)),
                           gate_inp_sh=view(w.gate_inp_sh, H * 2))
        weights["_buffer"] = buf
        hcx = None
        if with_hc:
            hd = hc.hc * H
            hcx = HyperConnection(H, hc.hc, hc.hc_lr, view(hc.norm, hd * 4).view(torch.float32),
                                  view(hc.down, hc.hc_lr * hd * 2).view(torch.int16),
                                  view(hc.up, hd * hc.hc_lr * 2).view(torch.int16),
                                  view(hc.inject, hc.hc * hd * 2).view(torch.int16), eps=float(hc.eps))
        return g, weights, hcx


# ------------------------------------------------------------------------------------------------ expert tier

def expert_blob_bytes(g: Geom) -> int:
    """Bytes of one routed expert's blob [gate rows | up rows | down rows] (smoe_expert_blob_bytes)."""
    n = int(lib().smoe_expert_blob_bytes(C.byref(g.c())))
    if n == 0:
        raise SmoeError(-1, lib().smoe_last_error().decode())
    return n


def pack_expert(g: Geom, weights: Dict, expert: int, blob, stream=None):
    """Copies expert `expert`'s rows from the planes in `weights` into `blob` (uint8, expert_blob_bytes)."""
    import torch
    _need(blob, "blob", torch.uint8, numel=expert_blob_bytes(g))
    _check(lib().smoe_expert_pack(C.byref(g.c()), C.byref(_weights_c(weights)), expert, blob.data_ptr(),
                                  _stream(stream)))
    return blob


def expert_table(ptrs, device="cuda"):
    """A device table of one blob address per expert (0: not held) from a list of tensors or None."""
    import torch
    a = [0 if t is None else t.data_ptr() for t in ptrs]
    return torch.tensor(a, dtype=torch.int64, device=device)


def expert_group(ids, k_per_tok: int, n_expert: int, table, stream=None) -> Dict:
    """The hit/miss split of the routed entries `ids` (int32, T * k_per_tok) by the expert table (int64 device
    addresses, 0 = not held), on the device (smoe_expert_group): grp_ptr, grp_expert, grp_start, ent_dst,
    ent_tok, miss_dst and counts {groups, hits, misses, 0}.  The lists are views of two allocations."""
    import torch
    _need(ids, "ids", torch.int32)
    _need(table, "table", torch.int64, numel=n_expert)
    n = ids.numel()
    G = max(1, min(n, n_expert))
    dev, m = ids.device, max(n, 1)
    # two fills, not one per list: the lists that start as zeros and those that start as -1
    ptr, start, counts = _parts(torch.zeros(2 * G + G + 1 + 4, dtype=torch.int32, device=dev), 2 * G, G + 1, 4)
    expert, dst, tok, miss = _parts(torch.full((G + 3 * m,), -1, dtype=torch.int32, device=dev), G, m, m, m)
    out = dict(grp_ptr=ptr.view(torch.int64), grp_expert=expert, grp_start=start, ent_dst=dst, ent_tok=tok,
               miss_dst=miss, counts=counts)
    _check(lib().smoe_expert_group(ids.data_ptr(), n, k_per_tok, n_expert, table.data_ptr(),
                                   out["grp_ptr"].data_ptr(), out["grp_start"].data_ptr(),
                                   out["grp_expert"].data_ptr(), out["ent_dst"].data_ptr(), out["ent_tok"].data_ptr(),
                                   out["miss_dst"].data_ptr(), out["counts"].data_ptr(), _stream(stream)))
    return out


def expert_grouped(g: Geom, groups: Dict, x_q8, n_tokens: int, out, cap_groups: int = None, cap_entries: int = None,
                   stream=None):
    """Grouped expert evaluation (smoe_expert_grouped) over the lists in `groups` (expert_group's keys): each
    entry's expert output row written to out[ent_dst] (out: (rows, n_embd) f32)."""
    import torch
    cg = groups["grp_ptr"].numel() if cap_groups is None else cap_groups
    ce = groups["ent_dst"].numel() if cap_entries is None else cap_entries
    # the kernels read the lists up to the caps: every list must hold them
    lists = (("grp_ptr", torch.int64, cg), ("grp_start", torch.int32, cg + 1), ("ent_dst", torch.int32, ce),
             ("ent_tok", torch.int32, ce), ("counts", torch.int32, 2))
    for key, _, n in lists:
        if groups[key].numel() < n:
            raise SmoeError(-2, f"{key} has {groups[key].numel()} elements, needs {n}")
    if out.dim() != 2 or out.shape[1] != g.n_embd:
        raise SmoeError(-2, f"out has shape {tuple(out.shape)}, needs (rows, {g.n_embd})")
    for key, dtype, n in lists:
        _need(groups[key], key, dtype, numel=n)
    _need(x_q8, "x_q8", torch.uint8, numel=n_tokens * (g.n_embd // 32) * 36)
    _need(out, "out", torch.float32)
    gc = C.byref(g.c())
    nb = int(lib().smoe_expert_grouped_workspace_bytes(gc, n_tokens, cg, ce))
    ws = torch.empty(max(nb, 1), dtype=torch.uint8, device=out.device)
    _check(lib().smoe_expert_grouped(gc, groups["grp_ptr"].data_ptr(), groups["grp_start"].data_ptr(),
                                     groups["ent_dst"].data_ptr(), groups["ent_tok"].data_ptr(),
                                     groups["counts"].data_ptr(), cg, ce, x_q8.data_ptr(), n_tokens, out.data_ptr(),
                                     out.shape[0], ws.data_ptr(), nb, _stream(stream)))
    return out


class VerifyWindow:
    """The verify window with the hit/miss split (smoe_verify_begin / smoe_verify_end): `begin` routes the tokens,
    computes the hits from the expert table and the shared expert into rows, and returns the misses for the caller
    to fill (miss_dst and counts, views of one small allocation); `end` combines the rows into y."""

    def __init__(self, g: Geom, weights: Dict, max_tokens: int, device="cuda"):
        import torch
        self.g, self.w = g, weights
        self._gc, self._wc = g.c(), _weights_c(weights)
        self.ws_bytes = int(lib().smoe_verify_workspace_bytes(C.byref(self._gc), max_tokens))
        if self.ws_bytes == 0:
            raise SmoeError(-1, f"verify window refused for {max_tokens} tokens: {lib().smoe_last_error().decode()}")
        self.ws = torch.empty(self.ws_bytes, dtype=torch.uint8, device=device)
        self.max_tokens = max_tokens

    def begin(self, x, table, stream=None) -> Dict:
        import torch
        _need(x, "x", torch.float32)
        T, H, K = x.shape[0], self.g.n_embd, self.g.top_k
        if x.dim() != 2 or x.shape[1] != H:
            raise SmoeError(-2, f"x has shape {tuple(x.shape)}, needs (tokens, {H})")
        if T > self.max_tokens:
            raise SmoeError(-1, f"{T} tokens exceed the window's {self.max_tokens}")
        _need(table, "table", torch.int64, numel=self.g.n_expert)
        dev, m = x.device, max(T * K, 1)
        # the split writes every count; -1 is what the entries past the misses hold
        miss, counts = _parts(torch.full((m + 4,), -1, dtype=torch.int32, device=dev), m, 4)
        if T == 0:
            counts.zero_()
        r = dict(rows=torch.zeros((T * K + T, H), dtype=torch.float32, device=dev),
                 ids=torch.empty((T, K), dtype=torch.int32, device=dev),
                 weights=torch.empty((T, K), dtype=torch.float32, device=dev),
                 miss_dst=miss, counts=counts)
        _check(lib().smoe_verify_begin(C.byref(self._gc), C.byref(self._wc), table.data_ptr(), x.data_ptr(), T,
                                       r["rows"].data_ptr(), r["ids"].data_ptr(), r["weights"].data_ptr(),
                                       r["miss_dst"].data_ptr(), r["counts"].data_ptr(), self.ws.data_ptr(),
                                       self.ws_bytes, _stream(stream)))
        return r

    def end(self, r: Dict, add_shared: bool = True, y=None, stream=None):
        import torch
        T, H, K = r["ids"].shape[0], self.g.n_embd, self.g.top_k
        _need(r["rows"], "rows", torch.float32, numel=(T * K + T) * H)
        _need(r["weights"], "weights", torch.float32, numel=T * K)
        if y is None:
            y = torch.empty((T, H), dtype=torch.float32, device=r["rows"].device)
        _need(y, "y", torch.float32, numel=T * H)
        _check(lib().smoe_verify_end(C.byref(self._gc), T, r["rows"].data_ptr(), r["weights"].data_ptr(),
                                     int(add_shared), y.data_ptr(), self.ws.data_ptr(), self.ws_bytes,
                                     _stream(stream)))
        return y

