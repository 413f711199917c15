"""Controller-level replay of a serverless request stream over the swap engines.

Every request goes through the library's controller (``tsw_ctrl_*``, the request handling of
include/server/controller.hpp:130-262,392-453): it asks the scheduler for a GPU and a source,
pins the source replica, lets the eviction policy make room (victims are unloaded first) and
signals the load; on completion it registers the new replica, releases the pin and serves its
queue.  This module is the executor side: it carries those signals out on real engines.
Swap-ins are asynchronous (``tsw_swap_in`` returns once the kernel is enqueued), so swaps on
different GPUs overlap for real and compete for PCIe / NVLink as they would in service.
Requests arrive on the wall clock (optionally compressed by ``speedup``); the client's
inference itself is not run -- it is modelled as ``exec_ms`` of GPU occupancy per request,
a stated constant per architecture, because only the swap path is under test.  With
``--decode-tokens`` the functions of the language-model sets run the attention of that many generated
tokens instead (``PromptDecode``): over their own prompt, whose keys and values are parameters that the
swap brings along, and over a cache in the function's workspace.

    python -m torpor_b200.serving --gpus 8 --models 64 --rate 200 --duration 120 --cap-gb 40
    python -m torpor_b200.serving --archs llama_mid --models 4 --decode-tokens 16 --prompt-tokens 2048
"""
from __future__ import annotations

import argparse
import collections
import ctypes as C
import json
import time
from typing import Dict, List, Optional

import numpy as np

from . import _cabi
from . import workloads as W
from ._cabi import check
from .memory_manager import (Controller, MemoryManager, repo_reset, REQ_EXECUTE, REQ_EXECUTE_AFTER_LOAD,
                             SIGNAL_EXECUTE, SIGNAL_LOAD, SIGNAL_STARTUP, SIGNAL_UNLOAD)

# GPU occupancy per request once the weights are there (ms).  Stand-ins for the client's
# inference, in the range the reference's own node simulator uses (misc/tools/node_simu.py:98-99).
EXEC_MS = {"resnet50": 8.0, "bert_base": 12.0, "bert_large": 25.0, "vgg19": 12.0,
           "bert_tiny": 2.0, "llama_tiny": 4.0, "llama_mid": 20.0, "llama2_7b": 30.0}
LEVEL = {"resnet50": 0, "bert_tiny": 0, "bert_base": 1, "vgg19": 1, "llama_tiny": 1, "bert_large": 2,
         "llama_mid": 2, "llama2_7b": 2}


class PromptDecode:
    """One request of a language-model function on an engine: the attention of ``steps`` generated tokens, layer by
    layer, each appending its rotated keys and values to a cache of the request and attending to the
    function's prompt and to that cache.  Every operand is the function's own memory, named by its client
    addresses: the prompt lies among the parameters, the rest in one workspace block.  The projections around it are
    not run; queries, keys and values are taken from a fixed buffer.  Calls may be enqueued right behind a
    swap-in: the stream waits for the prompt of each layer, the host does not."""

    def __init__(self, arch: str, prompt_tokens: int, steps: int, page_size: int = 16, theta: float = 10000.0):
        if prompt_tokens < 1 or steps < 1:
            raise ValueError("a decode needs a prompt and at least one step")
        self.shape, self.prompt, self.steps, self.page_size = W.ATTENTION[arch], prompt_tokens, steps, page_size
        a = self.shape
        self.row = 2 * a.head_dim
        self.own_pages, self.prompt_pages = -(-steps // page_size), -(-prompt_tokens // page_size)
        rng = np.random.default_rng(steps)
        values = lambda heads: (rng.standard_normal(heads * a.head_dim) * 0.5).astype(np.float16)
        self.tables = {"inv_freq": theta ** (-np.arange(0, a.head_dim, 2, dtype=np.float64) / a.head_dim),
                       "prefix_table": np.arange(self.prompt_pages, dtype=np.int32),
                       "page_table": np.arange(self.own_pages, dtype=np.int32),
                       "lens": np.arange(1, steps + 1, dtype=np.int32), "cu_q": np.array([0, 1], dtype=np.int32),
                       "q": values(a.heads), "k": values(a.kv_heads), "v": values(a.kv_heads)}
        sizes = {n: t.nbytes for n, t in self.tables.items()}
        sizes["q_out"] = sizes["out"] = a.heads * self.row
        pages = self.own_pages * page_size * a.kv_heads * self.row
        for l in range(a.layers):
            sizes["keys", l] = sizes["values", l] = pages
        at, self.offset = 0, {}
        for n, size in sizes.items():
            self.offset[n] = at
            at += (size + 255) // 256 * 256
        # the tables lie in front: one copy to the block's own address brings them all
        self.image = np.zeros(self.offset["q_out"], dtype=np.uint8)
        for n, t in self.tables.items():
            self.image[self.offset[n]:self.offset[n] + t.nbytes] = t.view(np.uint8)
        self.offset["workspace"], self.workspace_bytes = at, 0
        need = C.c_uint64()
        check(_cabi.lib().tsw_prefix_attention_workspace(C.byref(self._attention(4096, lambda l, w: 4096, 0, 0)), C.byref(need)))
        self.workspace_bytes = need.value
        self.block_bytes = (at + need.value + W.MiB - 1) // W.MiB * W.MiB

    def _pages(self, k: int, v: int, pages: int) -> "_cabi.KvPages":
        a, row = self.shape, self.row
        token, page = a.kv_heads * row, self.page_size * a.kv_heads * row
        return _cabi.KvPages(k, v, page, token, row, page, token, row, pages, self.page_size)

    def _own(self, base: int, layer: int, step: int):
        o = self.offset
        return (self._pages(base + o["keys", layer], base + o["values", layer], self.own_pages),
                _cabi.KvBatch(base + o["page_table"], base + o["lens"] + 4 * step, base + o["cu_q"], 1, self.own_pages, self.own_pages, 1))

    def _append(self, base: int, layer: int, step: int) -> "_cabi.KvAppendArgs":
        a, o, x = self.shape, self.offset, _cabi.KvAppendArgs()
        x.cache, x.batch = self._own(base, layer, step)
        x.q, x.q_out, x.k, x.v = base + o["q"], base + o["q_out"], base + o["k"], base + o["v"]
        for n, heads in (("q", a.heads), ("q_out", a.heads), ("k", a.kv_heads), ("v", a.kv_heads)):
            setattr(x, n + "_token_stride", heads * self.row)
            setattr(x, n + "_head_stride", self.row)
        x.inv_freq, x.position_offset, x.rotary_dim = base + o["inv_freq"], self.prompt, a.head_dim
        x.dtype, x.q_heads, x.kv_heads, x.head_dim = _cabi.F16, a.heads, a.kv_heads, a.head_dim
        return x

    def _attention(self, base: int, prompt, layer: int, step: int) -> "_cabi.PrefixAttentionArgs":
        a, o, x = self.shape, self.offset, _cabi.PrefixAttentionArgs()
        x.cache, x.batch = self._own(base, layer, step)
        x.prefix = self._pages(prompt(layer, "keys"), prompt(layer, "values"), self.prompt_pages)
        x.prefix_table, x.prefix_len, x.max_q = base + o["prefix_table"], self.prompt, 1
        x.q, x.out = base + o["q_out"], base + o["out"]
        x.q_token_stride = x.out_token_stride = a.heads * self.row
        x.q_head_stride = x.out_head_stride = self.row
        x.dtype, x.q_heads, x.kv_heads, x.head_dim = _cabi.F16, a.heads, a.kv_heads, a.head_dim
        x.causal, x.scale = 1, a.head_dim ** -0.5
        x.workspace, x.workspace_bytes = base + o["workspace"], self.workspace_bytes
        return x

    def calls(self, engine: MemoryManager, func: str, model: "W.LoadedModel", block: int, stream: int):
        """Everything of one request onto ``stream`` (a cudaStream_t), a layer of a step each time the generator is asked on.
        ``model``: the function as its cold start left it; ``block``: client address of a workspace block of ``block_bytes``."""
        at = {t.name: model.tensor_vaddr[i] for i, t in enumerate(model.ws.tensors) if ".prompt." in t.name}
        prompt = lambda l, what: at[f"model.layers.{l}.prompt.{what}"]
        check(engine.cudaMemcpyAsyncBackendHtoD(block, self.image, stream, False, func))
        for step in range(self.steps):
            for l in range(self.shape.layers):
                engine.kv_append(func, self._append(block, l, step), stream)
                engine.prefix_attention(func, self._attention(block, prompt, l, step), stream)
                yield

    def enqueue(self, engine: MemoryManager, func: str, model: "W.LoadedModel", block: int, stream: int) -> None:
        """All of ``calls`` at once."""
        collections.deque(self.calls(engine, func, model, block, stream), maxlen=0)


def decodes(arch: str, decode_tokens: int) -> bool:
    return decode_tokens > 0 and arch in W.ATTENTION


def served_set(arch: str, decode_tokens: int, prompt_tokens: int, seed: Optional[int] = None) -> "W.WeightSet":
    """The weights of a function of this architecture, with its prompt when it decodes."""
    ws = W.weight_set(arch, seed=seed)
    return W.with_prompt(ws, arch, prompt_tokens) if decodes(arch, decode_tokens) else ws


class SwapServer:
    """N engines under the library's controller (``tsw_ctrl_*``): this class only carries out the
    signals the controller sends -- unload, load (from the host store or a replica), execute -- on
    real engines, and reports completions back, as the reference's executors do
    (include/server/cuda_server.hpp:243-300)."""

    def __init__(self, n_gpus: int, cap_bytes: int, evict_policy: str = "LRU", sched_policy: str = "IA",
                 devices: Optional[List[int]] = None, host_arena_bytes: int = 0, pcie_pairs=None, nvlink=None,
                 shard_min_bytes: int = 0, decode_tokens: int = 0, prompt_tokens: int = 1024):
        self.n = n_gpus
        self.devices = devices or list(range(n_gpus))
        if decode_tokens < 0 or prompt_tokens < 1:
            raise ValueError("decode_tokens must not be negative, and a prompt has a token at least")
        if decode_tokens and min(self.devices) < 0:
            raise ValueError("decode_tokens needs engines on a GPU")
        self.engines = [MemoryManager(cap_bytes, device=self.devices[g], server_id=g, gpu_count=n_gpus,
                                      host_arena_bytes=host_arena_bytes if g == 0 else 0)
                        for g in range(n_gpus)]
        self.ctrl = Controller(n_gpus, cap_bytes, sched_policy, evict_policy, pcie_pairs, nvlink)
        self.arch: Dict[str, str] = {}
        self.nbytes: Dict[str, int] = {}
        self.state = [dict(kind="idle") for _ in range(n_gpus)]
        self.pending = [None] * n_gpus              # a load signalled to GPU g, waiting for its execute signal
        self.arrivals = collections.deque()         # arrival times of queued requests, in the controller's FIFO order
        # 1-link or k-link: a swap-in from the host store of at least this many bytes borrows the PCIe links
        # of the GPUs the scheduler reports free (tsw_sched_helpers); 0 = always one link, as the reference
        self.shard_min_bytes = shard_min_bytes
        self.swaps: List[dict] = []
        self.evictions = 0
        self.local_hits = 0
        self.completed = 0
        self.decoded = 0                            # of them, requests that ran their attention
        # requests whose attention reported something (kv_cache.kv_status): dict(func, gpu, status).  They are not completed ones.
        # The word is one to a device: with several engines on it, the first request to end is charged.
        self.faults: List[dict] = []
        # functions of the language-model sets run the attention of decode_tokens generated tokens; 0 = the constant of every other
        self.decode_tokens, self.prompt_tokens = decode_tokens, prompt_tokens
        self.decode: Dict[str, tuple] = {}          # func -> (PromptDecode, its model, client address of its workspace block)
        self.streams = [0] * n_gpus
        if decode_tokens:
            import torch
            self.streams = [torch.cuda.Stream(device=d) for d in self.devices]

    def close(self):
        for s in self.streams:
            if s:
                s.synchronize()
        for e in self.engines:
            e.close()
        self.ctrl.close()
        repo_reset()

    def decodes(self, arch: str) -> bool:
        return decodes(arch, self.decode_tokens)

    def weight_set(self, arch: str, seed: Optional[int] = None) -> "W.WeightSet":
        """What a function of this architecture brings along: its weights, and its prompt when it decodes."""
        return served_set(arch, self.decode_tokens, self.prompt_tokens, seed)

    # ---- ExecuteAfterLoad (controller.hpp:141-162, 223-227): round-robin placement, load once
    def cold_start(self, func: str, arch: str, seed: int, tensor_data=None):
        ws = self.weight_set(arch, seed)
        decode, blocks = None, (W.SMALL_BLOCK,)
        if self.decodes(arch):
            decode = PromptDecode(arch, self.prompt_tokens, self.decode_tokens)
            blocks += (decode.block_bytes,)
        self.arch[func], self.nbytes[func] = arch, ws.nbytes
        events = self.ctrl.request(REQ_EXECUTE_AFTER_LOAD, func, str(LEVEL.get(arch, 1)))
        g = next(e[1] for e in events if e[0] == "S" and e[2] == SIGNAL_STARTUP)   # every GPU is idle at this point
        model = W.cold_start(self.engines[g], func, ws, tensor_data=tensor_data, workspace_blocks=blocks)
        if decode is not None:
            self.decode[func] = (decode, model, model.workspace_vaddr[1])
        self._carry_out(self.ctrl.complete(g), time.perf_counter())      # registers the replica; may unload others

    def _work(self, g: int, func: str):
        """The function's calls on GPU g, a layer at a time, or None (modelled as a constant)."""
        if func not in self.decode:
            return None
        decode, model, block = self.decode[func]
        return decode.calls(self.engines[g], func, model, block, self.streams[g].cuda_stream)

    def _advance(self, g: int, st: dict) -> None:
        """Enqueue one layer of the work on GPU g; behind the last one an event to wait for."""
        if next(st["work"], self) is self:
            import torch
            st["work"], st["event"] = None, torch.cuda.Event()
            st["event"].record(self.streams[g])

    def _decode_status(self, g: int) -> int:
        """What the kernels of the decode that has just ended on GPU g reported (0 = nothing)."""
        from . import kv_cache
        return kv_cache.kv_status(self.devices[g], self.streams[g].cuda_stream, clear=True)

    def _carry_out(self, events, t_arrival):
        """Executor side of the signals of one controller event."""
        for e in events:
            if e[0] != "S":
                continue
            _, g, sig, func = e
            if sig == SIGNAL_UNLOAD:
                self.engines[g].evict(func)
                self.evictions += 1
            elif sig >= SIGNAL_LOAD:
                src = sig - SIGNAL_LOAD - 1
                if self.engines[g].check_alloc(func):                    # resident: nothing to move (cuda_server.hpp:246)
                    self.pending[g] = None
                else:
                    helpers = []
                    if src < 0 and self.shard_min_bytes and self.nbytes[func] >= self.shard_min_bytes:
                        helpers = [h for h in self.ctrl.helpers(g) if self.state[h]["kind"] == "idle"]
                    self.pending[g] = dict(src=src, t_signal=time.perf_counter(), links=1 + len(helpers))
                    if helpers:                                          # asynchronous either way: kernels enqueued
                        self.engines[g].swap_in_sharded(func, [self.engines[h] for h in helpers])
                    else:
                        self.engines[g].swap_in(func, src)
            elif sig == SIGNAL_EXECUTE:
                st = dict(func=func, t_arrival=t_arrival, work=self._work(g, func), event=None)
                if self.pending[g] is None:
                    self.local_hits += 1
                    st.update(kind="exec", until=time.perf_counter() + EXEC_MS.get(self.arch[func], 10.0) / 1e3)
                else:
                    st.update(kind="swap", **self.pending[g])
                    self.pending[g] = None
                self.state[g] = st

    # ---- Execute (controller.hpp:163-185)
    def submit(self, func: str, now: float) -> bool:
        events = self.ctrl.request(REQ_EXECUTE, func)
        if not events:                                   # every GPU busy, or pinned replicas in the way: the controller queued it
            self.arrivals.append(now)
            return False
        self._carry_out(events, now)
        return True

    def poll(self):
        """Advance every GPU: finished swaps start executing, finished executions complete.  A decode is enqueued a layer to a
        poll, before its swap has ended as well as after: what a poll finds, and when, does not depend on how long a request's
        calls take the host."""
        for g in range(self.n):
            st, now = self.state[g], time.perf_counter()
            if st["kind"] == "swap" and self.engines[g].poll_ready(st["func"]) == 0:
                self.swaps.append(dict(func=st["func"], gpu=g, src=st["src"], bytes=self.nbytes[st["func"]],
                                       ms=(now - st["t_signal"]) * 1e3, t=st["t_signal"], links=st["links"]))
                st["kind"] = "exec"
                st["until"] = now + EXEC_MS.get(self.arch[st["func"]], 10.0) / 1e3
            if st.get("work") is not None:
                self._advance(g, st)
            elif st["kind"] == "exec" and (st["event"].query() if st["event"] is not None else now >= st["until"]):
                self.state[g] = dict(kind="idle")
                status = self._decode_status(g) if st["event"] is not None else 0
                if status:
                    self.faults.append(dict(func=st["func"], gpu=g, status=status))
                else:
                    self.completed += 1
                    self.decoded += st["event"] is not None
                events = self.ctrl.complete(g)                           # replica registered, pin released, queue served
                started = any(e[0] == "S" and e[2] == SIGNAL_EXECUTE for e in events)
                self._carry_out(events, self.arrivals.popleft() if started and self.arrivals else now)

    def busy(self) -> bool:
        return any(st["kind"] != "idle" for st in self.state) or self.ctrl.queue_depth() > 0


def run_stream(n_gpus: int, n_models: int, rate: float, duration_s: float, cap_bytes: int, seed: int = 4,
               speedup: float = 1.0, archs=("resnet50", "bert_base", "bert_large", "vgg19"),
               evict_policy: str = "LRU", zero_weights: bool = True, devices: Optional[List[int]] = None,
               shard_min_bytes: int = 0, pcie_pairs=None, nvlink=None, decode_tokens: int = 0, prompt_tokens: int = 1024) -> dict:
    """The mixed serverless stream: ``n_models`` functions, Zipf popularity, Poisson arrivals."""
    arch_of, times, picks = W.mixed_stream(seed=seed, n_models=n_models, rate=rate, duration_s=duration_s, archs=archs)
    store = sum(W.host_store_bytes(served_set(a, decode_tokens, prompt_tokens)) for a in arch_of)      # refuses unknown sets before any engine
    srv = SwapServer(n_gpus, cap_bytes, evict_policy=evict_policy, host_arena_bytes=0, devices=devices,
                     shard_min_bytes=shard_min_bytes, pcie_pairs=pcie_pairs, nvlink=nvlink, decode_tokens=decode_tokens,
                     prompt_tokens=prompt_tokens)
    t0 = time.time()
    for i, a in enumerate(arch_of):
        ws = srv.weight_set(a)
        data = (lambda k, ws=ws: np.zeros(ws.tensors[k].nbytes, dtype=np.uint8)) if zero_weights else None
        srv.cold_start(f"fn{i}", a, 1000 + i, tensor_data=data)
    cold_s = time.time() - t0
    ev_cold = srv.evictions
    start = time.perf_counter()
    k = 0
    n_req = len(times)
    while k < n_req or srv.busy():
        now = time.perf_counter() - start
        while k < n_req and times[k] / speedup <= now:
            srv.submit(f"fn{int(picks[k])}", now)
            k += 1
        srv.poll()
    wall = time.perf_counter() - start
    ms = np.array([s["ms"] for s in srv.swaps]) if srv.swaps else np.zeros(1)
    by = np.array([s["bytes"] for s in srv.swaps], dtype=np.float64) if srv.swaps else np.zeros(1)
    rel = np.array([s["t"] - start for s in srv.swaps]) if srv.swaps else np.zeros(1)
    fill = rel < wall * 0.25
    host = [s for s in srv.swaps if s["src"] < 0]
    multi = [s for s in host if s["links"] > 1]
    host_ms = np.array([s["ms"] for s in host]) if host else np.zeros(1)
    host_by = np.array([s["bytes"] for s in host], dtype=np.float64) if host else np.zeros(1)
    out = {
        "gpus": n_gpus, "models": n_models, "requests": n_req, "completed": srv.completed, "rate_req_s": rate * speedup,
        "duration_s": wall, "cap_bytes": cap_bytes, "host_store_bytes": store, "cold_start_s": cold_s,
        "evictions_at_cold_start": ev_cold, "evictions_in_service": srv.evictions - ev_cold,
        "local_hits": srv.local_hits, "swaps": len(srv.swaps), "swaps_from_host": len(host),
        "swaps_from_replica": len(srv.swaps) - len(host),
        "host_swaps_over_several_links": len(multi),
        "links_per_host_swap_mean": float(np.mean([s["links"] for s in host])) if host else 0.0,
        "host_swap_ms_p50": float(np.percentile(host_ms, 50)), "host_swap_ms_p99": float(np.percentile(host_ms, 99)),
        "host_swap_gbs_p50": float(np.percentile(host_by / (host_ms / 1e3) / 1e9, 50)) if host else 0.0,
        "swapped_bytes": float(by.sum()) if srv.swaps else 0.0,
        "sustained_swap_gbs": float(by.sum()) / wall / 1e9 if srv.swaps else 0.0,
        "fill_phase_swap_gbs": float(by[fill].sum()) / max(wall * 0.25, 1e-9) / 1e9 if srv.swaps else 0.0,
        "steady_swap_gbs": float(by[~fill].sum()) / max(wall * 0.75, 1e-9) / 1e9 if srv.swaps else 0.0,
        "swap_ms_p50": float(np.percentile(ms, 50)), "swap_ms_p99": float(np.percentile(ms, 99)),
        "swap_ms_max": float(ms.max()),
        "per_swap_gbs_p50": float(np.percentile(by / (ms / 1e3) / 1e9, 50)) if srv.swaps else 0.0,
        "exec_model": "GPU occupancy per request modelled as a constant per architecture (EXEC_MS); inference not run" if not srv.decode else
                      f"attention of {decode_tokens} generated tokens behind a prompt of {prompt_tokens} for the language-model sets; others EXEC_MS",
        "requests_decoded": srv.decoded, "requests_failed": len(srv.faults),
    }
    srv.close()
    return out


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--models", type=int, default=64)
    ap.add_argument("--rate", type=float, default=200.0)
    ap.add_argument("--duration", type=float, default=120.0)
    ap.add_argument("--cap-gb", type=float, default=40.0)
    ap.add_argument("--speedup", type=float, default=1.0)
    ap.add_argument("--policy", default="LRU")
    ap.add_argument("--archs", default="resnet50,bert_base,bert_large,vgg19")
    ap.add_argument("--shard-min-mb", type=float, default=0.0,
                    help="swap-ins from the host store of at least this size borrow idle GPUs' PCIe links (0 = one link)")
    ap.add_argument("--decode-tokens", type=int, default=0,
                    help="functions of the language-model sets run the attention of this many generated tokens per request")
    ap.add_argument("--prompt-tokens", type=int, default=1024, help="length of their own prompt, swapped with their weights")
    ap.add_argument("--seed", type=int, default=4)
    args = ap.parse_args()
    pairs = nvl = None
    if args.gpus > 1:
        from .memory_manager import discover_topology
        pairs, nvl = discover_topology(args.gpus)        # which GPUs share an uplink, which pairs are NVLink peers
    print(json.dumps(run_stream(args.gpus, args.models, args.rate, args.duration, int(args.cap_gb * (1 << 30)),
                                seed=args.seed, speedup=args.speedup, evict_policy=args.policy,
                                archs=tuple(args.archs.split(",")), shard_min_bytes=int(args.shard_min_mb * (1 << 20)),
                                pcie_pairs=pairs, nvlink=nvl, decode_tokens=args.decode_tokens,
                                prompt_tokens=args.prompt_tokens)), flush=True)


if __name__ == "__main__":
    main()
