"""Sequences that a backbone continues token by token.

The reference runs the whole sequence again for every call.  :class:`BackboneCache`
keeps what the next token needs -- keys and values in pages, the states and
convolution inputs of the linear attention layers -- so that a prompt is run once
(:meth:`~BackboneCache.prefill`), then continued (:meth:`~BackboneCache.step`) and
branched into candidate continuations that share its pages
(:meth:`~BackboneCache.fork`).  :class:`graphs.StepGraphs` serves steps from recorded
HIP graphs.  The layers run as in :mod:`qdc_amd.backbone`, with the
operators of :mod:`qdc_amd.cache_ops` for what the cache holds.
"""
from __future__ import annotations

import contextlib
import functools
import threading

import numpy as np
import torch

from . import _lib, backbone as bb
from . import cache_ops, ops


def _call(method):
    """A call of the cache: alone, on the model's device, without gradients."""
    @functools.wraps(method)
    def call(self, *args, **kwargs):
        with self._alone():
            return method(self, *args, **kwargs)
    return call


def _host(hidden: torch.Tensor) -> np.ndarray:
    return hidden.float().cpu().numpy()


class BackboneCache:
    """Up to ``rows`` sequences of one model, of up to ``max_tokens`` tokens each, whose
    attention layers share ``pages`` pages of ``page_size`` tokens.

    A sequence is a row number from :meth:`prefill` or :meth:`fork` until
    :meth:`free`.  Invalid ids, masks and rows raise ``ValueError`` before anything
    runs; too few free pages (or rows) raise ``RuntimeError``, and every sequence is
    as it was before the call.  (Where torch itself raises within a call, for want of
    memory say, or the call is interrupted, the rows that it was at are ended.)  One
    call at a time per instance (a lock), all of them on one stream, the device's
    current one, whichever the cache was made on; prefill, step and fork wait for their
    result.  The cache takes
    ``2 * attention layers * pages * kv_heads * page_size * head_dim`` values in the
    model's dtype, and per row and linear attention layer ``value_heads * value_dim *
    key_dim`` float32 values and ``conv_kernel`` rows of the convolution's channels."""

    def __init__(self, model: bb.QwenBackbone, rows: int, pages: int, page_size: int = 64,
                 max_tokens: int | None = None):
        cfg = model.cfg
        if max_tokens is None:
            max_tokens = pages * page_size
        if rows < 1 or pages < 1 or max_tokens < 1 or page_size not in cache_ops.PAGE_SIZES:
            raise ValueError("rows, pages and max_tokens must be positive, page_size one of "
                             f"{cache_ops.PAGE_SIZES}.")
        attention = [i for i, layer in enumerate(model.layers) if layer["kind"] == "full_attention"]
        linear = [i for i, layer in enumerate(model.layers) if layer["kind"] != "full_attention"]
        if attention and cfg.head_dim not in (64, 128, 256):
            raise ValueError("a cache needs attention heads of 64, 128 or 256 values.")
        if linear and (cfg.key_dim not in (32, 64, 128) or cfg.value_dim % 16
                       or cfg.value_dim > 256 or cfg.conv_kernel > 8):
            raise ValueError("a cache needs linear attention keys of 32, 64 or 128 values, values "
                             "of a multiple of 16 up to 256 and at most 8 convolution taps.")
        self.model, self.rows, self.max_tokens = model, rows, max_tokens
        dev, width = model.device, -(-max_tokens // page_size)
        # rows of one call, of which attention takes fewer the more tokens they may hold
        self._most = rows
        while attention and self._most and _lib.lib().qdc_paged_attention_workspace(
                self._most, cfg.heads, cfg.kv_heads, cfg.head_dim, width, page_size,
                ops._DTYPES[model.dtype]) < 0:
            self._most //= 2
        if not self._most:
            raise ValueError("max_tokens is too large.")
        self.book = cache_ops.page_table(rows, width, pages, page_size, dev)
        # planes 2 a and 2 a + 1: K and V of attention layer a
        self.pool = torch.zeros((2 * len(attention), pages, cfg.kv_heads, page_size, cfg.head_dim),
                                dtype=model.dtype, device=dev)
        channels = 2 * cfg.key_heads * cfg.key_dim + cfg.value_heads * cfg.value_dim
        self.states = torch.zeros((len(linear), rows, cfg.value_heads, cfg.value_dim, cfg.key_dim),
                                  dtype=torch.float32, device=dev)
        self.rings = torch.zeros((len(linear), rows, cfg.conv_kernel, channels), dtype=model.dtype,
                                 device=dev)
        self.plane = {i: a for a, i in enumerate(attention)} | {i: a for a, i in enumerate(linear)}
        self.tables = ops.rope_tables(max_tokens, cfg.rotary_dim, cfg.rope_theta, dev) \
            if attention and cfg.rotary_dim else None
        self.scale = float(np.float32(1) / np.sqrt(np.float32(cfg.head_dim)))
        self._flag = torch.zeros(1, dtype=torch.int32, device=dev)
        self._unused = list(range(rows - 1, -1, -1))
        self._lengths = {}     # tokens of every row in use
        self._lock = threading.Lock()
        # the calls may run on another stream than the one that has filled all this
        torch.cuda.current_stream(dev).synchronize()

    # ------------------------------------------------------------- calls --
    @_call
    def lengths(self) -> dict:
        """The rows in use and how many tokens each holds."""
        return dict(self._lengths)

    @_call
    def free_page_count(self) -> int:
        """Pages that no row holds."""
        return int(self.book.free[0].item())

    @_call
    def prefill(self, ids, mask=None):
        """New sequences from host prompts ``[B, S]`` (or one ``[S]``), left-padded where
        ``mask`` is 0.  Returns ``(rows, hidden)``: a row for each prompt and the
        final-normalised hidden state of its last token, ``[B, hidden]`` fp32, as
        ``backbone.batch_backbone_hidden`` gives."""
        ids = np.asarray(ids, np.int64)
        mask = np.ones(ids.shape, np.int64) if mask is None else np.asarray(mask, np.int64)
        ids, mask = np.atleast_2d(ids), np.atleast_2d(mask)
        if ids.ndim != 2 or mask.shape != ids.shape:
            raise ValueError("Input IDs and mask must be [batch, sequence] arrays of one shape.")
        bb.check_sequence(self.model, ids.reshape(-1), mask.reshape(-1))
        if (np.diff(mask, axis=1) < 0).any() or not mask[:, -1].all():
            raise ValueError("A cached prompt is masked only before its first token.")
        start = int(mask.argmax(1).min())        # columns that are padding in every row
        ids, mask = ids[:, start:], mask[:, start:]
        B, S = ids.shape
        counts = mask.sum(1)
        if counts.max() > self.max_tokens:
            raise ValueError(f"A sequence holds at most {self.max_tokens} tokens.")
        cfg = self.model.cfg
        if self._heads() and not ops.attention_fused_takes(self.model.dtype, cfg.head_dim, B, S,
                                                           cfg.heads, cfg.kv_heads):
            raise ValueError("Too many or too long prompts for one call.")
        rows = self._next(B)            # none is taken before the call is done
        self._check_count(B)
        d_ids, d_mask = bb._upload(self.model, ids, mask)
        at = np.arange(S) - (S - counts[:, None])
        d_rows, d_counts, d_at = self._ints(np.asarray(rows), counts, at)
        try:
            cache_ops.extend_pages(self.book, d_rows, d_counts, error_flag=self._flag)
            out = _host(self._prompt(d_ids, d_mask, d_rows, d_at.view(B, S)))
            done = self._settle(rows, counts)
        except BaseException:
            self._abandon(rows, d_rows)
            raise
        return self._answer(done, (rows, out))

    @_call
    def step(self, rows, ids) -> np.ndarray:
        """One more token for each of ``rows`` (distinct rows in use): the
        final-normalised hidden states after it, ``[n, hidden]`` fp32."""
        return self._step(*self._check_step(rows, ids))

    @_call
    def fork(self, rows) -> list:
        """A new sequence for each of ``rows`` (rows in use, any of them several times)
        that holds the same tokens.  Full pages are shared, the rest is copied."""
        parents = self._in_use(rows, distinct=False)
        if not parents:
            return []
        children = self._next(len(parents))
        src, dst = self._ints(np.asarray(parents), np.asarray(children))
        try:
            cache_ops.fork_pages(self.book, src, dst, self._pool(), error_flag=self._flag)
            if self.states.shape[0]:
                for part in zip(src.split(4096), dst.split(4096)):
                    cache_ops.copy_pages(self.states, *part)
                    cache_ops.copy_pages(self.rings, *part)
            done = self._settle(children, [self._lengths[p] for p in parents])
        except BaseException:
            self._abandon(children, dst)
            raise
        return self._answer(done, children)

    @_call
    def free(self, rows) -> None:
        """Ends sequences; their rows and the pages that no other row shares are free."""
        rows = self._in_use(rows)
        if rows:
            self._end(rows, *self._ints(np.asarray(rows)))
            self._unused += rows[::-1]

    @_call
    def compact(self) -> None:
        """Moves the pages in use to the low end of the pool."""
        cache_ops.compact_pages(self.book, self._pool())

    # --------------------------------------------------------- bookkeeping --
    @contextlib.contextmanager
    def _alone(self):
        """One call at a time, on the model's device, without gradients."""
        with self._lock, torch.cuda.device(self.model.device), torch.no_grad():
            yield

    def _check_step(self, rows, ids):
        rows = self._in_use(rows)
        ids = np.asarray(ids, np.int64).reshape(-1)
        if ids.size != len(rows) or not rows:
            raise ValueError("One token ID for each row is required.")
        ops.check_ids(ids, self.model.vocab)
        if any(self._lengths[r] >= self.max_tokens for r in rows):
            raise ValueError(f"A sequence holds at most {self.max_tokens} tokens.")
        self._check_count(len(rows))
        return rows, ids

    def _check_count(self, n: int) -> None:
        if n > self._most:
            raise ValueError(f"With {self.max_tokens} tokens a sequence a call takes at most "
                             f"{self._most} of them.")

    def _step(self, rows, ids) -> np.ndarray:
        d_rows, d_ids = self._ints(np.asarray(rows), ids)
        try:
            out = _host(self._advance(d_rows, d_ids))
            done = self._settle_step(rows)
        except BaseException:
            self._abandon(rows, d_rows)
            raise
        return self._answer(done, out)

    def _advance(self, rows, ids):
        """One more token of each row; an entry with row -1 is none."""
        at = cache_ops.extend_pages(self.book, rows, error_flag=self._flag)
        return self._token(ids, rows, at)

    def _heads(self) -> bool:
        return self.pool.shape[0] > 0

    def _pool(self):
        return self.pool if self._heads() else None

    def _in_use(self, rows, distinct=True) -> list:
        rows = [int(r) for r in np.asarray(rows, np.int64).reshape(-1)]
        if any(r not in self._lengths for r in rows):
            raise ValueError("A row is not in use.")
        if distinct and len(set(rows)) != len(rows):
            raise ValueError("A row is named twice.")
        return rows

    def _next(self, n: int) -> list:
        """The free rows that a call of ``n`` new sequences is to take."""
        if n > len(self._unused):
            raise RuntimeError("Too few free rows.")
        return self._unused[len(self._unused) - n:][::-1]

    def _settle(self, rows, lengths, flagged=None) -> bool:
        """Waits for a call and writes down what its rows hold now, new ones being those
        of :meth:`_next`; nothing, and False, where a kernel flagged it."""
        if int(self._flag.item() if flagged is None else flagged) != 0:
            self._flag.zero_()
            return False
        new = sum(r not in self._lengths for r in rows)
        self._lengths.update({r: int(n) for r, n in zip(rows, lengths)})
        del self._unused[len(self._unused) - new:]
        return True

    def _settle_step(self, rows, flagged=None) -> bool:
        return self._settle(rows, [self._lengths[r] + 1 for r in rows], flagged)

    @staticmethod
    def _answer(done, result):
        if not done:
            raise RuntimeError("Too few free pages.")
        return result

    def _end(self, rows, d_rows=None) -> None:
        # the host first: were what follows to raise, the rows would be lost, and not taken
        # for something that the device does not hold
        for r in rows:
            self._lengths.pop(r, None)
        cache_ops.free_pages(self.book, self._ints(np.asarray(rows))[0] if d_rows is None
                             else d_rows)

    def _abandon(self, rows, d_rows=None) -> None:
        """Ends the rows of a call that raised, wherever it did; what it flagged is not the
        next call's."""
        self._end(rows, d_rows)
        self._flag.zero_()
        free = set(self._unused)
        self._unused += [r for r in rows[::-1] if r not in free]

    def _ints(self, *arrays):
        """Host arrays to the device as int32 vectors, in one copy (what follows starts
        on 16 bytes)."""
        flat = [np.asarray(a).astype(np.int32).reshape(-1) for a in arrays]
        ends = np.cumsum([-(-a.size // 4) * 4 for a in flat])
        packed = np.zeros(int(ends[-1]), np.int32)
        for a, end in zip(flat, ends):
            start = end - -(-a.size // 4) * 4
            packed[start:start + a.size] = a
        dev = torch.from_numpy(packed).to(self.model.device)
        return tuple(dev[end - -(-a.size // 4) * 4:][:a.size] for a, end in zip(flat, ends))

    # -------------------------------------------------------------- layers --
    def _split_proj(self, proj):
        cfg, T = self.model.cfg, proj.shape[0]
        hd, H, KV = cfg.head_dim, cfg.heads, cfg.kv_heads
        return (proj[:, :H * hd].view(T, H, hd), proj[:, H * hd:(H + KV) * hd].view(T, KV, hd),
                proj[:, (H + KV) * hd:(H + 2 * KV) * hd].view(T, KV, hd),
                proj[:, (H + 2 * KV) * hd:].view(T, H, hd))

    def _prompt(self, ids, mask, rows, at):
        """The last-token forward of new prompts, storing keys, values and states."""
        model, cfg = self.model, self.model.cfg
        B, S = ids.shape
        keep = None if mask is None else mask.view(-1)
        token_rows = rows.repeat_interleave(S)
        token_at = at.reshape(-1)
        # the convolution inputs that the rings keep (padding has a projection of zeros)
        last = min(S, cfg.conv_kernel)
        held = rows.long()
        slots = (held[:, None] * cfg.conv_kernel
                 + at[:, -last:].long() % cfg.conv_kernel).view(-1)

        last_row = lambda t: t.view(B, S, *t.shape[1:])[:, -1]  # noqa: E731

        def mix(i, layer, proj):
            a = self.plane[i]
            final = i + 1 == len(model.layers)   # of it only the last tokens go on
            if layer["kind"] == "full_attention":
                q, k, v, gate = self._split_proj(proj)
                keys, values = self.pool[2 * a], self.pool[2 * a + 1]
                k_out = None if final else torch.empty(k.shape, dtype=k.dtype, device=k.device)
                q = cache_ops.prepare_paged(q, k, v, layer["q_norm"], layer["k_norm"], self.tables,
                                            cfg.rotary_dim if self.tables else 0, cfg.eps,
                                            token_rows, token_at, self.book.table, keys, values,
                                            k_out=k_out, error_flag=self._flag)
                out_dtype = model.gemm_in or model.dtype
                if final:
                    return cache_ops.paged_attention(last_row(q), keys, values, self.book.table,
                                                     rows, at[:, -1].contiguous(), self.scale,
                                                     gate=last_row(gate), out_dtype=out_dtype,
                                                     error_flag=self._flag)
                return ops.attention_fused(q, k_out, v, gate, mask, self.scale, B,
                                           out_dtype=out_dtype)
            kd, kh, vd, vh = cfg.key_dim, cfg.key_heads, cfg.value_dim, cfg.value_heads
            kw, vw = kd * kh, vd * vh
            channels = 2 * kw + vw
            q, k, v, beta, decay = ops.delta_prologue(proj, layer["conv"], layer["a_decay"],
                                                      layer["dt_bias"], S, kh, kd, vh, vd,
                                                      interleaved=True)
            state = torch.empty((B, vh, vd, kd), dtype=torch.float32, device=proj.device)
            x = ops.delta_scan(q.view(B, S, kh, kd), k.view(B, S, kh, kd), v.view(B, S, vh, vd),
                               beta.view(B, S, vh), decay.view(B, S, vh), model.dtype, state=state)
            self.states[a].index_copy_(0, held, state)
            self.rings[a].view(-1, channels).index_copy_(
                0, slots, proj.view(B, S, -1)[:, -last:, :channels].reshape(-1, channels))
            z = proj[:, channels:channels + vw].view(-1, vh, vd)
            x = ops.native_gated_rms(x.view(-1, vh, vd), z, layer["norm"], cfg.eps,
                                     out_dtype=model.gemm_in).view(B * S, -1)
            return last_row(x).contiguous() if final else x

        return self._through(ids.reshape(-1).contiguous(), keep, mix,
                             lambda h: last_row(h).contiguous())

    def _token(self, ids, rows, at):
        """One token of each row from and into the cache."""
        model, cfg = self.model, self.model.cfg

        def mix(i, layer, proj):
            a = self.plane[i]
            if layer["kind"] == "full_attention":
                q, k, v, gate = self._split_proj(proj)
                keys, values = self.pool[2 * a], self.pool[2 * a + 1]
                q = cache_ops.prepare_paged(q, k, v, layer["q_norm"], layer["k_norm"], self.tables,
                                            cfg.rotary_dim if self.tables else 0, cfg.eps, rows, at,
                                            self.book.table, keys, values, error_flag=self._flag)
                return cache_ops.paged_attention(q, keys, values, self.book.table, rows, at,
                                                 self.scale, gate=gate,
                                                 out_dtype=model.gemm_in or model.dtype,
                                                 error_flag=self._flag)
            return cache_ops.delta_step(proj, layer["conv"], layer["a_decay"], layer["dt_bias"],
                                        layer["norm"], cfg.eps, self.rings[a], self.states[a], rows,
                                        at, cfg.key_heads, cfg.key_dim, cfg.value_heads,
                                        cfg.value_dim, out_dtype=model.gemm_in,
                                        error_flag=self._flag)

        return self._through(ids, None, mix, lambda t: t)

    def _through(self, ids, keep, mix, last_rows):
        """``QwenBackbone.forward`` around the layers' mixing step; in the last layer it
        gives the rows that go on, of whose residuals ``last_rows`` takes the same."""
        model, cfg = self.model, self.model.cfg
        count = len(model.layers)
        masked = lambda i: keep if model.layers[i]["kind"] != "full_attention" else None  # noqa: E731
        h, normed = ops.native_gather_rms(model.embedding, ids, model.layers[0]["input_norm"],
                                          cfg.eps, token_mask=masked(0),
                                          normed_dtype=model.gemm_in)
        normed = model._first_rows(h, normed, masked(0))
        if model.fused_f32 and ops.linear_f32_takes(ids.shape[0], cfg.hidden, cfg.intermediate):
            return self._through_small(h, normed, masked, mix, last_rows)
        for i, layer in enumerate(model.layers):
            attention = layer["kind"] == "full_attention"
            mixed = mix(i, layer, model._mm(normed, layer["qkv" if attention else "proj"]))
            last = i + 1 == count
            if last:
                h = last_rows(h)
            h, normed = self._project_add_norm(h, mixed, layer, "out", layer["post_norm"],
                                               out_dtype=model.mlp_in)
            act = model._activate(normed, layer["gate_up"])
            norm = model.final_norm if last else model.layers[i + 1]["input_norm"]
            h, normed = self._project_add_norm(h, act, layer, "down", norm,
                                               token_mask=None if last else masked(i + 1),
                                               out_dtype=None if last else model.norm_in)
        return normed

    def _project_add_norm(self, h, a, layer, name, norm, token_mask=None, out_dtype=None):
        """``QwenBackbone._project_add_norm``, for few rows of a split input too through
        ``ops.linear_residual_rms``, which reads the weights once and not twice: with the
        norm, library / here, 1 to 48 rows, us: 3584 to 1024 27 to 29 / 13 to 16, 6144 to
        2048 47 to 55 / 18 to 23, 2048 to 1024 13 to 14 / 11 to 13; from 80 steps of 64 on
        16 parts (2560 to 512 11.9 / 11.1 for 8 / 16 parts, 2048 to 1024 13.4 / 14.6)."""
        rows = layer.get(name + "_rows")
        if rows is not None and a.shape[0] < 64 and a.shape[1] != rows.shape[1] \
                and norm.data_ptr() % 16 == 0:
            return ops.linear_residual_rms(h, a, rows, norm, self.model.cfg.eps,
                                           16 if a.shape[1] >= 80 * 64 else 8,
                                           token_mask=token_mask, out_dtype=out_dtype)
        return self.model._project_add_norm(h, a, layer, name, norm, token_mask=token_mask,
                                            out_dtype=out_dtype)

    def _through_small(self, h, normed, masked, mix, last_rows):
        """``QwenBackbone._forward_small`` around the layers' mixing step."""
        model, eps = self.model, self.model.cfg.eps
        due = None  # the MLP output not yet added to h
        for i, layer in enumerate(model.layers):
            w = layer["qkv" if layer["kind"] == "full_attention" else "proj"]
            if due is None:
                proj = ops.linear_f32(normed, w)
            else:
                h, proj = ops.linear_f32(h, w, add=due, weight=layer["input_norm"], eps=eps,
                                         token_mask=masked(i))
            mixed = mix(i, layer, proj)
            if i + 1 == len(model.layers):
                h = last_rows(h)
            h, act = ops.linear_f32(h, layer["gate_up"], add=ops.linear_f32(mixed, layer["out"]),
                                    weight=layer["post_norm"], eps=eps, swiglu=True)
            due = ops.linear_f32(act, layer["down"])
        return ops.native_residual_rms(h, due, model.final_norm, eps)[1]
