from natten_mps_amd.nn._base import _NeighborhoodAttentionND


class NeighborhoodAttention1D(_NeighborhoodAttentionND):
    """1-D neighbourhood attention module over [B, L, C] inputs (``nn/na1d.py`` of the reference).

    Args: embed_dim, num_heads, kernel_size, stride, dilation, is_causal,
    num_kv_heads (GQA/MQA when smaller than num_heads), qkv_bias, qk_scale,
    attn_drop, proj_drop, rotary (a RotaryPlan that turns queries and keys).

    ``cache``: a layer of a PagedKVCache (causal modules, without gradients).
    x then holds the tokens last reserved there, [B, L, C] padded: their keys
    and values are appended and their queries attend to the cache.
    """

    rank = 1

    def forward(self, x, seq_lens=None, *, cache=None):
        if cache is not None and seq_lens is not None:
            raise ValueError("seq_lens and cache exclude each other: the cache has the lengths.")
        return super().forward(x, seq_lens, cache)

    def _attend_cached(self, q, k, v, cache):
        if not self.is_causal[0] or self.stride[0] != 1:
            raise ValueError("a cache needs a causal module of stride 1.")
        if self.attn_drop_p > 0.0:
            raise ValueError("a cache needs attn_drop=0.")
        # fewer would be taken for the last ones, the slots before them left as they were
        if q.shape[1] < cache.cache.new_tokens:
            raise ValueError(f"the cache has {cache.cache.new_tokens} new tokens of a sequence reserved, "
                             f"x holds {q.shape[1]}.")
        turned = cache.append(k, v, query=q if self.rotary is not None else None, plan=self.rotary)
        return cache.attend(q if turned is None else turned, self.kernel_size, self.dilation, scale=self.scale)
