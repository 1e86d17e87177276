from .sharded import BatchShardedRunner, gather_batch, shard_bounds

__all__ = ["ExecutionEngine", "Torch_ExecutionEngine", "BatchShardedRunner", "gather_batch", "shard_bounds", "rotary",
           "kv_append", "paged_attention", "device_status"]


def __getattr__(name):
    # the engines and the decoder operators need the llcompiler_ extension (and a GPU); the sharding helpers do not
    if name in ("ExecutionEngine", "Torch_ExecutionEngine", "TORCH_DTYPE_TO_TYPE"):
        from . import engine as module
    elif name in ("rotary", "kv_append", "paged_attention", "device_status"):
        from . import paged as module
    else:
        raise AttributeError(name)
    value = globals()[name] = getattr(module, name)      # found without this function from now on
    return value
