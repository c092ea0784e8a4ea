"""Data-parallel helpers: the path shards by batch, and the only exchange it needs is the sum of
the weight / bias gradients over the ranks (the reference is single-device; its per-batch loop,
package/ext_modules/src/nn/cuda/mapped_convolution_layer.cu:174-190, is what makes the weight
gradient the one cross-batch reduction)."""
import torch
import torch.distributed as dist


def shard_batch(batch, rank, world):
    """Contiguous slice [begin, end) of a batch of `batch` elements owned by `rank`."""
    base, rem = divmod(batch, world)
    begin = rank * base + min(rank, rem)
    return begin, begin + base + (1 if rank < rem else 0)


def allreduce_gradients(tensors, group=None):
    """Sum the given gradient tensors over all ranks with ONE collective: they are flattened into a
    single fp32 bucket, all-reduced, and copied back in place (in their own dtype).
    Returns the bucket (fp32, summed)."""
    tensors = [t for t in tensors if t is not None]
    if not tensors:
        return None
    bucket = torch.cat([t.detach().reshape(-1).float() for t in tensors])
    if dist.is_available() and dist.is_initialized() and dist.get_world_size(group) > 1:
        dist.all_reduce(bucket, op=dist.ReduceOp.SUM, group=group)
    off = 0
    for t in tensors:
        n = t.numel()
        t.detach().copy_(bucket[off:off + n].view_as(t))
        off += n
    return bucket


def gradient_norm(tensors, norm_type=2.0):
    """Norm of all elements of the given gradient tensors together (None entries are left out): 2, 1 or infinity.
    CUDA tensors of one device, float32 / float64 / bfloat16 in any mixture.  Returns a 0-dim float32 tensor (float64 if
    one of the gradients is) without waiting for the device, or None if there is no gradient."""
    from .host import impl
    tensors = [t for t in tensors if t is not None]
    return impl.gradient_norm(tensors, float(norm_type)) if tensors else None


def clip_gradients(tensors, max_norm, norm_type=2.0, out=None):
    """Scale the gradients by min(1, max_norm / (norm + 1e-6)), with the norm over all of them together, as
    torch.nn.utils.clip_grad_norm_ does; behind allreduce_gradients every rank finds the same norm.

    In place, or into `out`: tensors of the same shapes (entries of None gradients are ignored), whose type may differ -
    float32 from bfloat16 gradients, say, rounded once.  Returns the norm before scaling, as gradient_norm does.  A NaN
    norm makes every element NaN; an infinite one makes finite elements zero.  Dense tensors that share memory are refused."""
    from .host import impl
    tensors = list(tensors)
    if out is not None:
        out = list(out)
        if len(out) != len(tensors):
            raise RuntimeError("out must have as many tensors as there are gradients")
        out = [o for o, t in zip(out, tensors) if t is not None]
    tensors = [t for t in tensors if t is not None]
    return impl.clip_gradients(tensors, float(max_norm), float(norm_type), out) if tensors else None
