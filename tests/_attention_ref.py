"""Plain 64-bit packed attention and its gradients, with elementwise bounds on what rounding may do to each result.

Bounds (u = eps / 2 of the 16-bit type, half a step relative): the kernels round p, ds and the results to 16 bits and keep everything
else in fp32.
  a score          its product of D terms and the additions around it: es = 2^-24 (D + 6) (scale sum |q||k| + |bias|) + 2^-24 |lse|
  p                relative error 2 es (exponent and sum) + 2^-20 (exp2, the sum's additions), then u
  out              (u + that) sum p |v|, then u |out|
  D = rowsum(do out), from the rounded out or in fp32: at most its error through out's bound
  ds               p (dp - D): p's error on |ds|, dp's 2^-24 (D + 2) sum |do||v|, D's error; then u
  fp16             values below 2^-14 are off by up to 2^-25 absolute: p counts from a reference at which the sum is at least 1
                   (backward: scaled by 2^12), ds as it is
  gradients        the sums of these, then u |gradient| (a table gradient stays fp32: 2^-18 of the sum of its terms' sizes)
Each is doubled where a factor of the neglected second order could enter (1.05)."""
import torch


def bucket_of(r, buckets, max_distance, bidirectional):
    """In whole numbers: logarithmic bucket t begins at the least d with (d / m)^(n - m) >= (M / m)^t."""
    n, d, first = buckets, max(-r, 0), 0
    if bidirectional:
        n, d = buckets // 2, abs(r)
        first = n if r > 0 else 0
    m = n // 2
    if d < m:
        return first + d
    d = min(d, max_distance)
    return first + min(n - 1, m + sum(d ** (n - m) >= max_distance ** t * m ** (n - m - t) for t in range(1, n - m)))


def reference(q, k, v, lens, causal, scale, key_mask=None, table=None, max_distance=128, bidirectional=True, dout=None):
    """q, k, v [tokens][heads][D] (any device), lens: the sequences' lengths, back to back from row 0.  Everything float64; returns a
    dict of results and of their bounds ("out", "out_tol", ...)."""
    T, H, D = q.shape
    G = H // k.shape[1]
    u = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[q.dtype]
    f32 = 2.0 ** -24
    low = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    dev = q.device
    r = {"out": torch.zeros(T, H, D, dtype=torch.float64, device=dev), "lse": torch.full((H, T), -float("inf"), dtype=torch.float64, device=dev),
         "dq": torch.zeros(T, H, D, dtype=torch.float64, device=dev), "dk": torch.zeros(k.shape, dtype=torch.float64, device=dev),
         "dv": torch.zeros(k.shape, dtype=torch.float64, device=dev)}
    if table is not None:
        r["dtable"] = torch.zeros(table.shape, dtype=torch.float64, device=dev)
    for name in list(r):
        r[name + "_tol"] = torch.zeros_like(r[name])
    start = 0
    for n in lens:
        rows = slice(start, start + n)
        start += n
        if n == 0:
            continue
        at = torch.arange(n, device=dev)
        rel = at[None, :] - at[:, None]
        ok = torch.ones(n, n, dtype=torch.bool, device=dev)
        if causal:
            ok &= rel <= 0
        if key_mask is not None:
            ok &= (key_mask[rows] != 0)[None, :]
        if table is not None:
            num = torch.tensor([bucket_of(x, table.shape[0], max_distance, bidirectional) for x in range(-n + 1, n)], device=dev)[rel + n - 1]
        for h in range(H):
            qh, kh, vh = q[rows, h].double(), k[rows, h // G].double(), v[rows, h // G].double()
            if key_mask is not None:
                off = (key_mask[rows] == 0)[:, None]
                kh, vh = kh.masked_fill(off, 0.0), vh.masked_fill(off, 0.0)
            s, size = qh @ kh.T * scale, qh.abs() @ kh.abs().T * scale
            if table is not None:
                b = table[num, h].double()
                b = torch.where(torch.isinf(b), b, b.clamp(-4096, 4096))       # a finite bias counts as at most 4096 in size
                s, size = s + b, size + torch.where(torch.isinf(b), 0.0, b.abs())
            s = s.masked_fill(~ok, -float("inf"))
            top = s.amax(1, keepdim=True)
            e = torch.where(torch.isinf(s), 0.0, (s - torch.where(torch.isinf(top), 0.0, top)).exp())
            total = e.sum(1, keepdim=True)
            p = e / torch.where(total == 0, 1.0, total)
            lse = torch.where(total == 0, -float("inf"), top + total.log())
            o = p @ vh
            es = f32 * (D + 6) * size + f32 * torch.where(torch.isinf(lse), 0.0, lse.abs())
            ep = (2 * es.masked_fill(~ok, 0.0).amax(1, keepdim=True) + 2.0 ** -20) * 1.05
            out_tol = 1.05 * (p * (u + ep) + low * ok) @ vh.abs() + u * o.abs() + low
            r["out"][rows, h], r["out_tol"][rows, h] = o, out_tol * 1.05 + 1e-30
            r["lse"][h, rows] = lse[:, 0]
            r["lse_tol"][h, rows] = (ep + f32 * 4 * torch.where(torch.isinf(lse), 0.0, lse.abs()))[:, 0]
            if dout is None:
                continue
            do = dout[rows, h].double()
            dp, dp_tol = do @ vh.T, f32 * (D + 2) * (do.abs() @ vh.abs().T)
            Dl = (p * dp).sum(1, keepdim=True)
            D_tol = (do.abs() * out_tol).sum(1, keepdim=True) + f32 * (D + 2) * (do.abs() * o.abs()).sum(1, keepdim=True)
            ds = p * (dp - Dl)
            x_tol = 1.05 * (ds.abs() * ep + p * dp_tol)                       # fp32 part without D
            ds_tol = 1.05 * (x_tol + p * D_tol + u * ds.abs()) + low * ok
            dq = scale * ds @ kh
            r["dq"][rows, h], r["dq_tol"][rows, h] = dq, 1.05 * (scale * ds_tol @ kh.abs() + u * dq.abs()) + low + 1e-30
            r["dk"][rows, h // G] += scale * ds.T @ qh
            r["dk_tol"][rows, h // G] += 1.05 * scale * ds_tol.T @ qh.abs()
            r["dv"][rows, h // G] += p.T @ do
            r["dv_tol"][rows, h // G] += 1.05 * (p * (u + ep) + low / 4096 * ok).T @ do.abs()
            if table is not None:
                each = x_tol + p * (x_tol.sum(1, keepdim=True) + 2.0 ** -18 * (p * dp.abs()).sum(1, keepdim=True)) + 2.0 ** -18 * (p * dp.abs())
                for b in torch.unique(num).tolist():
                    r["dtable"][b, h] += ds[num == b].sum()
                    r["dtable_tol"][b, h] += each[num == b].sum()
    for name in ("dk", "dv"):
        r[name + "_tol"] += u * r[name].abs() + low + 1e-30
    return r


def worst(got, ref, name):
    """max of |got - ref| / bound (values that are infinite in both count as equal)."""
    g, w, tol = got.double(), ref[name], ref[name + "_tol"]
    same = torch.isinf(w) & (g == w)
    if not torch.equal(torch.isfinite(g) | same, torch.ones_like(same)):
        return float("inf")
    x = torch.where(same, 0.0, (g - torch.where(same, g, w)).abs() / (tol + 1e-300))
    return float(x.max()) if x.numel() else 0.0
