"""Data formats either side of the hot path, host side, NumPy only.

    load_data(path)                3DGS .ply -> GaussianSet                 load_model.py:7-42
    save_ply(path, gaussians)      the inverse (official 3DGS vertex layout)
    save_gaussians / load_gaussians   npz checkpoint                         gaussian.py:54-56
    read_model(path, ext)          COLMAP cameras / images / points3D       colmap/read_write_model.py:490-509
    qvec2rotmat(qvec)                                                        colmap/read_write_model.py:524
    gaussians_from_point_cloud(points3D)   initial gaussians + kNN scales    gaussian.py:9-29,59-61

The reference reads PLY through `plyfile` and COLMAP through its vendored ETH/UNC reader; neither
is used here: the PLY and COLMAP binary layouts are public formats and are parsed directly.
`plyfile` is not installed in the build image, so PLY parity is pinned by byte-level fixtures written
from the format description, not by the third-party reader ("parity unpinned" against plyfile).
The COLMAP reader is pinned by fixtures written with the reference's own writer
(tests/golden/colmap/; the generating script is committed with the test infrastructure)."""
import collections
import os
import struct

import numpy as np

from .api import GaussianSet, _is_packed
from .packed_sh import WORDS, PackedSH

SH_C0 = 0.28209479177387814     # forward_pass.py:8

# ------------------------------------------------------------------------------------- PLY
_PLY_TYPES = {"char": "i1", "int8": "i1", "uchar": "u1", "uint8": "u1", "short": "i2", "int16": "i2",
              "ushort": "u2", "uint16": "u2", "int": "i4", "int32": "i4", "uint": "u4", "uint32": "u4",
              "float": "f4", "float32": "f4", "double": "f8", "float64": "f8"}


def read_ply_vertices(path):
    """Structured array of the `vertex` element of a PLY file (binary little/big endian or ascii;
    scalar properties only, which is all a 3DGS point cloud holds)."""
    with open(path, "rb") as f:
        if f.readline().strip() != b"ply":
            raise ValueError(f"{path}: not a PLY file")
        fmt, elements, cur = None, [], None
        while True:
            line = f.readline()
            if not line:
                raise ValueError(f"{path}: header has no end_header")
            tok = line.decode("ascii", "replace").split()
            if not tok or tok[0] == "comment" or tok[0] == "obj_info":
                continue
            if tok[0] == "format":
                fmt = tok[1]
            elif tok[0] == "element":
                cur = {"name": tok[1], "count": int(tok[2]), "props": []}
                elements.append(cur)
            elif tok[0] == "property":
                if tok[1] == "list":         # fine after the vertex element (faces); never inside it
                    cur["list"] = True
                    continue
                if tok[1] not in _PLY_TYPES:
                    raise ValueError(f"{path}: unknown property type {tok[1]}")
                cur["props"].append((tok[2], _PLY_TYPES[tok[1]]))
            elif tok[0] == "end_header":
                break
        if fmt not in ("binary_little_endian", "binary_big_endian", "ascii"):
            raise ValueError(f"{path}: unsupported PLY format {fmt}")
        for el in elements:
            if el.get("list"):
                raise ValueError(f"{path}: list properties in or before the vertex element (element {el['name']})")
            end = "<" if fmt != "binary_big_endian" else ">"
            dt = np.dtype([(n, end + t) for n, t in el["props"]])
            if fmt == "ascii":
                rows = [f.readline().split() for _ in range(el["count"])]
                arr = np.zeros(el["count"], dtype=dt)
                for k, (n, _) in enumerate(el["props"]):
                    arr[n] = [r[k] for r in rows]
            else:
                raw = f.read(dt.itemsize * el["count"])
                if len(raw) != dt.itemsize * el["count"]:
                    raise ValueError(f"{path}: truncated element {el['name']}")
                arr = np.frombuffer(raw, dtype=dt)
            if el["name"] == "vertex":
                return arr
    raise ValueError(f"{path}: no vertex element")


def _numbered(names, prefix):
    sel = [n for n in names if n.startswith(prefix)]
    return sorted(sel, key=lambda n: int(n.split("_")[-1]))


def load_data(path):
    """load_model.py:7-42: official-3DGS point_cloud.ply -> GaussianSet(xyz, shs[N,3,16],
    scales (log), rots (w,x,y,z), opacities[N,1] (logits), degrees=3)."""
    v = read_ply_vertices(path)
    names = v.dtype.names
    n = len(v)
    xyz = np.stack([np.asarray(v["x"]), np.asarray(v["y"]), np.asarray(v["z"])], axis=1)
    opacities = np.asarray(v["opacity"])[..., np.newaxis]
    features_dc = np.zeros((n, 3, 1), dtype=np.float32)
    for c in range(3):
        features_dc[:, c, 0] = np.asarray(v[f"f_dc_{c}"])
    rest = _numbered(names, "f_rest_")
    if len(rest) != 3 * 15:
        raise ValueError(f"{path}: expected 45 f_rest_* properties (SH degree 3), found {len(rest)}")
    features_extra = np.zeros((n, len(rest)), dtype=np.float32)
    for k, name in enumerate(rest):
        features_extra[:, k] = np.asarray(v[name])
    features_extra = features_extra.reshape(n, 3, 15)          # (P, F*SH) -> (P, F, SH except DC)
    scales = np.stack([np.asarray(v[s], dtype=np.float64) for s in _numbered(names, "scale_")], axis=1)
    rots = np.stack([np.asarray(v[s], dtype=np.float64) for s in _numbered(names, "rot")], axis=1)
    shs = np.concatenate((features_dc, features_extra), axis=2)                      # [N,3,16]
    return GaussianSet(xyz, shs, scales, rots, opacities)


def save_ply(path, gaussians):
    """Write the official 3DGS vertex layout load_data reads (binary little endian, all float32):
    x y z nx ny nz f_dc_0..2 f_rest_0..44 opacity scale_0..2 rot_0..3."""
    xyz = np.asarray(gaussians.center, dtype=np.float32)
    n = len(xyz)
    sh = gaussians.spherical_harmonics
    if _is_packed(sh):                    # the PLY layout has full-precision coefficients only
        sh = sh.dequantize().cpu().numpy()
    sh = np.asarray(sh, dtype=np.float32).reshape(n, 3, 16)
    names = (["x", "y", "z", "nx", "ny", "nz"] + [f"f_dc_{c}" for c in range(3)] +
             [f"f_rest_{k}" for k in range(45)] + ["opacity"] + [f"scale_{k}" for k in range(3)] +
             [f"rot_{k}" for k in range(4)])
    cols = np.concatenate([xyz, np.zeros((n, 3), np.float32), sh[:, :, 0], sh[:, :, 1:].reshape(n, 45),
                           np.asarray(gaussians.opacity, dtype=np.float32).reshape(n, 1),
                           np.asarray(gaussians.scaling, dtype=np.float32).reshape(n, 3),
                           np.asarray(gaussians.rotation, dtype=np.float32).reshape(n, 4)], axis=1)
    header = "ply\nformat binary_little_endian 1.0\nelement vertex %d\n" % n
    header += "".join(f"property float {nm}\n" for nm in names) + "end_header\n"
    with open(path, "wb") as f:
        f.write(header.encode("ascii"))
        f.write(np.ascontiguousarray(cols, dtype="<f4").tobytes())


# ------------------------------------------------------------------------------------- npz checkpoint
def save_gaussians(file_path, gaussians):
    """gaussian.py:54-56: np.savez with POSITIONAL arrays (arr_0..arr_5 = center, color, sh, scaling,
    rotation, opacity).  `color` is the DC colour ((sh[:, :, 0]) in the [N,3,16] layout): the live
    constructor never sets self.color, so the reference's own save() raises; this keeps its file
    layout.  Packed SH are stored as their records (arr_2 uint32 [N,8], 32 bytes per gaussian)."""
    packed = _is_packed(gaussians.spherical_harmonics)
    sh = gaussians.spherical_harmonics.numpy() if packed else np.asarray(gaussians.spherical_harmonics)
    color = getattr(gaussians, "color", None)
    if color is None:
        # a record starts with the three constant terms in half precision
        color = sh.view(np.float16)[:, :3].astype(np.float64) if packed else sh[:, :, 0]
    np.savez(file_path, np.asarray(gaussians.center), np.asarray(color), sh, np.asarray(gaussians.scaling),
             np.asarray(gaussians.rotation), np.asarray(gaussians.opacity))


def load_gaussians(file_path, degrees=3):
    """Inverse of save_gaussians (the reference has no loader for its own checkpoints).  A checkpoint with packed SH gives
    a GaussianSet whose spherical_harmonics are a PackedSH."""
    path = file_path if str(file_path).endswith(".npz") else str(file_path) + ".npz"
    with np.load(path, allow_pickle=False) as d:
        center, _color, sh, scaling, rotation, opacity = (d[f"arr_{k}"] for k in range(6))
    if sh.dtype == np.uint32:
        if sh.shape != (len(center), WORDS):
            raise ValueError(f"{path}: packed SH records must be [{len(center)},{WORDS}], found {list(sh.shape)}")
        sh = PackedSH(sh)
    return GaussianSet(center, sh, scaling, rotation, opacity, degrees)


# ------------------------------------------------------------------------------------- COLMAP
Camera = collections.namedtuple("Camera", ["id", "model", "width", "height", "params"])
Image = collections.namedtuple("Image", ["id", "qvec", "tvec", "camera_id", "name", "xys", "point3D_ids"])
Point3D = collections.namedtuple("Point3D", ["id", "xyz", "rgb", "error", "image_ids", "point2D_idxs"])

# model id -> (name, number of parameters)   (COLMAP src/base/camera_models.h)
CAMERA_MODELS = {0: ("SIMPLE_PINHOLE", 3), 1: ("PINHOLE", 4), 2: ("SIMPLE_RADIAL", 4), 3: ("RADIAL", 5),
                 4: ("OPENCV", 8), 5: ("OPENCV_FISHEYE", 8), 6: ("FULL_OPENCV", 12), 7: ("FOV", 5),
                 8: ("SIMPLE_RADIAL_FISHEYE", 4), 9: ("RADIAL_FISHEYE", 5), 10: ("THIN_PRISM_FISHEYE", 12)}
_MODEL_BY_NAME = {name: (mid, n) for mid, (name, n) in CAMERA_MODELS.items()}


def _unpack(f, fmt):
    size = struct.calcsize(fmt)
    raw = f.read(size)
    if len(raw) != size:
        raise ValueError("truncated COLMAP file")
    return struct.unpack(fmt, raw)


def read_cameras_binary(path):
    cams = {}
    with open(path, "rb") as f:
        (count,) = _unpack(f, "<Q")
        for _ in range(count):
            cid, model_id, width, height = _unpack(f, "<iiQQ")
            if model_id not in CAMERA_MODELS:
                raise ValueError(f"{path}: unknown camera model id {model_id}")
            name, npar = CAMERA_MODELS[model_id]
            params = np.array(_unpack(f, "<%dd" % npar))
            cams[cid] = Camera(cid, name, width, height, params)
    return cams


def read_images_binary(path):
    images = {}
    with open(path, "rb") as f:
        (count,) = _unpack(f, "<Q")
        for _ in range(count):
            vals = _unpack(f, "<i7di")
            iid, qvec, tvec, cid = vals[0], np.array(vals[1:5]), np.array(vals[5:8]), vals[8]
            name = bytearray()
            while True:
                ch = f.read(1)
                if not ch:
                    raise ValueError(f"{path}: truncated image name")
                if ch == b"\x00":
                    break
                name += ch
            (n2d,) = _unpack(f, "<Q")
            rec = np.frombuffer(f.read(24 * n2d), dtype=np.dtype([("x", "<f8"), ("y", "<f8"), ("id", "<i8")]))
            if len(rec) != n2d:
                raise ValueError(f"{path}: truncated 2D points")
            xys = np.stack([rec["x"], rec["y"]], axis=1) if n2d else np.zeros((0, 2))
            images[iid] = Image(iid, qvec, tvec, cid, name.decode("utf-8"), xys, rec["id"].astype(np.int64))
    return images


def read_points3D_binary(path):
    points = {}
    with open(path, "rb") as f:
        (count,) = _unpack(f, "<Q")
        for _ in range(count):
            vals = _unpack(f, "<Q3d3BdQ")
            pid, xyz, rgb, err, tlen = vals[0], np.array(vals[1:4]), np.array(vals[4:7]), vals[7], vals[8]
            track = np.frombuffer(f.read(8 * tlen), dtype="<i4")
            if len(track) != 2 * tlen:
                raise ValueError(f"{path}: truncated track")
            points[pid] = Point3D(pid, xyz, rgb, err, track[0::2].astype(np.int64), track[1::2].astype(np.int64))
    return points


def _data_lines(path):
    with open(path, "r") as f:
        for line in f:
            line = line.strip()
            if line and not line.startswith("#"):
                yield line


def read_cameras_text(path):
    cams = {}
    for line in _data_lines(path):
        e = line.split()
        cid, model = int(e[0]), e[1]
        if model not in _MODEL_BY_NAME:
            raise ValueError(f"{path}: unknown camera model {model}")
        cams[cid] = Camera(cid, model, int(e[2]), int(e[3]), np.array([float(x) for x in e[4:]]))
    return cams


def read_images_text(path):
    images = {}
    with open(path, "r") as f:
        lines = [ln.rstrip("\n") for ln in f if not ln.lstrip().startswith("#")]
    # two lines per image; the second (2D points) may be empty
    k = 0
    while k < len(lines):
        if not lines[k].strip():
            k += 1
            continue
        e = lines[k].split()
        pts = lines[k + 1].split() if k + 1 < len(lines) else []
        iid = int(e[0])
        xys = np.array([[float(pts[j]), float(pts[j + 1])] for j in range(0, len(pts), 3)]).reshape(-1, 2)
        ids = np.array([int(pts[j + 2]) for j in range(0, len(pts), 3)], dtype=np.int64)
        images[iid] = Image(iid, np.array([float(x) for x in e[1:5]]), np.array([float(x) for x in e[5:8]]),
                            int(e[8]), e[9], xys, ids)
        k += 2
    return images


def read_points3D_text(path):
    points = {}
    for line in _data_lines(path):
        e = line.split()
        track = [int(x) for x in e[8:]]
        points[int(e[0])] = Point3D(int(e[0]), np.array([float(x) for x in e[1:4]]),
                                    np.array([int(x) for x in e[4:7]]), float(e[7]),
                                    np.array(track[0::2], dtype=np.int64), np.array(track[1::2], dtype=np.int64))
    return points


def read_model(path, ext=""):
    """colmap/read_write_model.py:490-509 -> (cameras, images, points3D) dicts keyed by id."""
    if ext == "":
        if os.path.isfile(os.path.join(path, "cameras.bin")):
            ext = ".bin"
        elif os.path.isfile(os.path.join(path, "cameras.txt")):
            ext = ".txt"
        else:
            raise FileNotFoundError(f"no cameras.bin / cameras.txt under {path}")
    if ext == ".txt":
        return (read_cameras_text(os.path.join(path, "cameras.txt")),
                read_images_text(os.path.join(path, "images.txt")),
                read_points3D_text(os.path.join(path, "points3D.txt")))
    if ext == ".bin":
        return (read_cameras_binary(os.path.join(path, "cameras.bin")),
                read_images_binary(os.path.join(path, "images.bin")),
                read_points3D_binary(os.path.join(path, "points3D.bin")))
    raise ValueError(f"unknown COLMAP model extension {ext!r}")


def qvec2rotmat(qvec):
    """colmap/read_write_model.py:524: rotation matrix of the (w,x,y,z) quaternion; for a unit
    quaternion this equals what train.py:25 builds with numpy-quaternion."""
    w, x, y, z = (float(v) for v in qvec)
    return np.array([[1 - 2 * y * y - 2 * z * z, 2 * x * y - 2 * w * z, 2 * z * x + 2 * w * y],
                     [2 * x * y + 2 * w * z, 1 - 2 * x * x - 2 * z * z, 2 * y * z - 2 * w * x],
                     [2 * z * x - 2 * w * y, 2 * y * z + 2 * w * x, 1 - 2 * x * x - 2 * y * y]])


def quat_to_rotmat(qvec):
    """numpy-quaternion's as_rotation_matrix (train.py:25, gaussian.py:41): like qvec2rotmat but
    divides by the squared norm, so it also accepts non-unit quaternions."""
    w, x, y, z = (float(v) for v in qvec)
    s = 2.0 / (w * w + x * x + y * y + z * z)
    return np.array([[1 - s * (y * y + z * z), s * (x * y - z * w), s * (x * z + y * w)],
                     [s * (x * y + z * w), 1 - s * (x * x + z * z), s * (y * z - x * w)],
                     [s * (x * z - y * w), s * (y * z + x * w), 1 - s * (x * x + y * y)]])


# ------------------------------------------------------------------------------------- initial gaussians
def knn_distances(points):
    """gaussian.py:59-61: mean squared distance to the 3 nearest neighbours."""
    from scipy.spatial import KDTree
    k = min(4, len(points))
    distances, _ = KDTree(points).query(points, k=k)
    distances = np.asarray(distances).reshape(len(points), k)
    return (distances[:, 1:] ** 2).mean(1) if k > 1 else np.zeros(len(points))


def gaussians_from_point_cloud(point_cloud_data, rgb_scale=255.0):
    """The reference's first GaussianSet constructor (gaussian.py:9-29; shadowed at HEAD, defect B1):
    centres = point positions, DC colour = (rgb - .5)/C0, log-scale = log(mean squared distance to
    the 3 nearest neighbours) (clipped at 1e-7) on all three axes, rotation [0,0,0,1] in (w,x,y,z)
    storage, opacity .1, degree 0.  COLMAP stores rgb as 0..255 bytes; the reference subtracts .5
    from them unscaled -- here they are first divided by rgb_scale (pass 1.0 to reproduce the
    reference).  SH is laid out [N,3,16] as the live forward path needs."""
    pts = list(point_cloud_data.values()) if hasattr(point_cloud_data, "values") else list(point_cloud_data)
    n = len(pts)
    center = np.array([p.xyz for p in pts], dtype=np.float64).reshape(n, 3)
    color = (np.array([p.rgb for p in pts], dtype=np.float64).reshape(n, 3) / rgb_scale - .5) / SH_C0
    sh = np.zeros((n, 3, 16))
    sh[:, :, 0] = color
    distances = np.clip(knn_distances(center), a_min=.0000001, a_max=None)
    scaling = np.repeat(np.log(distances), 3).reshape(n, 3)
    rotation = np.full((n, 4), [0.0, 0.0, 0.0, 1.0])
    opacity = np.full(n, .1)
    g = GaussianSet(center, sh, scaling, rotation, opacity, degrees=0)
    g.color = color
    return g
