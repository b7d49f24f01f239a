"""Host-side target preparation and file conventions of the reference, restated for Python 3.

These are the steps either side of the search path (a1, a2, a5) that a drop-in
must reproduce bit for bit so that the engine receives the same query vectors and finds the
same database file.  Plain numpy, no GPU involved.
"""
import os
import re
import numpy as np

SPECIAL_UV_VALUE = -1000.0        # const.py:13
UV_SCALING_FACTOR = 20.0          # const.py:15
VUV_STREAM_NAMES = ['f0', 'lf0']  # const.py:9
TARGET_REP_WIDTHS = {'onepoint': 1, 'twopoint': 2, 'threepoint': 3, 'epoch': 1, 'sample': 1}  # const.py:17


def load_config(config_file):
    """A config is a Python source file exec'd into a dict (synth_simple.py:56-58)."""
    config = {}
    with open(config_file) as f:
        exec(compile(f.read(), config_file, 'exec'), config)
    del config['__builtins__']
    return config


def make_train_condition_name(config):
    """file_naming.py:20-31."""
    if not config['target_representation'] == 'sample':
        jstreams = '-'.join(config['stream_list_join'])
        tstreams = '-'.join(config['stream_list_target'])
        return '%s_utts_jstreams-%s_tstreams-%s_rep-%s' % (
            config['n_train_utts'], jstreams, tstreams, config.get('target_representation', 'twopoint'))
    streams = '-'.join(config['stream_list_target'])
    return '%s_utts_streams-%s_rep-%s' % (config['n_train_utts'], streams,
                                          config.get('target_representation', 'twopoint'))


def get_data_dump_name(config):
    """file_naming.py:5-18 (without creating directories)."""
    return os.path.join(config['workdir'], 'data_dumps', make_train_condition_name(config) + '.hdf5')


def make_synthesis_condition_name(config):
    """file_naming.py:33-67."""
    smooth = 'smooth_' if config.get('synth_smooth', False) else ''
    greedy = 'greedy-yes_' if config.get('greedy_search', False) else 'greedy-no_'
    target_weights = '-'.join([str(val) for val in config['target_stream_weights']])
    if config['target_representation'] == 'sample':
        return 'sample_target-%s' % (target_weights)
    join_weights = '-'.join([str(val) for val in config['join_stream_weights']])
    name = '%s%starget-%s_join-%s_scale-%s_presel-%s_jmetric-%s_cand-%s_taper-%s' % (
        greedy, smooth, target_weights, join_weights, config['join_cost_weight'],
        config['preselection_method'], config.get('join_cost_type', 'natural2'),
        config.get('n_candidates', 30), config.get('taper_length', 50))
    name += 'multiepoch-%s' % (config.get('multiepoch', 1))
    return name


def get_speech(infile, dim):
    """speech_manip.py:102-111: raw little-endian float32 matrix."""
    data = np.fromfile(infile, dtype=np.float32)
    assert data.size % float(dim) == 0.0, 'specified dimension %s not compatible with data' % (dim)
    return data.reshape((-1, dim))


def locate_stream_directories(directories, streams):
    """data_manipulation.py:72-92."""
    stream_directories = {}
    for stream in streams:
        for directory in directories:
            candidate_dir = os.path.join(directory, stream)
            if os.path.isdir(candidate_dir):
                if stream in stream_directories:
                    raise ValueError('Found at least 2 directories for stream %s: %s and %s' % (
                        stream, stream_directories[stream], candidate_dir))
                stream_directories[stream] = candidate_dir
    for stream in streams:
        if stream not in stream_directories:
            raise ValueError('No subdirectory found under %s for stream %s' % (','.join(directories), stream))
    return stream_directories


def compose_speech(feat_dir_dict, base, stream_list, datadims, ignore_streams=('triphone',)):
    """data_manipulation.py:12-70: hstack the streams, unvoiced (<= 0) lf0/f0 -> -1000, trim to
    the shortest stream.  A missing file is signalled by a (1,1) zero matrix, as in the reference."""
    stream_list = [s for s in stream_list if s not in ignore_streams]
    stream_data_list = []
    for stream in stream_list:
        fname = os.path.join(feat_dir_dict[stream], base + '.' + stream)
        if not os.path.isfile(fname):
            return np.zeros((1, 1))
        data = get_speech(fname, datadims[stream])
        if stream == 'aef':
            data = np.vstack([np.zeros((1, datadims[stream])), data, np.zeros((1, datadims[stream]))])
        if stream in VUV_STREAM_NAMES:
            data[data <= 0.0] = SPECIAL_UV_VALUE
        stream_data_list.append(data)
    nframe = min(d.shape[0] for d in stream_data_list)
    return np.hstack([d[:nframe, :] for d in stream_data_list])


def standardise(speech, mean_vec, std_vec):
    """data_manipulation.py:162-186: (x - mean) / std; unvoiced cells become std * -20."""
    uv_positions = (speech == SPECIAL_UV_VALUE)
    mean_vec = np.asarray(mean_vec).reshape((1, -1))
    std_vec = np.asarray(std_vec).reshape((1, -1))
    speech = (speech - mean_vec) / std_vec
    uv_values = std_vec * -1.0 * UV_SCALING_FACTOR
    for column in range(speech.shape[1]):
        speech[:, column][uv_positions[:, column]] = uv_values[0, column]
    return speech


def weight(speech, weight_vec):
    """speech_manip.py:209-213."""
    return speech * np.array(weight_vec).reshape((1, -1))


def stream_weight_vector(weights, stream_list, datadims):
    vec = []
    for i, stream in enumerate(stream_list):
        vec.extend([weights[i]] * datadims[stream])
    return vec


def get_selection_vector(stream_list, stream_dims, truncation_values):
    """synth_simple.py:968-980."""
    assert len(truncation_values) == len(stream_list), (truncation_values, stream_list)
    selection_vector = []
    start = 0
    for stream, trunc in zip(stream_list, truncation_values):
        stream_dim = stream_dims[stream]
        if trunc == -1:
            trunc = stream_dim
        assert trunc <= stream_dim, 'stream %s has only %s dims, cannot truncate to %s' % (stream, stream_dim, trunc)
        selection_vector.extend(range(start, start + trunc))
        start += stream_dim
    return selection_vector


DATABASE_DATASETS = ['train_unit_features', 'train_unit_names', 'filenames', 'mean_target', 'std_target',
                     'mean_join', 'std_join', 'join_contexts', 'unit_index_within_sentence_dset', 'cutpoints',
                     'duration_monophones', 'duration_stats',
                     'start_join_feats', 'end_join_feats',       # the .joindata.hdf5 file of dump_join_data (train_halfphone.py:277-282)
                     'mp_mag', 'mp_imag', 'mp_real', 'mp_fz']    # store_full_magphase (train_simple.py:145-149, synth_simple.py:100-104)


def full_magphase_rows(config, base, m):
    """store_full_magphase (train_simple.py:260-275 = train_halfphone.py:504-517): the utterance's full-resolution analysis
    frames `<full_magphase_dir>/<stream>_full/<base>.<stream>` (mag / imag / real 513 wide, f0 1 wide) without their first
    and last row, in the order (mag, imag, real, f0).  One row per unit is what the reference's HDF5 assignment needs."""
    parts = []
    for extn in ('mag', 'imag', 'real', 'f0'):
        full = get_speech(os.path.join(config['full_magphase_dir'], extn + '_full', base + '.' + extn), 1 if extn == 'f0' else 513)[1:-1, :]
        if full.shape[0] != m:
            raise ValueError('store_full_magphase: %s_full/%s has %d rows without its first and last one, the utterance has %d units'
                             % (extn, base, full.shape[0], m))
        parts.append(full)
    return parts


def load_database(datafile):
    """The train_simple.py / train_halfphone.py unit database as a dict of arrays, read from
    the HDF5 file itself as the reference does (synth_simple.py:72-106): with h5py where it is installed,
    else through libhdf5's C API (snickery_amd.hdf5_io: the target image ships the library but no h5py),
    else from the ``<datafile>.npz`` sidecar of an older writer."""
    if os.path.isfile(datafile):
        try:
            import h5py
        except ImportError:
            h5py = None
        if h5py is not None:
            out = {}
            with h5py.File(datafile, 'r') as f:
                for k in DATABASE_DATASETS:
                    if k in f:
                        out[k] = f[k][...]
            return out
        from . import hdf5_io
        if hdf5_io.available():
            return hdf5_io.read_datasets(datafile, DATABASE_DATASETS)
    npz = datafile + '.npz'
    if os.path.isfile(npz):
        z = np.load(npz, allow_pickle=False)
        return dict((k, z[k]) for k in z.files)
    if os.path.isfile(datafile):
        raise RuntimeError('%s exists but this interpreter has neither h5py nor a loadable libhdf5 (set SNK_LIBHDF5); '
                           'convert it once with\n  /opt/conda/bin/python3.9 tools/hdf5_to_npz.py %s' % (datafile, datafile))
    raise RuntimeError('data: \n   %s   \ndoes not exist -- try other?' % (datafile))


def gather_stored_magphase(mp_mag, mp_imag, mp_real, mp_fz, path, fzero=None):
    """concatenateMagPhaseEpoch (synth_simple.py:655-674) up to the vocoder call: the analysis frames stored with the
    voice (store_full_magphase), one per selected unit -- (mag, real, imag, fz), what the reference hands to
    magphase.synthesis_from_lossless; a non-empty fzero replaces the stored f0 track."""
    path = np.asarray(path, dtype=np.int64)
    fz = np.asarray(mp_fz)[path, :].reshape((-1, 1))
    if fzero is not None and np.size(fzero) > 0:
        fz = fzero
    return np.asarray(mp_mag)[path, :], np.asarray(mp_real)[path, :], np.asarray(mp_imag)[path, :], fz


def store_database(datafile, db):
    """Write a unit database as the reference's HDF5 (train_simple.py:95-149: one root-level dataset per
    array, first dimension resizable): h5py where installed, else libhdf5 through ctypes; the ``.npz``
    sidecar only where neither exists.  Returns the path written."""
    try:
        import h5py
    except ImportError:
        h5py = None
    if h5py is not None:
        with h5py.File(datafile, 'w') as f:
            for key, arr in db.items():
                kind = '|S50' if arr.dtype.kind == 'S' else ('i' if arr.dtype.kind == 'i' else 'f')
                dset = f.create_dataset(key, arr.shape, dtype=kind, track_times=False)
                dset[...] = arr
        return datafile
    from . import hdf5_io
    if hdf5_io.available():
        hdf5_io.write_datasets(datafile, db)
        return datafile
    np.savez(datafile + '.npz', **db)
    return datafile + '.npz'


# --------------------------------------------------------------------------
# Label-driven halfphone targets (synth_halfphone.py:1527-1549): the host side
# that turns a state-aligned HTK label + frame-level speech into one target row
# per halfphone.  Pinned by tests/golden/reference_mini.npz (halfphone_* keys).
# --------------------------------------------------------------------------
LABEL_DELIMITER = '/'              # const.py:19
HTK_UNITS_PER_FRAME = 50000        # train_halfphone.py:924 (5 ms frames in 100 ns units)
STATES_PER_PHONE = 5


def extract_quinphone(label, quinphone_regex):
    """label_manip.py:7-14: the five phones (ll, l, c, r, rr) of a full-context label."""
    found = re.match(quinphone_regex, label)
    assert found, 'quinphone_regex does not match label %s' % (label,)
    phones = found.groups()
    assert len(phones) == 5
    return phones


def read_label(labfile, quinphone_regex):
    """train_halfphone.py:905-929.  One entry per label line:
    ((start_frame, end_frame), [ll, l, c, r, rr, state]); times floor-divided to frames (the
    reference relies on Python-2 integer division)."""
    entries = []
    with open(labfile, 'r') as f:
        for line in f:
            fields = re.split(r'\s+', line.strip(' \n'))
            if len(fields) < 3:
                raise ValueError('label line with fewer than 3 fields in %s: %r' % (labfile, line))
            start, end, lab = fields[:3]
            state = lab.strip(']').split('[')[-1]
            entries.append(((int(start) // HTK_UNITS_PER_FRAME, int(end) // HTK_UNITS_PER_FRAME),
                            list(extract_quinphone(lab, quinphone_regex)) + [state]))
    return entries


def reinsert_terminal_silence(speech, labels, silence_symbols=('#',)):
    """train_halfphone.py:643-670: zero frames for the leading / trailing silence the label has
    but the (trimmed) speech lacks."""
    lead = 0
    for (_, end), lab in labels:
        if lab[2] not in silence_symbols:
            break
        lead = end
    trail_from = -1
    for (start, _), lab in reversed(labels):
        if lab[2] not in silence_symbols:
            break
        trail_from = start
    trail = labels[-1][0][1] - trail_from
    width = speech.shape[1]
    return np.vstack([np.zeros((lead, width)), speech, np.zeros((trail, width))])


def suppress_weird_festival_pauses(labels, replace_list=('B_150',), replacement='pau'):
    """synth_halfphone.py:116-126."""
    return [(times, [replacement if phone in replace_list else phone for phone in lab])
            for (times, lab) in labels]


def get_halfphone_stats(speech, labels, representation_type='twopoint'):
    """train_halfphone.py:956-1071.  HTK states 2,3 form the left halfphone and 4,5,6 the right
    one; a unit is described by the frame at its start (first frame of state 2 / 4), middle (last
    frame of state 2 / 5) and end (last frame of state 3 / 6), end frames clamped to the speech.
    Returns (names (2P,) str array, features (2P, reps*dim), timings [(start, end)] * 2P)."""
    if representation_type not in ('onepoint', 'twopoint', 'threepoint'):
        raise ValueError('Unknown halfphone representation type: %s ' % (representation_type,))
    n_frames = speech.shape[0]
    assert len(labels) % STATES_PER_PHONE == 0, 'There must be 5 states for each phone in label'
    n_units = 2 * (len(labels) // STATES_PER_PHONE)
    side_of_state = {'2': '_L', '4': '_R'}
    names, starts, middles, ends = [], [], [], []
    for (start, end), lab in labels:
        end = min(end, n_frames - 1)
        assert len(lab) == 6
        state = lab[5]
        if state in side_of_state:
            phones = list(lab[:5])
            phones[2] += side_of_state[state]
            assert LABEL_DELIMITER not in ''.join(phones), \
                'delimiter %s occurs in one or more name element (%s)' % (LABEL_DELIMITER, phones)
            names.append(LABEL_DELIMITER.join(phones))
            starts.append(start)
        if state in ('2', '5'):
            middles.append(end)
        elif state in ('3', '6'):
            ends.append(end)
        elif state != '4':
            raise ValueError('bad state number %r' % (state,))
    assert len(names) == n_units == len(starts) == len(ends) == len(middles)
    points = {'onepoint': [middles], 'twopoint': [starts, ends],
              'threepoint': [starts, middles, ends]}[representation_type]
    features = np.hstack([speech[p, :] for p in points])
    return np.array(names), features, list(zip(starts, ends))


def get_norm_durations(unit_names, timings, duration_stats, oov_stats=(5.0, 5.0)):
    """train_halfphone.py:1122-1132: (frames - mean) / std per halfphone, statistics looked up by
    the unit's monophone (with _L/_R); (N, 1) float64."""
    out = np.empty((len(unit_names), 1), dtype=np.float64)
    for i, (name, (start, end)) in enumerate(zip(unit_names, timings)):
        mean, std = duration_stats.get(name.split(LABEL_DELIMITER)[2], oov_stats)
        out[i, 0] = (float(end - start) - mean) / std
    return out


# --------------------------------------------------------------------------
# Pieces of the halfphone / pitch-synchronous database writer (train_halfphone.py)
# --------------------------------------------------------------------------
LABEL_LENGTH_DIFF_TOLERANCE = 5          # const.py:10
TARGET_REP_WIDTHS = {'onepoint': 1, 'twopoint': 2, 'threepoint': 3, 'epoch': 1, 'sample': 1}    # const.py:17


def read_pm(fname):
    """train_halfphone.py:852-875: pitch-mark times (seconds) of an EST track file -- first field
    of every line after 'EST_Header_End'.  Times that are not non-decreasing: a (1, 1) array of
    ones, the reference's signal for an unusable file."""
    with open(fname, 'r') as f:
        lines = f.readlines()
    start = None
    for i, line in enumerate(lines):
        if line.startswith('EST_Header_End'):
            start = i + 1
            break
    if start is None:
        raise ValueError('%s: no EST_Header_End line' % (fname,))
    times = np.array([float(re.split(r'\s+', line)[0]) for line in lines[start:]])
    if np.any(np.diff(times) < 0.0):
        return np.ones((1, 1))
    return times


def get_cutpoints(timings, pms, sample_rate):
    """train_halfphone.py:933-955: for every unit (start, end) in 5 ms frames, the pitch marks
    nearest to its two ends (first of equally near ones).  Returns (cutpoints in samples (n, 2) int,
    pitch-mark indices (n, 2) int)."""
    indices = np.empty((len(timings), 2), dtype=int)
    for i, (start, end) in enumerate(timings):
        indices[i, 0] = np.argmin(np.abs(pms - start * 0.005))
        indices[i, 1] = np.argmin(np.abs(pms - end * 0.005))
    cutpoints = pms[indices].reshape((-1, 2)) * sample_rate
    return np.array(cutpoints, dtype=int), indices


def get_contexts_for_pitch_synchronous_joincost(speech, pm_indices):
    """train_halfphone.py:1135-1162: row p = the pitch-synchronous join frame at the START of unit p
    (= end of unit p-1), plus one last row for the end of the last unit: (n + 1, dim)."""
    starts = np.append(pm_indices[:, 0], pm_indices[-1, 1])
    return speech[starts, :]


def pad_speech_to_length(speech, labels):
    """train_halfphone.py:1333-1356: zero-pad or trim the speech to the label's frame count; more
    than LABEL_LENGTH_DIFF_TOLERANCE frames apart: a (1, 1) zero matrix (utterance is skipped)."""
    m, dim = speech.shape
    nframe = labels[-1][0][1]
    if abs(nframe - m) > LABEL_LENGTH_DIFF_TOLERANCE:
        return np.array([[0.0]])
    if nframe > m:
        return np.vstack([speech, np.zeros((nframe - m, dim))])
    return speech[:nframe, :]


def get_halfphone_lengths(label):
    """train_halfphone.py:1098-1119: (monophone + '_L' / '_R', frames) per halfphone; HTK states
    2-3 form the left halfphone, 4-6 the right one."""
    vals, curr_dur = [], 0
    for (start, end), quinphone in label:
        curr_dur += end - start
        state = quinphone[-1]
        if state == '3':
            vals.append((quinphone[2] + '_L', curr_dur))
            curr_dur = 0
        if state == '6':
            vals.append((quinphone[2] + '_R', curr_dur))
            curr_dur = 0
    return vals


# --------------------------------------------------------------------------
# Per-stream standardisation statistics of the database writer
# (data_manipulation.py:96-234; used by train_simple.py:86-87)
# --------------------------------------------------------------------------
def _readable_streams(flist, dim, exclude_uv):
    """The stream files that exist and hold only finite values; for VUV streams only the voiced
    frames (first column > 0)."""
    for fname in flist:
        if not os.path.isfile(fname):
            continue
        speech = get_speech(fname, dim)
        if np.sum(np.isnan(speech)) + np.sum(np.isinf(speech)) > 0:
            continue                                   # the reference prints 'EXCLUDE' and moves on
        if exclude_uv:
            speech = speech[speech[:, 0] > 0.0, :]
        yield speech


def get_mean(flist, dim, exclude_uv=False):
    """data_manipulation.py:96-123: per-coefficient mean over all frames -> (mean_vec, frame_count)."""
    frame_sum = np.zeros(dim)
    frame_count = 0
    for speech in _readable_streams(flist, dim, exclude_uv):
        frame_sum += speech.sum(axis=0)
        frame_count += speech.shape[0]
    return frame_sum / float(frame_count), frame_count


def get_std(flist, dim, mean_vec, exclude_uv=False):
    """data_manipulation.py:125-160: ONE value per stream -- the largest per-coefficient standard
    deviation -- replicated to a (1, dim) row (the reference's shape)."""
    diff_sum = np.zeros(dim)
    frame_count = 0
    mean_row = np.asarray(mean_vec).reshape((1, -1))
    for speech in _readable_streams(flist, dim, exclude_uv):
        diff_sum += ((speech - mean_row) ** 2).sum(axis=0)
        frame_count += speech.shape[0]
    std_val = (diff_sum.max() / float(frame_count)) ** 0.5
    return np.ones((1, dim)) * std_val


def get_mean_std(feat_dir_dict, stream_list, datadims, flist):
    """data_manipulation.py:205-234: hstack of the per-stream vectors: mean (D,), std (1, D)."""
    means, stds = [], []
    for stream in stream_list:
        stream_files = [os.path.join(feat_dir_dict[stream], base + '.' + stream) for base in flist]
        uv = stream in VUV_STREAM_NAMES
        mean, _ = get_mean(stream_files, datadims[stream], exclude_uv=uv)
        means.append(mean)
        stds.append(get_std(stream_files, datadims[stream], mean, exclude_uv=uv))
    return np.hstack(means), np.hstack(stds)


# --------------------------------------------------------------------------
# Waveform side: analysis frames of the selected units (synth_simple.py:507-747)
# --------------------------------------------------------------------------
FFTHALFLEN = 513                   # const.py: bins of the full-resolution magphase spectra


def lin_interp_f0(fz):
    """speech_manip.py:222-244: f0 linearly interpolated (and extrapolated) through the unvoiced
    stretches, and the voicing flag; both (n, 1).  Same scipy call as the reference."""
    import scipy.interpolate
    y = np.asarray(fz).flatten()
    voiced_ix = np.where(y > 0.0)[0]
    voicing_flag = np.zeros(y.shape)
    voicing_flag[voiced_ix] = 1.0
    if voiced_ix.shape[0] == 0:
        v_interpolated = np.asarray(fz)
    else:
        interpolator = scipy.interpolate.interp1d(voiced_ix, y[voiced_ix], kind='linear', axis=0,
                                                  bounds_error=False, fill_value='extrapolate')
        v_interpolated = interpolator(np.arange(y.shape[0]))
    return (v_interpolated.reshape((-1, 1)), voicing_flag.reshape((-1, 1)))


def in_taper(taper_length):
    """matrix_operations.py:19: the rising half of the Hann cross-fade (the falling half is its mirror)."""
    return np.hanning(((taper_length + 1) * 2) + 1)[1:taper_length + 1]


def load_full_spectra(full_magphase_dir, names, fft_half_len=FFTHALFLEN):
    """The mag / real / imag / f0 analysis files of the given utterances (synth_simple.py:558-563),
    concatenated: spec (rows, 3*H) float32, fzv (rows, 2) float64 = [interpolated f0, voicing], and
    {name: (first_row, end_row)}."""
    specs, fzvs, spans, row = [], [], {}, 0
    for name in names:
        parts = [get_speech(os.path.join(full_magphase_dir, s, name + '.' + s), fft_half_len) for s in ('mag', 'real', 'imag')]
        f0 = get_speech(os.path.join(full_magphase_dir, 'f0', name + '.f0'), 1)
        n = parts[0].shape[0]
        if not all(p.shape[0] == n for p in parts) or f0.shape[0] != n:
            raise ValueError('analysis streams of %s differ in length' % name)
        f0_interp, vuv = lin_interp_f0(f0)
        specs.append(np.hstack(parts))
        fzvs.append(np.hstack([f0_interp.astype(np.float64), vuv]))
        spans[name] = (row, row + n)
        row += n
    return np.vstack(specs), np.vstack(fzvs), spans


def position_bucket_edges(n_buckets, max_distance):
    """Edges of n_buckets buckets of the distance between consecutive units (engine.set_position_bias): the steps 0 (the same
    unit again) and 1 (its natural successor) in buckets of their own, growing distances up to max_distance either side."""
    if n_buckets < 4:
        raise ValueError('position_bucket_edges: at least 4 buckets')
    behind, ahead = (n_buckets - 4) // 2, (n_buckets - 4) - (n_buckets - 4) // 2

    def far(n):
        # n distances from 2 to max_distance, growing by a constant factor where that is more than one step
        out = []
        for i in range(n):
            d = int(round(2.0 * (max_distance / 2.0) ** ((i + 1.0) / n)))
            out.append(max(d, out[-1] + 1 if out else 3))
        return out
    return [-d + 1 for d in reversed(far(behind))] + [0, 1, 2] + far(ahead)
